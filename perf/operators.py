"""What a model over symbols (quantised waveform samples, text tokens) has this framework do at its two ends and in its update, as cases
that can be timed and compared.

A case is a dict of plain values with an `op`:

  embed         rows of a table looked up by token and scaled
  embed_grad    the table's gradient from the errors of the looked-up rows
  logprob       log probabilities of given tokens with the distribution's entropy, and the most probable alternatives
  train         a loss over log probabilities and entropies: their values and the gradient of the logits, in one call
  logprob_grad  the gradient of the logits from saved statistics, once the errors of log probabilities and entropies are known
  clip          global norm of a list of gradients, and the gradients scaled down to a norm

Tokens follow the usual skewed distribution (token k about as often as 1 / (k + 1)); a fiftieth of the slots holds no token (-1), as
the padding behind a fraction's shorter sequences does.
"""
import importlib
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _capi():
    return importlib.import_module("project-currennt-public_amd").capi


# ---- the cases --------------------------------------------------------------------------------------------------


def listed():
    return [
        # one generation step of a batch of sixteen: a handful of rows, so the call itself is what costs
        {"name": "embed_step", "op": "embed", "V": 50000, "D": 512, "N": 16, "table": "f16", "out": "f32"},
        # the prompts of a batch: as many rows as a large fraction has slots
        {"name": "embed_prompt", "op": "embed", "V": 100003, "D": 2048, "N": 16381, "table": "bf16", "out": "bf16"},
        # symbols of a quantised waveform into the WaveNet stack's residual size, two waveforms of 16000 samples: every row is long
        {"name": "embed_grad_classes", "op": "embed_grad", "V": 256, "D": 64, "N": 32000, "err": "f32", "grad": "f32"},
        # a large vocabulary: most rows empty or short, a few very long
        {"name": "embed_grad_large", "op": "embed_grad", "V": 65536, "D": 1024, "N": 16384, "err": "bf16", "grad": "f32"},
        # sampling the next token of four sequences from a large vocabulary: few rows, so a row has to be shared out
        {"name": "logprob_step", "op": "logprob", "N": 4, "V": 131072, "type": "bf16", "K": 8, "masked": 0.0},
        # scoring prompts: odd vocabulary, so rows start at any alignment; a part of the vocabulary is ruled out
        {"name": "logprob_prompt", "op": "logprob", "N": 2047, "V": 100003, "type": "bf16", "K": 16, "masked": 0.05},
        # scoring a quantised waveform of 8 bits: very many short rows
        {"name": "logprob_classes", "op": "logprob", "N": 32000, "V": 256, "type": "f32", "K": 4, "masked": 0.0},
        # the WaveNet stack's 1024 output classes over two waveforms of 16000 samples
        {"name": "train_classes", "op": "train", "N": 32000, "V": 1024, "type": "f32"},
        # a training fraction over a large vocabulary
        {"name": "train_large", "op": "train", "N": 4096, "V": 65536, "type": "bf16"},
        # gradient behind a loss that is only known after all rows' log probabilities (a reward, a ratio of two models)
        {"name": "logprob_grad_ratio", "op": "logprob_grad", "N": 3001, "V": 32000, "type": "f16"},
        # the acoustic benchmark model's weights, layer by layer: a small update between two fractions
        {"name": "clip_acoustic", "op": "clip", "count": 9, "least": 512, "most": 1576448, "types": "f32"},
        # a large model's gradients: many tensors of odd sizes and two types
        {"name": "clip_large", "op": "clip", "count": 301, "least": 1001, "most": 6000000, "types": "bf16,f32"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "logprob", "train", "logprob_grad", "clip"])
    one = lambda: rng.choice(["f32", "bf16", "f16"])
    if op in ("embed", "embed_grad"):
        D = _spread(rng, 8, 4096)
        V = min(_spread(rng, 16, 131072), 100_000_000 // D)
        N = min(_spread(rng, 1, 65536), 40_000_000 // D)
        if op == "embed":
            return {"op": op, "V": V, "D": D, "N": N, "table": one(), "out": one()}
        return {"op": op, "V": V, "D": D, "N": N, "err": one(), "grad": one()}
    if op == "clip":
        most = _spread(rng, 1000, 4_000_000)
        return {"op": op, "count": rng.randint(1, 300), "least": _spread(rng, 1, 1000), "most": most,
                "types": rng.choice(["f32", "bf16", "f16", "bf16,f32", "f32,f16"])}
    V = _spread(rng, 24, 131072)
    N = min(_spread(rng, 1, 65536), 130_000_000 // V)
    if op == "logprob":
        return {"op": op, "N": N, "V": V, "type": one(), "K": rng.choice([0, 1, 2, 5, 8, 20]), "masked": rng.choice([0.0, 0.0, 0.1])}
    return {"op": op, "N": N, "V": V, "type": one()}


def _clip_sizes(case):
    """Sizes of the tensors, spread over the logarithm and in no order."""
    n, lo, hi = case["count"], case["least"], case["most"]
    return [int(round(lo * (hi / lo) ** (((k * 37) % n) / max(1, n - 1)))) for k in range(n)]


def _clip_types(case):
    names = case["types"].split(",")
    return [names[k % len(names)] for k in range(case["count"])]


# ---- inputs -----------------------------------------------------------------------------------------------------


def _tokens(g, N, V):
    ids = (torch.rand(N, device="cuda", generator=g, dtype=torch.float64) * math.log(V)).exp().floor().clamp(1, V).int() - 1
    return torch.where(torch.rand(N, device="cuda", generator=g) < 0.02, torch.full_like(ids, -1), ids)


def _logits(g, case):
    N, V = case["N"], case["V"]
    x = torch.randn(N, V, device="cuda", generator=g)
    x *= 2.5
    tokens = _tokens(g, N, V)
    # a trained model has the given token among its better ones
    rows = torch.arange(N, device="cuda")
    x[rows, tokens.clamp(min=0).long()] = 6.0 + torch.randn(N, device="cuda", generator=g)
    if case.get("masked"):
        out = torch.rand(V, device="cuda", generator=g) < case["masked"]
        out[0] = False
        hit = out[tokens.clamp(min=0).long()]
        tokens = torch.where(hit, torch.zeros_like(tokens), tokens)
        x.masked_fill_(out, float("-inf"))
    return x.to(TYPES[case["type"]]), tokens


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    s = {"case": case}
    f32 = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")
    if op == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        s["table"] = torch.randn(V, D, device="cuda", generator=g).to(TYPES[case["table"]])
        s["tokens"] = _tokens(g, N, V)
        s["scale"] = math.sqrt(D)
        s["out"] = torch.empty(N, D, dtype=TYPES[case["out"]], device="cuda")
    elif op == "embed_grad":
        N, V, D = case["N"], case["V"], case["D"]
        s["err"] = torch.randn(N, D, device="cuda", generator=g).mul_(0.01).to(TYPES[case["err"]])
        s["tokens"] = _tokens(g, N, V)
        s["scale"] = math.sqrt(D)
        s["grad"] = torch.empty(V, D, dtype=TYPES[case["grad"]], device="cuda")
        if own:
            s["scratch"] = torch.empty(_capi().embed_scratch(V, D, N), dtype=torch.uint8, device="cuda")
    elif op in ("logprob", "train", "logprob_grad"):
        N, V = case["N"], case["V"]
        s["logits"], s["tokens"] = _logits(g, case)
        # three quarters of the usual temperature when scoring, none in training
        s["scale"] = 4.0 / 3.0 if op == "logprob" else 1.0
        s["logp"], s["lse"], s["entropy"] = f32(N), f32(N), f32(N)
        if op == "logprob":
            K = case["K"]
            s["top_logp"] = f32(N, K)
            s["top_tokens"] = torch.empty(N, K, dtype=torch.int32, device="cuda")
        else:
            # a mean over the slots, weighted; entropies are pushed up a little.  16-bit floats of a short exponent are given the sum
            # instead, as a scaled loss does
            share = 1.0 if case["type"] == "f16" else 1.0 / N
            s["logp_err"] = torch.randn(N, device="cuda", generator=g) * (0.5 * share) - share
            s["entropy_err"] = torch.full((N,), -0.01 * share, device="cuda")
            s["err"] = torch.empty(N, V, dtype=TYPES[case["type"]], device="cuda")
        if op == "logprob_grad":
            # from the forward pass of the same fraction, made here as a user's program has it: in 32 bits
            for a in range(0, N, 512):
                z = s["logits"][a:a + 512].double()
                lse = torch.logsumexp(z, 1)
                s["lse"][a:a + 512] = lse.float()
                s["entropy"][a:a + 512] = (lse - (torch.softmax(z, 1) * z).sum(1)).float()
        if own and op != "logprob_grad":
            s["scratch"] = torch.empty(_capi().logprob_scratch(N, V, case.get("K", 0)), dtype=torch.uint8, device="cuda")
    elif op == "clip":
        sizes, types = _clip_sizes(case), _clip_types(case)
        s["max_norm"] = 1.0
        # one buffer for each type, the tensors side by side in it as a flat list of weights keeps them
        s["flat"], s["clipped"], s["sizes"], s["types"] = {}, {}, sizes, types
        at = {t: 0 for t in set(types)}
        for t in sorted(at):
            total = sum(n for n, k in zip(sizes, types) if k == t)
            s["flat"][t] = torch.randn(total, device="cuda", generator=g).mul_(0.02).to(TYPES[t])
            s["clipped"][t] = torch.empty_like(s["flat"][t])
        s["grads"], s["outs"] = [], []
        for n, t in zip(sizes, types):
            s["grads"].append(s["flat"][t][at[t]:at[t] + n])
            s["outs"].append(s["clipped"][t][at[t]:at[t] + n])
            at[t] += n
        s["result"] = f32(2)
        if own:
            s["set"] = _capi().GradientSet(s["grads"], s["outs"])
    else:
        raise ValueError(op)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    capi, op = _capi(), s["case"]["op"]
    if op == "embed":
        capi.embed_forward(s["table"], s["tokens"], s["out"], scale=s["scale"])
        return s["out"]
    if op == "embed_grad":
        capi.embed_backward(s["tokens"], s["err"], s["grad"], scale=s["scale"], scratch=s["scratch"])
        return s["grad"]
    if op == "logprob":
        top = {"top_logp": s["top_logp"], "top_tokens": s["top_tokens"]} if s["case"]["K"] else {}
        capi.logprob_forward(s["logits"], s["tokens"], s["logp"], s["lse"], s["entropy"], scale=s["scale"], scratch=s["scratch"], **top)
        return {"logp": s["logp"], "lse": s["lse"], "entropy": s["entropy"], **top}
    if op == "train":
        capi.logprob_error_backward(s["logits"], s["tokens"], s["logp_err"], s["entropy_err"], s["logp"], s["lse"], s["entropy"], s["err"],
                                    scale=s["scale"], scratch=s["scratch"])
        return {"logp": s["logp"], "entropy": s["entropy"], "err": s["err"]}
    if op == "logprob_grad":
        capi.logprob_backward(s["logits"], s["tokens"], s["lse"], s["entropy"], s["logp_err"], s["entropy_err"], s["err"], scale=s["scale"])
        return s["err"]
    capi.opt_clip(s["set"], s["max_norm"], s["result"])
    return {"result": s["result"], **s["clipped"]}


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "embed":
        ids = s["tokens"].long()
        rows = s["table"][ids.clamp(min=0)].float() * s["scale"]
        return torch.where((ids >= 0)[:, None], rows, torch.zeros((), device=rows.device)).to(TYPES[case["out"]])
    if op == "embed_grad":
        ids = s["tokens"].long()
        # slots without a token go to a row behind the table
        grad = torch.zeros(case["V"] + 1, case["D"], device="cuda")
        grad.index_add_(0, torch.where(ids >= 0, ids, case["V"]), s["err"].float())
        return (grad[:-1] * s["scale"]).to(TYPES[case["grad"]])
    if op == "clip":
        sums = torch.stack([(g.float() * g.float()).sum() for g in s["grads"]])
        norm = sums.double().sum().sqrt()
        coefficient = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
        result = torch.stack([norm.float(), coefficient])
        return {"result": result, **{t: (x.float() * coefficient).to(x.dtype) for t, x in s["flat"].items()}}
    ids = s["tokens"].long()
    held = ids >= 0
    at = ids.clamp(min=0)[:, None]
    z = s["logits"].float() * s["scale"]
    if op == "logprob_grad":
        logp_all = z - s["lse"][:, None]
        p = logp_all.exp()
        return _plain_gradient(s, p, logp_all, s["entropy"], held, at).to(s["err"].dtype)
    z = z - z.amax(1, keepdim=True)
    peak = s["logits"].float().amax(1) * s["scale"]
    e = z.exp()
    total = e.sum(1)
    log_total = total.log()
    logp = torch.where(held, z.gather(1, at)[:, 0] - log_total, torch.zeros_like(total))
    entropy = log_total - torch.where(e > 0, e * z, torch.zeros_like(e)).sum(1) / total
    if op == "train":
        p = e / total[:, None]
        return {"logp": logp, "entropy": entropy,
                "err": _plain_gradient(s, p, z - log_total[:, None], entropy, held, at).to(s["err"].dtype)}
    out = {"logp": logp, "lse": peak + log_total, "entropy": entropy}
    if case["K"]:
        # the order is that of the logits, and of the tokens where two are the same: one whole number for both
        V = case["V"]
        bits = s["logits"].float().view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 20) + ((1 << 20) - 1 - torch.arange(V, device="cuda"))
        key = key.topk(case["K"], dim=1).values
        top = (1 << 20) - 1 - (key & ((1 << 20) - 1))
        out["top_logp"] = z.gather(1, top) - log_total[:, None]
        out["top_tokens"] = top.int()
    return out


def _plain_gradient(s, p, logp_all, entropy, held, at):
    given = torch.where(held, s["logp_err"], torch.zeros_like(s["logp_err"]))
    err = -given[:, None] * p
    err -= torch.where(p > 0, s["entropy_err"][:, None] * p * (logp_all + entropy[:, None]), torch.zeros_like(p))
    err.scatter_add_(1, at, given[:, None])
    return err * s["scale"]


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        out = torch.zeros(case["N"], case["D"], dtype=torch.float64, device="cuda")
        held = (s["tokens"] >= 0).nonzero()[:, 0]
        out[held] = s["table"].index_select(0, s["tokens"][held]).double() * s["scale"]
        return out
    if op == "embed_grad":
        # the errors in the order of their tokens; a token's sum is the difference of two running sums
        tokens, order = s["tokens"].sort(stable=True)
        vocabulary = torch.arange(case["V"], device="cuda", dtype=torch.int32)
        first, behind = torch.searchsorted(tokens, vocabulary), torch.searchsorted(tokens, vocabulary, right=True)
        grad = torch.empty(case["V"], case["D"], dtype=torch.float64, device="cuda")
        for a in range(0, case["D"], 256):
            run_sum = torch.zeros(case["N"] + 1, min(256, case["D"] - a), dtype=torch.float64, device="cuda")
            run_sum[1:] = s["err"][:, a:a + 256][order].double().cumsum(0)
            grad[:, a:a + 256] = torch.where((behind > first)[:, None], run_sum[behind] - run_sum[first], 0.0)
        return grad * s["scale"]
    if op == "clip":
        squares = 0.0
        for x in s["flat"].values():
            squares += float(x.double().square().sum())
        norm = math.sqrt(squares)
        coefficient = min(1.0, s["max_norm"] / norm) if norm > 0 else 1.0
        return {"result": torch.tensor([norm, coefficient], dtype=torch.float64, device="cuda"),
                **{t: x.double() * coefficient for t, x in s["flat"].items()}}
    N, V, K = case["N"], case["V"], case.get("K", 0)
    out = {n: torch.zeros(N, dtype=torch.float64, device="cuda") for n in ("logp", "lse", "entropy")}
    if K:
        out["top_logp"] = torch.empty(N, K, dtype=torch.float64, device="cuda")
        out["top_tokens"] = torch.empty(N, K, dtype=torch.int32, device="cuda")
    if op != "logprob":
        out["err"] = torch.empty(N, V, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 25) // V)
    for a in range(0, N, step):
        b = min(N, a + step)
        raw = s["logits"][a:b].double()
        logs = torch.log_softmax(raw * s["scale"], 1)
        probs = logs.exp()
        out["lse"][a:b] = torch.logsumexp(raw * s["scale"], 1)
        surprise = torch.nan_to_num(probs * logs, nan=0.0)  # 0 * -inf where a token is ruled out
        out["entropy"][a:b] = -surprise.sum(1)
        token = s["tokens"][a:b].long()
        for_given = torch.zeros(b - a, V, dtype=torch.float64, device="cuda") if op != "logprob" else None
        rows = (token >= 0).nonzero()[:, 0]
        out["logp"][a:b][rows] = logs[rows, token[rows]]
        if op != "logprob":
            given = torch.zeros(b - a, dtype=torch.float64, device="cuda")
            given[rows] = s["logp_err"][a:b][rows].double()
            for_given[rows, token[rows]] = given[rows]
            err = for_given - given[:, None] * probs
            err -= s["entropy_err"][a:b].double()[:, None] * (surprise + probs * out["entropy"][a:b, None])
            out["err"][a:b] = err * s["scale"]
        if K:
            order = raw.sort(dim=1, descending=True, stable=True).indices[:, :K]
            out["top_tokens"][a:b] = order.int()
            out["top_logp"][a:b] = logs.gather(1, order)
    if op == "logprob_grad":
        return out["err"]
    if op == "train":
        return {n: out[n] for n in ("logp", "entropy", "err")}
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "embed":
        N, D = case["N"], case["D"]
        # a row that several slots ask for is read once: at the skewed distribution about this many different ones
        rows = sum(1.0 - (1.0 - math.log1p(1.0 / k) / math.log(case["V"] + 1.0)) ** N for k in range(1, case["V"] + 1))
        return {"bytes": int(rows * D * SIZE[case["table"]] + N * (4 + D * SIZE[case["out"]])), "flops": N * D}
    if op == "embed_grad":
        N, D, V = case["N"], case["D"], case["V"]
        return {"bytes": N * (4 + D * SIZE[case["err"]]) + V * D * SIZE[case["grad"]], "flops": N * D}
    if op == "clip":
        total = sum(n * SIZE[t] for n, t in zip(_clip_sizes(case), _clip_types(case)))
        return {"bytes": 2 * total + 8, "flops": 3 * sum(_clip_sizes(case))}
    N, V = case["N"], case["V"]
    size = SIZE[case["type"]]
    if op == "logprob":
        return {"bytes": N * (V * size + 4 + 12 + 8 * case["K"]), "flops": 6 * N * V}
    return {"bytes": N * (2 * V * size + 4 + 20), "flops": 12 * N * V}
