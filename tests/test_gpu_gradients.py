"""Norm of all gradients and clipping against 64 bits, the clipped optimizer step and the network's clipped update (through the C ABI)."""
import numpy as np
import pytest
import torch

import parity_cases as PC
import symbols as S

pytestmark = pytest.mark.gpu


def _tensors(rng, sizes, types, spread=1.0):
    """tensors side by side in one buffer of their type, so that they begin anywhere"""
    out = []
    for i, n in enumerate(sizes):
        dtype = types[i % len(types)]
        whole = torch.full((n + 12,), 55.0, device="cuda", dtype=dtype)
        whole[1 + i % 7:1 + i % 7 + n] = torch.from_numpy(rng.standard_normal(n) * spread).cuda().to(dtype)
        out.append((whole, whole[1 + i % 7:1 + i % 7 + n]))
    return out


def _norm(tensors):
    return float(np.sqrt(sum((S.f64(t) ** 2).sum() for t in tensors)))


@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.float16], S.TYPES])
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5, 0], [4096], [4097, 3, 2048], [100003] * 3, [1, 2, 3, 5, 8, 13] * 60, [8191, 2 ** 20 + 17]])
def test_norm_and_clipping(sizes, types):
    capi = PC.pkg().capi
    rng = np.random.default_rng(len(sizes))
    held = _tensors(rng, sizes, types)
    grads = [t for _, t in held]
    before = [t.clone() for t in grads]
    norm = _norm(grads)
    result = torch.zeros(2, device="cuda")
    gset = capi.GradientSet(grads)
    capi.opt_grad_norm(gset, 0.5 * norm, result)
    first = result.clone()
    # 64-bit sums: what is left is the rounding to 32 bits
    S.assert_close(S.f64(result), [norm, 0.5], 0.0 if norm == 0 else 1e-12 * norm)
    places = _tensors(rng, sizes, types)
    other = capi.GradientSet(grads, [t for _, t in places])
    capi.opt_clip(other, 0.5 * norm, result)
    assert torch.equal(result, first)
    factor = result[1].item()
    for a, b, (whole, place) in zip(before, grads, places):
        assert torch.equal(a, b)
        want = S.f64(a) * factor
        S.assert_close(S.f64(place), want, S.U * np.abs(want), a.dtype)
        assert whole.double().sum().item() == pytest.approx((place.double().sum() + 55.0 * 12).item())
    capi.opt_clip(gset, 0.5 * norm, result)  # in place
    for b, (_, place), (whole, _) in zip(grads, places, held):
        assert torch.equal(b, place)
        assert (whole == 55.0).sum() >= 12
    capi.opt_clip(gset, 10 * norm, result)   # below the limit: as they are
    for b, (_, place) in zip(grads, places):
        assert torch.equal(b, place)
    assert result[1].item() == 1.0


def test_no_tensors_zeros_and_the_limits_of_values():
    capi = PC.pkg().capi
    result = torch.full((2,), 7.0, device="cuda")
    capi.opt_clip(capi.GradientSet([]), 1.0, result)
    assert result.tolist() == [0.0, 1.0]
    g = torch.zeros(1000, device="cuda")
    capi.opt_clip(capi.GradientSet([g]), 1.0, result)
    assert result.tolist() == [0.0, 1.0] and torch.all(g == 0)
    g = torch.full((1000,), 2.0 ** 100, device="cuda")  # squares overflow 32 bits, the norm does not
    capi.opt_clip(capi.GradientSet([g]), 1.0, result)
    norm = 2.0 ** 100 * np.sqrt(1000.0)
    S.assert_close(S.f64(result), [norm, 1.0 / norm], 0.0)
    S.assert_close(S.f64(g), np.full(1000, 1 / np.sqrt(1000.0)), 3 * S.U)
    g = torch.full((1000,), 2.0 ** -120, device="cuda")  # squares vanish in 32 bits
    capi.opt_grad_norm(capi.GradientSet([g]), float("inf"), result)
    S.assert_close(S.f64(result), [2.0 ** -120 * np.sqrt(1000.0), 1.0], 0.0)


def test_read_twice_and_side_by_side():
    # the same tensor may be read twice, and tensors may touch
    capi = PC.pkg().capi
    g, result = torch.randn(300, device="cuda"), torch.zeros(2, device="cuda")
    capi.opt_grad_norm(capi.GradientSet([g, g], [torch.empty_like(g), torch.empty_like(g)]), 1.0, result)
    assert result[0].item() == pytest.approx(_norm([g, g]), rel=1e-6)
    before = g.clone()
    capi.opt_clip(capi.GradientSet([g[:100], g[100:137], g[137:]]), 0.5, result)
    assert torch.equal(g, before * result[1])


def test_more_than_two_to_the_31_elements():
    capi = PC.pkg().capi
    n = 2 ** 31 + 4099
    g, result = torch.full((n,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16), torch.zeros(2, device="cuda")
    g[-1] = 3.0
    capi.opt_clip(capi.GradientSet([g]), 1.0, result)
    norm = np.sqrt((n - 1) * 2.0 ** -20 + 9.0)
    S.assert_close(S.f64(result), [norm, 1 / norm], 1e-9 * norm)
    f = result[1].item()
    S.assert_close(S.f64(g[-3:]), [2.0 ** -10 * f, 2.0 ** -10 * f, 3 * f], S.U * 3, torch.bfloat16)
    assert g[0] == g[n - 2] == g[2 ** 31] == g[2 ** 31 - 1]


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
def test_a_norm_that_is_no_number_leaves_zeros(bad):
    capi = PC.pkg().capi
    grads = [torch.randn(5001, device="cuda"), torch.randn(77, device="cuda").bfloat16()]
    grads[0][4999] = bad
    result = torch.zeros(2, device="cuda")
    capi.opt_clip(capi.GradientSet(grads), 1.0, result)
    assert not np.isfinite(result[0].item()) and result[1].item() == 0.0
    assert all(torch.all(g == 0) for g in grads)


def test_replayed_from_a_graph_and_on_another_stream():
    capi = PC.pkg().capi
    grads = [torch.randn(n, device="cuda") for n in (100, 70001, 3)]
    places = [torch.empty_like(g) for g in grads]
    result, eager = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
    gset, own = capi.GradientSet(grads, places), capi.GradientSet(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    capi.opt_clip(gset, 1.0, result, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.opt_clip(gset, 1.0, result)
    for k in range(4):
        for g in grads:
            g.normal_()
        result.zero_()
        graph.replay()
        torch.cuda.synchronize()
        copies = [p.clone() for p in places]
        capi.opt_clip(own, 1.0, eager)
        assert torch.equal(result, eager), k
        assert all(torch.equal(a, b) for a, b in zip(copies, grads)), k


@pytest.mark.parametrize("option", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("n", [1, 1000, 2 ** 21 + 5])
def test_clipped_step_is_the_step_on_clipped_gradients(option, n):
    capi = PC.pkg().capi
    g, w = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    stats, deltas = torch.rand(2 * n, device="cuda") + 0.1, torch.randn(n, device="cuda") * 0.01
    clip = torch.zeros(2, device="cuda")
    for poison in (False, True):
        if poison:
            g[n // 2] = float("nan")
        clipped = torch.empty_like(g)
        capi.opt_clip(capi.GradientSet([g], [clipped]), 0.25, clip)
        A = [t.clone() for t in (w, torch.zeros(n, device="cuda"), stats, deltas)]
        B = [t.clone() for t in A]
        tail = (None, 3.0, 0.9, 0.999, 1e-2, 0.5)
        capi.opt_step_clipped(option, A[0], g, A[1], A[2], A[3], *tail, clip)
        capi.opt_step(option, B[0], clipped, B[1], B[2], B[3], *tail)
        for a, b in zip(A, B):
            assert torch.equal(a, b)
        assert all(torch.isfinite(a).all() for a in A)


def _network():
    import json

    capi = PC.pkg().capi
    doc = {"layers": [{"size": 5, "name": "input", "type": "input"}, {"size": 12, "name": "h", "type": "feedforward_tanh", "bias": 1.0},
                      {"size": 3, "name": "out", "type": "feedforward_identity", "bias": 1.0},
                      {"size": 3, "name": "post", "type": "sse"}]}
    net = capi.Network(json.dumps(doc), 4, 10)
    net.randomize(3, 0.2)
    return net


@pytest.mark.parametrize("option", [0, 5])
def test_clipped_update_of_a_network(option):
    rng = np.random.default_rng(0)
    T, Sq = 10, 4
    pat = np.full((T, Sq), 2, np.int8)
    pat[0], pat[-1] = 1, 3
    pat = torch.from_numpy(pat.reshape(-1)).cuda()
    x, y = (torch.from_numpy(rng.standard_normal(T * Sq * d).astype(np.float32)).cuda() for d in (5, 3))
    results = []
    for clipped in (True, False):
        net = _network()
        norm = torch.zeros(2, device="cuda")
        for step in range(3):
            net.load_sequences(pat, T, T, x, y)
            net.forward()
            net.calculate_error()
            net.backward()
            if clipped:
                net.update_clipped(option, 1e-2, 0.9, 40.0, 0.5, norm)
            else:
                PC.pkg().capi.opt_clip(PC.pkg().capi.GradientSet([net.updates]), 0.5, norm)
                net.update(option, 1e-2, 0.9, 40.0)
        results.append((net.weights.clone(), norm.clone()))
        net.close()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert 0 < results[0][1][1].item() < 1


def test_symbols_in_symbols_out_and_the_update():
    """A model of next symbols as it is trained: lookup, dense layer, losses with their gradient, table gradient, clipped step; its gradients
    against 64-bit autograd, whose own rounding is nothing beside fp32's.  Products of 40 and 48 terms on three bf16 parts per value, sums
    over 60 slots: 1e-4 of a tensor's norm, the bar of every product here."""
    capi = PC.pkg().capi
    rng = np.random.default_rng(11)
    V, D, N, scale = 48, 40, 60, 6.0
    tokens = rng.integers(0, V, N).astype(np.int32)
    given = np.roll(tokens, -1).astype(np.int32)
    tokens[7], given[-5:] = -1, -1
    table, W = rng.standard_normal((V, D)).astype(np.float32) * 0.2, rng.standard_normal(D * V + V).astype(np.float32) * 0.2
    dev = lambda a: torch.from_numpy(a).cuda()
    td, gd, tab, Wd = dev(tokens), dev(given), dev(table), dev(W)
    x, logits, err = torch.empty(N, D, device="cuda"), torch.empty(N, V, device="cuda"), torch.empty(N, V, device="cuda")
    prev, dW, dtab = torch.empty(N, D, device="cuda"), torch.empty(D * V + V, device="cuda"), torch.empty(V, D, device="cuda")
    logp, lse, ent = (torch.empty(N, device="cuda") for _ in range(3))
    share = torch.full((N,), -1.0 / N, device="cuda")
    capi.embed_forward(tab, td, x, scale=scale)
    capi.dense_forward(D, V, N, 0, 1.0, Wd, x, logits)
    capi.logprob_error_backward(logits, gd, share, None, logp, lse, ent, err)
    capi.dense_backward(D, V, N, 0, 1.0, Wd, x, logits, err, prev, dW)
    capi.embed_backward(td, prev, dtab, scale=scale)
    result = torch.zeros(2, device="cuda")
    capi.opt_clip(capi.GradientSet([dW, dtab]), 0.1, result)
    # the same in 64 bits: weights are V columns of D inputs, then V biases
    tab64 = torch.from_numpy(table).double().requires_grad_()
    W64 = torch.from_numpy(W).double().requires_grad_()
    ids = torch.from_numpy(tokens.astype(np.int64))
    x64 = torch.where((ids >= 0)[:, None], tab64[ids.clamp(min=0)] * scale, 0.0)
    z = x64 @ W64[:D * V].reshape(V, D).T + W64[D * V:]
    held = torch.from_numpy(given >= 0)
    want_logp = torch.log_softmax(z, 1)[torch.arange(N), torch.from_numpy(given.astype(np.int64)).clamp(min=0)] * held
    (-want_logp.sum() / N).backward()
    norm = float(torch.sqrt((W64.grad ** 2).sum() + (tab64.grad ** 2).sum()))
    assert norm > 0.1
    rel = lambda got, want: float((got.double().cpu() - want).norm() / want.norm())
    assert rel(logp, want_logp.detach()) < 1e-4 and abs(result[0].item() / norm - 1) < 1e-4
    assert rel(dW, W64.grad * (0.1 / norm)) < 1e-4 and rel(dtab, tab64.grad * (0.1 / norm)) < 1e-4
