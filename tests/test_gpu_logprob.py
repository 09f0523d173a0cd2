"""Log probabilities of given tokens, entropies, alternatives and gradients against 64 bits (through the C ABI)."""
import numpy as np
import pytest
import torch

import parity_cases as PC
import symbols as S

pytestmark = pytest.mark.gpu


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _logits(rng, N, V, dtype, spread=2.5):
    return _dev(rng.standard_normal((N, V)) * spread, dtype)


def _forward(capi, x, t, K, scale=1.0):
    N = x.shape[0]
    out = {n: torch.full((N,), 7.0, device="cuda") for n in ("logp", "lse", "entropy")}
    if K:
        out["top_logp"] = torch.full((N, K), 7.0, device="cuda")
        out["top_tokens"] = torch.full((N, K), -7, dtype=torch.int32, device="cuda")
    capi.logprob_forward(x, t, scale=scale, **out)
    return out


def _check_forward(capi, x, tokens, K, scale=1.0):
    scale = float(np.float32(scale))
    got = _forward(capi, x, _dev(tokens), K, scale)
    R = S.Rows(S.f64(x), scale)
    rows = np.arange(len(tokens))
    held = (tokens >= 0) & (tokens < x.shape[1])
    at = np.where(held, tokens, 0)
    S.assert_close(S.f64(got["logp"]), np.where(held, R.logp[rows, at], 0.0), np.where(held, R.tol_logp[rows, at], 0.0))
    S.assert_close(S.f64(got["lse"]), R.lse, R.tol_lse)
    S.assert_close(S.f64(got["entropy"]), R.entropy, R.tol_entropy)
    if K:
        top = got["top_tokens"].cpu().numpy()
        want = R.top(K)
        nans = np.isnan(R.x).sum(1)
        for n in rows:
            left = min(K, x.shape[1] - nans[n])
            assert np.array_equal(top[n, :left], want[n, :left]) and np.all(top[n, left:] == -1), n
        logp = np.where(top >= 0, R.logp[rows[:, None], np.maximum(top, 0)], np.nan)
        S.assert_close(S.f64(got["top_logp"]), logp, R.tol_logp[rows[:, None], np.maximum(top, 0)])
    return got, R


def _tokens(rng, N, V):
    t = rng.integers(0, V, N)
    t[rng.random(N) < 0.15] = -1
    return t.astype(np.int32)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("N,V,K", [
    (1, 1, 1), (1, 2, 2), (3, 63, 5), (5, 64, 64), (9, 255, 4), (6, 256, 1), (4, 257, 8), (7, 512, 3), (3, 513, 20), (2, 1024, 2),
    (3, 2047, 64), (2, 2048, 7), (2, 2049, 7), (3, 8192, 16), (1, 8193, 16), (2, 50001, 33), (1, 131072, 8), (600, 2500, 6), (513, 300, 0),
    (511, 16400, 2), (1, 600000, 50),
    (5, 300, 20), (9, 511, 32), (7, 512, 33), (6, 700, 9), (6, 1024, 32), (5, 1500, 3), (5, 1500, 40), (4, 2048, 32), (2100, 2600, 5), (2049, 2100, 32),
    (2060, 2500, 33), (2048, 2049, 0)])
def test_forward(N, V, K, dtype):
    rng = np.random.default_rng(N * 31 + V)
    _check_forward(PC.pkg().capi, _logits(rng, N, V, dtype), _tokens(rng, N, V), K, scale=0.8)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("V", [70, 900, 5000, 40000])
@pytest.mark.parametrize("times", [1, 50, 200])
def test_rows_that_masks_leave_little_of(times, V, dtype):
    rng = np.random.default_rng(V)
    x = _logits(rng, 12, V, dtype)
    low, inf = torch.finfo(dtype).min, float("inf")
    x[0] = -inf                      # nothing left
    x[1] = low                       # the type's lowest value everywhere: all the same
    x[2] = -inf
    x[2, V - 1] = 1.5                # one token left, the last
    x[3] = low
    x[3, 5] = -3.0
    x[4, 1:V // 2] = -inf
    x[5, V // 2:] = low
    x[6, 3] = float("nan")
    x[7, V - 2] = inf
    x[8] = -inf
    x[8, 4] = float("nan")           # NaN in a masked place
    x[9] = 2.0                       # all equal: ties
    x[10] = torch.finfo(dtype).max
    x[11, :] = float("nan")
    t = np.array([3, 3, V - 1, 5, 0, 0, 3, 3, 5, 7, 9, 1], np.int32)
    capi = PC.pkg().capi
    got, _ = _check_forward(capi, x, t, 6)
    if times > 1:  # among so many that a row is one workgroup's: sums in another order, so values against 64 bits again, tokens the same
        many = _forward(capi, x.repeat(times, 1), _dev(np.tile(t, times)), 6)
        R = S.Rows(S.f64(x), 1.0)
        for k in (0, 1, times - 1):
            part = {n: v[12 * k:12 * k + 12] for n, v in many.items()}
            assert torch.equal(part["top_tokens"], got["top_tokens"])
            S.assert_close(S.f64(part["lse"]), R.lse, R.tol_lse)
            S.assert_close(S.f64(part["entropy"]), R.entropy, R.tol_entropy)
    t[:] = 2
    _check_forward(capi, x, t, 1)


@pytest.mark.parametrize("V", [200, 400, 900, 1500, 3000, 30000, 70001])
def test_alternatives_of_sorted_and_repeated_logits(V):
    capi = PC.pkg().capi
    up = np.linspace(-5, 5, V).astype(np.float32)
    rng = np.random.default_rng(V)
    few = rng.integers(0, 4, V).astype(np.float32)
    x = _dev(np.stack([up, up[::-1], few, np.zeros(V, np.float32), np.where(np.arange(V) % 97 == 96, 3.0, -np.inf).astype(np.float32)]))
    for K in (1, 5, 20, 64):
        got, _ = _check_forward(capi, x, np.zeros(5, np.int32), K)
        if V in (3000, 30000):  # and where a row is a wave's, or a workgroup's
            many = _forward(capi, x.repeat(420, 1), _dev(np.zeros(2100, np.int32)), K)
            assert torch.equal(many["top_tokens"], got["top_tokens"].repeat(420, 1))


def test_rows_anywhere_and_results_that_nobody_asks_for():
    capi = PC.pkg().capi
    rng = np.random.default_rng(2)
    for dtype in S.TYPES:
        for V in (61, 700, 9001):
            wide = _logits(rng, 5, V + 9, dtype)
            x = wide[:, 3:3 + V]
            t = _tokens(rng, 5, V)
            got, _ = _check_forward(capi, x, t, 3)
            _check_forward(capi, wide[1:2, :V].expand(5, V), t, 3)
            lse = torch.zeros(5, device="cuda")
            capi.logprob_forward(x, lse=lse)
            assert torch.equal(lse, got["lse"])
            top = torch.zeros(5, 3, dtype=torch.int32, device="cuda")
            capi.logprob_forward(x, top_tokens=top)
            assert torch.equal(top, got["top_tokens"])
            capi.logprob_forward(x[:0], lse=lse[:0])


def _check_gradients(capi, x, tokens, scale, g, h):
    """both calls that form gradients, also in the logits' place"""
    N, V = x.shape
    scale = float(np.float32(scale))
    t, gd, hd = _dev(tokens), _dev(g), _dev(h)
    f32 = lambda: torch.full((N,), 7.0, device="cuda")
    logp, lse, entropy = f32(), f32(), f32()
    err = torch.full((N, V), 7.0, dtype=x.dtype, device="cuda")
    capi.logprob_error_backward(x, t, gd, hd, logp, lse, entropy, err, scale=scale)
    R = S.Rows(S.f64(x), scale)
    want, tol = R.gradient(tokens, g.astype(np.float64), h.astype(np.float64), False)
    S.assert_close(S.f64(err), want, tol, x.dtype)
    S.assert_close(S.f64(lse), R.lse, R.tol_lse)
    S.assert_close(S.f64(entropy), R.entropy, R.tol_entropy)
    held = (tokens >= 0) & (tokens < V)
    at, rows = np.where(held, tokens, 0), np.arange(N)
    S.assert_close(S.f64(logp), np.where(held, R.logp[rows, at], 0.0), np.where(held, R.tol_logp[rows, at], 0.0))
    saved = torch.full((N, V), 7.0, dtype=x.dtype, device="cuda")
    capi.logprob_backward(x, t, lse, entropy, gd, hd, saved, scale=scale)
    want, tol = R.gradient(tokens, g.astype(np.float64), h.astype(np.float64), True)
    S.assert_close(S.f64(saved), want, tol, x.dtype)
    place = x.clone()
    capi.logprob_backward(place, t, lse, entropy, gd, hd, place, scale=scale)
    assert torch.equal(place.view(torch.uint8), saved.view(torch.uint8))
    place = x.clone()
    again = f32()
    capi.logprob_error_backward(place, t, gd, hd, again, lse, entropy, place, scale=scale)
    assert torch.equal(place.view(torch.uint8), err.view(torch.uint8)) and torch.equal(again.view(torch.int32), logp.view(torch.int32))


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (2, 5), (3, 64), (5, 255), (9, 256), (4, 257), (3, 1024), (5, 1025), (3, 2048), (2, 2049), (7, 4001), (5, 4096), (6, 4097), (3, 9001),
                                 (1, 131072), (64, 50001), (520, 2500), (514, 8200), (600, 20001)])
def test_gradient(N, V, dtype):
    rng = np.random.default_rng(N + V)
    g, h = rng.standard_normal(N).astype(np.float32), (0.3 * rng.standard_normal(N)).astype(np.float32)
    _check_gradients(PC.pkg().capi, _logits(rng, N, V, dtype), _tokens(rng, N, V), 0.75, g, h)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("N,V", [(513, V) for V in (2049, 2500, 4096, 4097, 4090, 8150, 16350, 30001, 60001, 65540, 100003, 131072, 140001)] +
                         [(2100, 2049), (2100, 2500), (2100, 4096), (2100, 4097)])
def test_gradient_of_many_long_rows(N, V, dtype):
    # every form that a row of its own wave or workgroup takes; some of the rows are checked
    capi = PC.pkg().capi
    rng, some = np.random.default_rng(V), [0, 1, 2, 255, 511, N - 1]
    x = torch.randn(N, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V)).mul_(2.5).to(dtype)
    g, h = rng.standard_normal(N).astype(np.float32), (0.3 * rng.standard_normal(N)).astype(np.float32)
    t = _tokens(rng, N, V)
    t[some] = [0, V - 1, -1, 5, V // 2, V - 3]
    f, err = [torch.empty(N, device="cuda") for _ in range(3)], torch.empty_like(x)
    capi.logprob_error_backward(x, _dev(t), _dev(g), _dev(h), *f, err, scale=0.75)
    R = S.Rows(S.f64(x[some]), 0.75)
    want, tol = R.gradient(t[some], g[some].astype(np.float64), h[some].astype(np.float64), False)
    S.assert_close(S.f64(err[some]), want, tol, dtype)
    S.assert_close(S.f64(f[1][some]), R.lse, R.tol_lse)
    S.assert_close(S.f64(f[2][some]), R.entropy, R.tol_entropy)
    held = t[some] >= 0
    at, rows = np.maximum(t[some], 0), np.arange(len(some))
    S.assert_close(S.f64(f[0][some]), np.where(held, R.logp[rows, at], 0.0), np.where(held, R.tol_logp[rows, at], 0.0))
    again, logp = x, torch.empty(N, device="cuda")
    capi.logprob_error_backward(again, _dev(t), _dev(g), _dev(h), logp, f[1], f[2], again, scale=0.75)
    assert torch.equal(again, err) and torch.equal(logp, f[0])


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("V", [70, 900, 5000, 40000])
@pytest.mark.parametrize("times", [1, 80])
def test_gradient_of_masked_rows(times, V, dtype):
    rng = np.random.default_rng(V)
    x = _logits(rng, 7, V, dtype)
    x[0] = -float("inf")
    x[1] = -float("inf")
    x[1, 2] = 0.5
    x[2, 3:V - 1] = -float("inf")
    x[3, V // 2:] = torch.finfo(dtype).min
    x[4, 5] = float("nan")
    x[5, 6] = float("inf")
    t = np.array([2, 2, 1, 0, 3, 3, -1], np.int32)
    if times == 1:
        _check_gradients(PC.pkg().capi, x, t, 1.0, np.ones(7, np.float32), np.full(7, 0.5, np.float32))
        return
    # the same rows among so many that a row is one workgroup's
    N, capi = 7 * times, PC.pkg().capi
    many, g, h = x.repeat(times, 1), np.ones(7), np.full(7, 0.5)
    f, err = [torch.empty(N, device="cuda") for _ in range(3)], torch.empty_like(many)
    capi.logprob_error_backward(many, _dev(np.tile(t, times)), torch.ones(N, device="cuda"), torch.full((N,), 0.5, device="cuda"), *f, err)
    R = S.Rows(S.f64(x), 1.0)
    want, tol = R.gradient(t, g, h, False)
    for k in (0, 1, times - 1):
        S.assert_close(S.f64(err[7 * k:7 * k + 7]), want, tol, dtype)
        S.assert_close(S.f64(f[1][7 * k:7 * k + 7]), R.lse, R.tol_lse)
        S.assert_close(S.f64(f[2][7 * k:7 * k + 7]), R.entropy, R.tol_entropy)


def test_gradient_of_a_row_of_the_types_lowest_value():
    # all the same: the probabilities are 1 / V.  (From a saved lse they cannot be had in 32 bits, so this is the joint call's alone.)
    capi = PC.pkg().capi
    for dtype in S.TYPES:
        x = torch.full((3, 300), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        err, f = torch.empty_like(x), [torch.empty(3, device="cuda") for _ in range(3)]
        capi.logprob_error_backward(x, _dev(np.array([1, 2, 3], np.int32)), torch.ones(3, device="cuda"), None, *f, err)
        want = np.full((3, 300), -1 / 300.0)
        want[np.arange(3), [1, 2, 3]] += 1
        S.assert_close(S.f64(err), want, 64 * S.U, dtype)


def test_gradient_without_one_of_the_errors():
    capi = PC.pkg().capi
    rng = np.random.default_rng(6)
    x, t = _logits(rng, 6, 333, torch.float32), _dev(_tokens(rng, 6, 333))
    one, zero = torch.randn(6, device="cuda"), torch.zeros(6, device="cuda")
    f = [torch.empty(6, device="cuda") for _ in range(3)]
    err, other = torch.empty_like(x), torch.empty_like(x)
    for call in (lambda g, h, e: capi.logprob_error_backward(x, t, g, h, *f, e), lambda g, h, e: capi.logprob_backward(x, t, f[1], f[2], g, h, e)):
        call(one, None, err)
        call(one, zero, other)
        assert torch.equal(err, other)
        call(None, one, err)
        call(zero, one, other)
        assert torch.equal(err, other)
    capi.logprob_backward(x, None, f[1], f[2], None, one, other)
    assert torch.equal(err, other)


def test_gradient_against_differences():
    capi = PC.pkg().capi
    rng = np.random.default_rng(9)
    N, V, scale = 3, 11, 1.25
    x = rng.standard_normal((N, V)).astype(np.float32)
    t, g, h = np.array([4, -1, 0], np.int32), rng.standard_normal(N), rng.standard_normal(N)

    def loss(z):
        R = S.Rows(z, scale)
        return sum(g[n] * (R.logp[n, t[n]] if t[n] >= 0 else 0.0) + h[n] * R.entropy[n] for n in range(N))

    want, step = np.zeros((N, V)), 1e-5
    for i in range(N):
        for j in range(V):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[i, j] += step
            down[i, j] -= step
            want[i, j] = (loss(up) - loss(down)) / (2 * step)
    err, f = torch.empty(N, V, device="cuda"), [torch.empty(N, device="cuda") for _ in range(3)]
    capi.logprob_error_backward(_dev(x), _dev(t), _dev(g.astype(np.float32)), _dev(h.astype(np.float32)), *f, err, scale=scale)
    # differences: third derivatives times step^2 / 6 and 64-bit rounding over the step, both below 1e-9; fp32: some hundred u
    S.assert_close(S.f64(err), want, 1e-8 + 200 * S.U * (np.abs(g) + np.abs(h))[:, None])


def test_on_another_stream_and_replayed_from_a_graph():
    capi = PC.pkg().capi
    rng = np.random.default_rng(5)
    N, V, K = 3, 70000, 5
    x, t = _logits(rng, N, V, torch.bfloat16), _dev(_tokens(rng, N, V))
    new = lambda: [torch.zeros(N, device="cuda") for _ in range(3)] + [torch.zeros(N, K, device="cuda"), torch.zeros(N, K, dtype=torch.int32, device="cuda")]
    out, eager = new(), new()
    err, eager_err, g = torch.zeros_like(x), torch.zeros_like(x), torch.randn(N, device="cuda")
    assert capi.logprob_scratch(N, V, K) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    capi.logprob_forward(x, t, *eager, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.logprob_forward(x, t, *out)
        capi.logprob_error_backward(x, t, g, g, *out[:3], err)
    for k in range(4):
        x.copy_(_logits(rng, N, V, torch.bfloat16))
        g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        capi.logprob_forward(x, t, *eager)
        capi.logprob_error_backward(x, t, g, g, *eager[:3], eager_err)
        for a, b in zip(out + [err], eager + [eager_err]):
            assert torch.equal(a, b), k


def test_more_than_two_to_the_31_logits():
    # the last rows' addresses are beyond 32 bits
    capi = PC.pkg().capi
    N, V = 16400, 131072
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    x[N - 1, V - 3] = 9.0
    t = torch.full((N,), V - 3, dtype=torch.int32, device="cuda")
    logp, lse, ent = (torch.empty(N, device="cuda") for _ in range(3))
    top = torch.empty(N, 2, dtype=torch.int32, device="cuda")
    capi.logprob_forward(x, t, logp, lse, ent, top_tokens=top)
    assert top[N - 1].tolist() == [V - 3, 0] and top[N - 2].tolist() == [0, 1]
    R = S.Rows(S.f64(x[N - 1:]), 1.0)
    S.assert_close(S.f64(logp[N - 1:]), R.logp[:, V - 3], R.tol_logp[:, V - 3])
    g = torch.full((N,), 0.5, device="cuda")
    capi.logprob_error_backward(x, t, g, None, logp, lse, ent, x)
    want, tol = R.gradient(np.array([V - 3]), np.array([0.5]), np.zeros(1), False)
    S.assert_close(S.f64(x[N - 1:]), want, tol, torch.bfloat16)
