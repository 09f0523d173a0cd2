"""Log probabilities and their gradients at the ends of what calls may ask for, in every form that a row's length and the number of rows choose:
masks between ordinary logits and the type's lowest value, scales far from 1, rows far from zero.  Against 64 bits (through the C ABI)."""
import numpy as np
import pytest
import torch

import parity_cases as PC
import symbols as S

pytestmark = pytest.mark.gpu

ROWS = 6
# a V for each form: 16 lanes, a wave, a workgroup of growing size, shared or read twice (the last two: by the number of rows and their type)
LENGTHS = [300, 1500, 3000, 9001, 30001, 70001, 140001]
# a few rows, many
TIMES = [1, 88]


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _joint(x, tokens, g, h, scale, times):
    """Results of the joint call for `times` copies of the rows: those of the first, of a middle and of the last copy."""
    N, V = x.shape
    many = x.repeat(times, 1)
    f = [torch.full((N * times,), 7.0, device="cuda") for _ in range(3)]
    err = torch.full_like(many, 7.0)
    tile = lambda a: _dev(np.tile(a, times))
    PC.pkg().capi.logprob_error_backward(many, tile(tokens), tile(g), tile(h), *f, err, scale=scale)
    return [[t[N * k:N * k + N] for t in f + [err]] for k in sorted({0, times // 2, times - 1})]


def _check_joint(x, tokens, g, h, scale, times):
    scale = float(np.float32(scale))
    R = S.Rows(S.f64(x), scale)
    want, tol = R.gradient(tokens, g.astype(np.float64), h.astype(np.float64), False)
    # probabilities below 2^-126 may be flushed to zero: at most |log p| = 90 then, in front of which stand the scale and the errors
    tol = tol + S.TINY[torch.float32] * scale * (np.abs(g) + np.abs(h) * (90 + np.where(R.bad, 0.0, R.entropy)))[:, None]
    rows = np.arange(len(tokens))
    held = (tokens >= 0) & (tokens < x.shape[1])
    at = np.where(held, tokens, 0)
    with np.errstate(over="ignore"):
        lse = R.lse.astype(np.float32)  # infinite where 32 bits cannot hold it
    for logp, got_lse, entropy, err in _joint(x, tokens, g, h, scale, times):
        S.assert_close(S.f64(err), want, tol, x.dtype)
        S.assert_close(S.f64(entropy), R.entropy, R.tol_entropy)
        S.assert_close(S.f64(logp), np.where(held, R.logp[rows, at], 0.0), np.where(held, R.tol_logp[rows, at], 0.0))
        S.assert_close(S.f64(got_lse), lse, R.tol_lse)


# scale, value of the mask, error of the entropies
VANISHING = [(1.0, -1e33, 1e6), (1.0, -1e36, 65536.0), (1.0, -1e37, 100.0), (1.0, -5e37, 7.0), (1.0, -7e37, 1e4), (1e19, -1e18, 10.0), (1e20, -30.0, 1.0),
             (1e30, -30.0, 1e4)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,times", [(V, times) for V in LENGTHS for times in TIMES] + [(3000, 350)])
def test_gradient_where_probabilities_vanish(V, times, dtype):
    """A probability of 0 makes an error of 0, however large the logarithm and what stands in front of it."""
    rng = np.random.default_rng(V)
    x = rng.standard_normal((ROWS, V)) * 2.5
    masked = rng.random((ROWS, V)) < 0.1
    masked[:, 7] = False
    masked[2] = np.arange(V) != 7      # one token left
    masked[3] = np.arange(V) >= V // 2
    masked[4] = False
    masked[4, V - 5] = True            # one ruled out
    tokens = np.array([7, -1, 7, 3, V - 5, 9], np.int32)
    g = np.array([1.0, 1.0, -2.0, 0.0, 3.0, -1.0], np.float32)
    for scale, low, error in VANISHING:
        h = np.array([1.0, -1.0, 0.5, 1.0, -1.0, 1.0], np.float32) * np.float32(error)
        _check_joint(_dev(np.where(masked, low, x), dtype), tokens, g, h, scale, times)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("V", LENGTHS)
def test_gradient_of_rows_far_from_zero(V, times, dtype):
    """The joint call's probabilities come from the row's maximum: what 32 bits of the log sum cannot hold does not reach them."""
    rng = np.random.default_rng(V + 1)
    x = rng.standard_normal((ROWS, V)) * 2.5
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[0] = low
    x[1] += 1e4
    x[2] -= 1e4
    x[3] = low
    x[3, 5] = -3.0
    x[4] = high
    x[5] = low
    x[5, V // 3:V // 2] = -np.inf
    tokens = np.array([1, 2, V - 1, 5, -1, V - 2], np.int32)
    g, h = np.array([1.0, -1.0, 0.5, 1.0, 1.0, 2.0], np.float32), np.array([0.5, 1.0, -1.0, 0.0, 2.0, 0.5], np.float32)
    _check_joint(_dev(x, dtype), tokens, g, h, 1.0, times)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("V", LENGTHS)
def test_gradient_of_rows_whose_log_sum_is_beyond_32_bits(V, times, dtype):
    """A row is without choices if all of its logits are -inf, not if its log sum is -inf in 32 bits."""
    x = np.zeros((ROWS, V))
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[0] = low
    x[1] = low
    x[1, 4:V - 3] = -np.inf
    x[2] = high
    x[3] = -np.inf
    x[4] = low
    x[4, 7] = 0.5 * low
    tokens = np.array([1, 2, V - 1, 5, 7, 2], np.int32)
    g, h = np.array([1.0, -1.0, 0.5, 1.0, 2.0, 1.0], np.float32), np.array([0.5, 1.0, -1.0, 1.0, 2.0, 0.0], np.float32)
    for scale in (1.5, 64.0, 1e30):
        _check_joint(_dev(x, dtype), tokens, g, h, scale, times)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("scale", [1.0, 1e5, 1e20, 1e30])
@pytest.mark.parametrize("V", [3, 300, 1500, 3000, 70001])
def test_gradient_from_a_log_sum_that_is_off_stays_within_bounds(V, scale, dtype):
    """A probability from a log sum in 32 bits is off by a factor exp(|lse| 2^-24), but none is above 1: with |log p| <= 1000 in front of one of
    at least 2^-126, p |log p| <= 1 / e, an error is at most scale * (2 |g| + |h| (1 + H))."""
    rng = np.random.default_rng(V)
    N = 64
    x = _dev(rng.standard_normal((N, V)) * 30, dtype)
    x[5:9] = torch.finfo(dtype).min
    x[9] = torch.finfo(dtype).max
    g, h = rng.standard_normal(N).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    t = rng.integers(-1, V, N).astype(np.int32)
    lse, entropy = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    capi, err = PC.pkg().capi, torch.full_like(x, 7.0)
    capi.logprob_forward(x, lse=lse, entropy=entropy, scale=scale)
    capi.logprob_backward(x, _dev(t), lse, entropy, _dev(g), _dev(h), err, scale=scale)
    most = scale * (2 * np.abs(g) + np.abs(h) * (1 + S.f64(entropy)))
    top = torch.finfo(dtype).max
    got = S.f64(err)
    assert not np.isnan(got).any()
    assert np.all(np.abs(got) <= np.where(most < top, most * (1 + 4 * S.HALF[dtype]), np.inf)[:, None] + S.TINY[dtype])


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("V", LENGTHS)
def test_log_probabilities_of_rows_that_masks_leave_little_of(V, times, dtype):
    rng = np.random.default_rng(V + 2)
    x = rng.standard_normal((ROWS, V)) * 2.5
    low, K = torch.finfo(dtype).min, 6
    x[0] = low
    x[1] += 1e4
    x[2] = -np.inf
    x[2, V - 1] = 1.5
    x[3] = low
    x[3, 5] = -3.0
    x[4] = -np.inf
    x[5, 3:V - 1] = low
    x = _dev(x, dtype)
    tokens = np.array([1, 2, V - 1, 4, 3, 9], np.int32)
    out = {n: torch.full((ROWS * times,), 7.0, device="cuda") for n in ("logp", "lse", "entropy")}
    out["top_logp"] = torch.full((ROWS * times, K), 7.0, device="cuda")
    out["top_tokens"] = torch.full((ROWS * times, K), -7, dtype=torch.int32, device="cuda")
    PC.pkg().capi.logprob_forward(x.repeat(times, 1), _dev(np.tile(tokens, times)), **out)
    R, rows = S.Rows(S.f64(x), 1.0), np.arange(ROWS)
    want = R.top(K)
    for k in sorted({0, times // 2, times - 1}):
        part = {n: t[ROWS * k:ROWS * k + ROWS] for n, t in out.items()}
        assert np.array_equal(part["top_tokens"].cpu().numpy(), want)
        S.assert_close(S.f64(part["top_logp"]), R.logp[rows[:, None], want], R.tol_logp[rows[:, None], want])
        S.assert_close(S.f64(part["logp"]), R.logp[rows, tokens], R.tol_logp[rows, tokens])
        S.assert_close(S.f64(part["lse"]), R.lse, R.tol_lse)
        S.assert_close(S.f64(part["entropy"]), R.entropy, R.tol_entropy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_rows_on_two_streams_at_once(dtype):
    """What the three launches of a call hand on is in the call's own scratch memory."""
    capi, N, V = PC.pkg().capi, 5, 140001
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for k in range(2):
        x = (torch.randn(N, V, device="cuda") * 2.5 + 1e4 * k).to(dtype)
        x[3] = torch.finfo(dtype).min
        t = torch.randint(0, V, (N,), device="cuda", dtype=torch.int32)
        new = lambda: [torch.zeros(N, device="cuda") for _ in range(3)] + [torch.zeros_like(x)]
        sets.append((x, t, torch.randn(N, device="cuda"), torch.randn(N, device="cuda"), new(), new()))
    for x, t, g, h, alone, _ in sets:
        capi.logprob_error_backward(x, t, g, h, *alone)
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (x, t, g, h, _, out) in zip(streams, sets):
            capi.logprob_error_backward(x, t, g, h, *out, stream=stream)
    torch.cuda.synchronize()
    for _, _, _, _, alone, out in sets:
        assert all(torch.equal(a, b) for a, b in zip(alone, out))
