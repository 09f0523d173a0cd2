"""Embedding lookup and its gradient by sorted tokens against 64 bits (through the C ABI)."""
import numpy as np
import pytest
import torch

import parity_cases as PC
import symbols as S

pytestmark = pytest.mark.gpu


def _tokens(rng, N, V, none=0.1):
    t = np.floor(np.exp(rng.random(N) * np.log(V + 1.0))).astype(np.int64) - 1
    t = np.clip(t, 0, V - 1)
    t[rng.random(N) < none] = -1
    return t.astype(np.int32)


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("out", S.TYPES)
@pytest.mark.parametrize("table", S.TYPES)
@pytest.mark.parametrize("V,D,N", [(1, 1, 1), (5, 7, 3), (256, 64, 130), (300, 8, 1000), (1000, 129, 33), (50, 2051, 9), (7, 4100, 2)])
def test_lookup(V, D, N, table, out):
    capi = PC.pkg().capi
    rng = np.random.default_rng(V + D)
    w, t = _dev(rng.standard_normal((V, D)), table), _tokens(rng, N, V)
    t[0] = V  # behind the table: no row either
    got = torch.full((N, D), 9.0, device="cuda", dtype=out)
    capi.embed_forward(w, _dev(t), got, scale=1.7)
    want = S.embed_rows(S.f64(w), t, float(np.float32(1.7)))
    S.assert_close(S.f64(got), want, S.U * np.abs(want), out)


def test_lookup_rows_anywhere_and_no_rows():
    capi = PC.pkg().capi
    rng = np.random.default_rng(1)
    for dtype in S.TYPES:
        wide, place = _dev(rng.standard_normal((40, 77)), dtype), torch.full((23, 90), 3.0, device="cuda", dtype=dtype)
        w, got, t = wide[:, 3:68], place[:, 5:70], _tokens(rng, 23, 40)
        capi.embed_forward(w, _dev(t), got)
        S.assert_close(S.f64(got), S.embed_rows(S.f64(w), t, 1.0), 0.0, dtype)
        assert torch.all(place[:, :5] == 3.0) and torch.all(place[:, 70:] == 3.0)
        capi.embed_forward(w, _dev(t[:0]), got[:0])
        one = wide[:1].expand(40, 77)  # one row for all tokens
        got = torch.empty(23, 77, device="cuda", dtype=dtype)
        capi.embed_forward(one, _dev(t), got)
        S.assert_close(S.f64(got), S.embed_rows(S.f64(one), t, 1.0), 0.0, dtype)


def _check_gradient(capi, V, D, t, err_type, grad_type, rng, accumulate=False, scale=0.37):
    N = len(t)
    e = _dev(rng.standard_normal((N, D)), err_type) if N else torch.empty(0, D, device="cuda", dtype=err_type)
    start = _dev(rng.standard_normal((V, D)), grad_type)
    grad, again = start.clone(), start.clone()
    capi.embed_backward(_dev(t), e, grad, scale=scale, accumulate=accumulate)
    capi.embed_backward(_dev(t), e, again, scale=scale, accumulate=accumulate)
    assert torch.equal(grad.view(torch.uint8), again.view(torch.uint8))  # one order, one result
    want, size, count = S.embed_grad(t, S.f64(e), V, float(np.float32(scale)))
    # n - 1 additions and the product with the scale, each off by u of a value that is at most the sum of the absolute ones
    tol = S.U * (count[:, None] + 1.0) * size
    if accumulate:
        want = want + S.f64(start)
        tol = tol + S.U * (np.abs(want) + tol)
        untouched = count == 0
        assert np.array_equal(S.f64(grad)[untouched], S.f64(start)[untouched])
    S.assert_close(S.f64(grad), want, tol, grad_type)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad", S.TYPES)
@pytest.mark.parametrize("err", S.TYPES)
@pytest.mark.parametrize("V,D,N", [(1, 1, 1), (3, 5, 64), (256, 64, 3000), (1000, 130, 700), (40, 1030, 301), (110000, 130, 1500)])
def test_gradient(V, D, N, err, grad, accumulate):
    rng = np.random.default_rng(V * 7 + D)
    _check_gradient(PC.pkg().capi, V, D, _tokens(rng, N, V), err, grad, rng, accumulate)


@pytest.mark.parametrize("V,D,N", [
    (1, 3, 1024), (1, 1, 1000), (2, 300, 1023), (9, 64, 1025), (50, 7, 513), (3000, 100, 1024), (100003, 33, 1000), (20000, 1030, 300), (5, 70, 49),
    (1, 3, 5000), (2, 4, 70001), (256, 8, 66000), (1024, 5, 9001), (1025, 5, 9001), (65536, 3, 5000), (65537, 3, 5000),
    (1 << 20, 1, 3000), ((1 << 20) + 1, 1, 3000), (700, 1, 600000), (5, 2, 0), (100003, 17, 1), (64, 513, 4097),
    (600, 300, 9000), (1024, 1030, 1500), (64, 515, 33000), (3, 140000, 1000), (16400, 2051, 512),
    (600, 1100, 16000), (1024, 1030, 17000), (1025, 1030, 17000), (65536, 37, 9001), (65537, 37, 9001), (1 << 20, 1, 21000), ((1 << 20) + 1, 1, 21000), (100003, 400, 600)])
def test_gradient_sizes(V, D, N):
    rng = np.random.default_rng(N + D)
    _check_gradient(PC.pkg().capi, V, D, _tokens(rng, N, V, 0.02), torch.float32, torch.float32, rng)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad", S.TYPES)
@pytest.mark.parametrize("err", [torch.float32, torch.float16])
@pytest.mark.parametrize("V,D,N", [
    (1, 1, 129), (1, 70, 512), (2, 3, 513), (7, 130, 511), (1000, 9, 1025), (1023, 5, 500), (1024, 33, 512), (1024, 1, 3001), (1025, 5, 512), (256, 64, 16001),
    (300, 1030, 200), (512, 8, 140000), (16, 4, 65537), (65, 300, 5000), (1025, 9, 400), (100003, 17, 512), (2047, 65, 3000), (40007, 6, 1500),
    (3001, 1, 60000)])
def test_gradient_by_slabs(V, D, N, err, grad, accumulate):
    rng = np.random.default_rng(V + N)
    _check_gradient(PC.pkg().capi, V, D, _tokens(rng, N, V, 0.02), err, grad, rng, accumulate)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad", S.TYPES)
@pytest.mark.parametrize("V,D,N", [(70001, 64, 5000), (90007, 257, 3000), (131072, 301, 40000), (8200, 520, 9000)])
def test_gradient_of_tables_that_are_filled_on_the_way(V, D, N, grad, accumulate):
    rng = np.random.default_rng(V)
    _check_gradient(PC.pkg().capi, V, D, _tokens(rng, N, V, 0.02), torch.bfloat16, grad, rng, accumulate)


@pytest.mark.parametrize("N,D", [(100, 33), (500, 33), (1000, 33), (2500, 33), (1000, 1400), (2500, 6800)])
@pytest.mark.parametrize("kind", ["none", "one", "last", "ascending", "descending", "outside"])
def test_gradient_orders_of_tokens(kind, N, D):
    rng = np.random.default_rng(3)
    V = 300
    t = {"none": np.full(N, -1), "one": np.full(N, 17), "last": np.full(N, V - 1), "ascending": np.sort(rng.integers(0, V, N)),
         "descending": -np.sort(-rng.integers(0, V, N)), "outside": rng.integers(-V, 3 * V, N)}[kind].astype(np.int32)
    t[:1] = -2 ** 31 if kind == "outside" else t[:1]
    _check_gradient(PC.pkg().capi, V, D, t, torch.bfloat16, torch.float32, rng)
    _check_gradient(PC.pkg().capi, V, D, t, torch.float32, torch.bfloat16, rng, True)


@pytest.mark.parametrize("V,N", [(50, 70), (50, 300), (50, 700), (7000, 700), (330000, 700)])
def test_gradient_rows_anywhere_and_broadcast_errors(V, N):
    capi = PC.pkg().capi
    rng = np.random.default_rng(8)
    D = 65
    t = _tokens(rng, N, V)
    for dtype in S.TYPES:
        wide, place = _dev(rng.standard_normal((N, 80)), dtype), torch.full((V, 71), 3.0, device="cuda")
        for e in (wide[:, 7:72], wide[3:4, 1:66].expand(N, D)):
            scratch = torch.full((capi.embed_scratch(V, D, N) + 512,), 0xAB, dtype=torch.uint8, device="cuda")
            capi.embed_backward(_dev(t), e, place[:, 1:66], scratch=scratch[:-512])
            want, size, count = S.embed_grad(t, S.f64(e), V, 1.0)
            S.assert_close(S.f64(place[:, 1:66]), want, S.U * (count[:, None] + 1.0) * size)
            assert torch.all(place[:, :1] == 3.0) and torch.all(place[:, 66:] == 3.0) and torch.all(scratch[-512:] == 0xAB)


@pytest.mark.parametrize("V,D", [(300, 40), (9000, 700)])
def test_scratch_of_the_longest_list_serves_the_others(V, D):
    capi = PC.pkg().capi
    rng = np.random.default_rng(6)
    e = _dev(rng.standard_normal((20000, D)).astype(np.float32))
    scratch = torch.full((capi.embed_scratch(V, D, 20000) + 512,), 0xAB, dtype=torch.uint8, device="cuda")
    for N in (20000, 9000, 3000, 600, 300, 100):
        t, grad = _tokens(rng, N, V), torch.empty(V, D, device="cuda")
        capi.embed_backward(_dev(t), e[:N], grad, scratch=scratch[:-512])
        want, size, count = S.embed_grad(t, S.f64(e[:N]), V, 1.0)
        S.assert_close(S.f64(grad), want, S.U * (count[:, None] + 1.0) * size)
        assert torch.all(scratch[-512:] == 0xAB)


def test_more_than_two_to_the_31_values():
    # rows whose addresses are beyond 32 bits
    capi = PC.pkg().capi
    V, D = 66000, 32800
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    t = torch.tensor([V - 1, 0, -1, V - 2, V - 1], dtype=torch.int32, device="cuda")
    rows = torch.randn(5, D, device="cuda").bfloat16()
    w[V - 1], w[0] = rows[0], rows[1]
    out = torch.empty(5, D, device="cuda")
    capi.embed_forward(w, t, out, scale=2.0)
    zero = torch.zeros_like(rows[0])
    assert torch.equal(out, 2 * torch.stack([rows[0], rows[1], zero, zero, rows[0]]).float())
    w.fill_(7.0)
    capi.embed_backward(t, rows, w)
    assert torch.equal(w[V - 1], (rows[0].float() + rows[4].float()).bfloat16()) and torch.equal(w[V - 2], rows[3]) and torch.equal(w[0], rows[1])
    w[V - 2:] = 0
    w[0] = 0
    assert not w.any()


def test_gradient_against_differences():
    # the loss sum(c * out) is linear in the table: its differences are exact up to the rounding of 64 bits
    capi = PC.pkg().capi
    rng = np.random.default_rng(4)
    V, D, N, scale = 9, 3, 40, 1.25
    t, c, w = _tokens(rng, N, V), rng.standard_normal((N, D)).astype(np.float32), rng.standard_normal((V, D))
    grad = torch.empty(V, D, device="cuda")
    capi.embed_backward(_dev(t), _dev(c), grad, scale=scale)
    want = np.zeros((V, D))
    for v in range(V):
        for d in range(D):
            up, down = w.copy(), w.copy()
            up[v, d] += 0.5
            down[v, d] -= 0.5
            want[v, d] = (c * (S.embed_rows(up, t, scale) - S.embed_rows(down, t, scale))).sum()
    _, size, count = S.embed_grad(t, c.astype(np.float64), V, scale)
    S.assert_close(S.f64(grad), want, S.U * (count[:, None] + 1.0) * size + 1e-12)


@pytest.mark.parametrize("V,N", [(500, 100), (500, 400), (500, 4000), (9000, 4000), (120000, 4000)])
def test_on_another_stream_and_replayed_from_a_graph(V, N):
    capi = PC.pkg().capi
    rng = np.random.default_rng(5)
    D = 48
    w, t, e = _dev(rng.standard_normal((V, D)).astype(np.float32)), _dev(_tokens(rng, N, V)), _dev(rng.standard_normal((N, D)).astype(np.float32))
    out, grad = torch.zeros(N, D, device="cuda"), torch.zeros(V, D, device="cuda")
    scratch = torch.empty(capi.embed_scratch(V, D, N), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    capi.embed_forward(w, t, out, stream=side)
    capi.embed_backward(t, out, grad, stream=side)  # (its scratch belongs to that stream)
    side.synchronize()
    first = grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.embed_forward(w, t, out)
        capi.embed_backward(t, e, grad, scratch=scratch)
    for k in range(4):
        e.copy_(torch.randn(N, D, device="cuda"))
        t.copy_(_dev(_tokens(rng, N, V)))
        out.zero_()
        grad.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        eager_out, eager = torch.empty_like(out), torch.empty_like(grad)
        capi.embed_forward(w, t, eager_out)
        capi.embed_backward(t, e, eager)
        assert torch.equal(out, eager_out) and torch.equal(grad, eager), k
    assert torch.isfinite(first).all()
