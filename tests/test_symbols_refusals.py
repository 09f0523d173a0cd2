"""What the operators over symbols refuse, before any device call: runs without a GPU."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from __graft_entry__ import load_package

P, Q = C.c_void_p(4096), C.c_void_p(1 << 40)  # some addresses: no refused call may touch them


def _refused(status, what):
    L = load_package().capi.lib()
    assert status == 1, status
    assert what in L.cnt_last_error().decode()


def test_embedding():
    L = load_package().capi.lib()
    f = L.cnt_embed_forward
    for bad, what in (((0, 4, 2), "sizes"), ((4, 0, 2), "sizes"), ((4, 4, -1), "sizes")):
        _refused(f(None, *bad, 0, P, 4, P, 1.0, 0, P, 4), what)
    _refused(f(None, 4, 4, 2, 3, P, 4, P, 1.0, 0, P, 4), "element type")
    _refused(f(None, 4, 4, 2, 0, P, 4, P, 1.0, -1, P, 4), "element type")
    _refused(f(None, 4, 4, 2, 0, P, -4, P, 1.0, 0, P, 4), "stride")
    _refused(f(None, 4, 4, 2, 0, P, 4, P, 1.0, 0, P, 3), "overlap")
    _refused(f(None, 4, 4, 2, 0, None, 4, P, 1.0, 0, P, 4), "null")
    _refused(f(None, 4, 4, 2, 0, P, 4, None, 1.0, 0, P, 4), "null")
    _refused(f(None, 4, 4096, 1 << 26, 0, P, 4096, P, 1.0, 0, P, 4096), "too many")
    assert f(None, 4, 4, 0, 0, P, 4, None, 1.0, 0, None, 4) == 0
    assert L.cnt_embed_scratch(0, 4, 2) == -1 and L.cnt_embed_scratch(4, 4, -1) == -1 and L.cnt_embed_scratch(4, 4, 2 ** 31) == -1
    need = L.cnt_embed_scratch(100, 8, 50)
    b = lambda **k: [None, 100, 8, 50, P, 1.0, 0, P, 8, 0, P, 8, 0, P, need] if not k else None
    g = L.cnt_embed_backward

    def call(**changes):
        a = dict(zip("stream V D N tokens scale et err es gt grad gs acc scratch bytes".split(), b()))
        a.update(changes)
        return g(*a.values())

    for changes, what in (({"V": 0}, "sizes"), ({"N": -1}, "sizes"), ({"N": 2 ** 31}, "sizes"), ({"V": 2 ** 23 + 1}, "sizes"), ({"D": 2 ** 21 + 1}, "sizes"), ({"V": 2 ** 20, "D": 2 ** 14 + 1}, "sizes"), ({"N": 2 ** 20, "D": 2 ** 14 + 1}, "sizes"), ({"et": 7}, "element type"),
                          ({"gt": 7}, "element type"), ({"es": -1}, "stride"), ({"gs": 7}, "overlap"), ({"err": None}, "null"),
                          ({"grad": None}, "null"), ({"scratch": None}, "null"), ({"bytes": need - 1}, "scratch"),
                          ({"scratch": C.c_void_p(4100)}, "aligned")):
        _refused(call(**changes), what)


def test_embedding_scales():
    L = load_package().capi.lib()
    for scale in (float("inf"), float("nan")):
        _refused(L.cnt_embed_forward(None, 4, 4, 2, 0, P, 4, P, scale, 0, P, 4), "finite")
        _refused(L.cnt_embed_backward(None, 4, 4, 2, P, scale, 0, P, 4, 0, P, 4, 0, P, 2 ** 20), "finite")


@pytest.mark.parametrize("V,D", [(1, 1), (31, 8), (256, 64), (1000, 130), (5000, 64), (46356, 13), (1 << 20, 1), (577, 801), (33005, 1602), (3, 140000)])
def test_scratch_serves_fewer_slots(V, D):
    # a caller keeps what its longest fraction needs
    L = load_package().capi.lib()
    sizes = sorted({n + d for k in range(1, 21) for n in (1 << k, 3 << k, 64 * k * k, 512 * k, 4096 * k) for d in (-1, 0, 1)} | {0, 524288, 524289, 1 << 20})
    needs = [L.cnt_embed_scratch(V, D, n) for n in sizes if n * D <= 2 ** 33]
    assert needs == sorted(needs) and needs[0] >= 0


def test_scratch_of_shared_rows_is_bounded():
    L = load_package().capi.lib()
    for K in (0, 1, 2, 8, 31, 64):
        for V in (2049, 5000, 40000, 131072, 1000000, 1 << 30):
            assert all(0 <= L.cnt_logprob_scratch(n, V, K) <= (20 + 13 * K) * 1024 for n in range(0, 600))


def test_sizes_that_no_launch_takes():
    L = load_package().capi.lib()
    _refused(L.cnt_embed_forward(None, 4, 2 ** 30 + 1, 2, 0, P, 2 ** 31, P, 1.0, 0, P, 2 ** 31), "sizes")
    assert L.cnt_embed_scratch(2 ** 23, 2 ** 10, 2 ** 23) > 0
    for V, D, N in ((2 ** 23, 2 ** 10 + 1, 5), (5, 2 ** 10 + 1, 2 ** 23), (2 ** 12 + 1, 2 ** 21, 5)):
        assert L.cnt_embed_scratch(V, D, N) == -1
        _refused(L.cnt_embed_backward(None, V, D, N, P, 1.0, 0, P, D, 0, P, D, 0, P, 2 ** 40), "sizes")


def test_log_probabilities():
    L = load_package().capi.lib()

    def forward(**changes):
        a = dict(stream=None, N=4, V=10, type=0, logits=P, stride=10, scale=1.0, tokens=P, logp=P, lse=P, entropy=P, K=2, top=P, ids=P,
                 scratch=None, bytes=0)
        a.update(changes)
        return L.cnt_logprob_forward(*a.values())

    for changes, what in (({"N": -1}, "sizes"), ({"V": 0}, "sizes"), ({"V": 2 ** 31 - 1}, "sizes"), ({"N": 1 << 24}, "sizes"),
                          ({"type": 3}, "element type"), ({"stride": -1}, "stride"), ({"logits": None}, "null"), ({"scale": 0.0}, "scale"),
                          ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
                          ({"scale": 2e30}, "scale"), ({"scale": 0.5e-30}, "scale"),
                          ({"K": -1}, "alternatives"), ({"K": 65, "V": 100}, "alternatives"), ({"K": 11}, "alternatives"),
                          ({"top": None, "ids": None}, "alternatives"), ({"tokens": None}, "which tokens"),
                          ({"V": 100000, "stride": 100000}, "scratch")):
        _refused(forward(**changes), what)
    assert forward(N=0) == 0 and forward(N=0, V=100000, stride=100000) == 0

    def backward(**changes):
        a = dict(stream=None, N=4, V=10, type=0, logits=P, stride=10, scale=1.0, tokens=P, lse=P, entropy=P, g=P, h=P, err=Q, es=10)
        a.update(changes)
        return L.cnt_logprob_backward(*a.values())

    for changes, what in (({"V": 0}, "sizes"), ({"type": 9}, "element type"), ({"es": 9}, "overlap"), ({"lse": None}, "null"),
                          ({"err": None}, "null"), ({"entropy": None}, "entropies"), ({"tokens": None}, "which tokens"), ({"scale": 0.0}, "scale"),
                          ({"err": P, "es": 11}, "in their places"), ({"err": C.c_void_p(4096 + 159)}, "in their places"),
                          ({"err": C.c_void_p(4096 - 156)}, "in their places"), ({"err": P, "stride": 0}, "in their places")):
        _refused(backward(**changes), what)
    assert backward(N=0) == 0

    def both(**changes):
        a = dict(stream=None, N=4, V=10, type=0, logits=P, stride=10, scale=1.0, tokens=P, g=P, h=P, logp=P, lse=P, entropy=P, err=Q, es=10,
                 scratch=None, bytes=0)
        a.update(changes)
        return L.cnt_logprob_error_backward(*a.values())

    for changes, what in (({"V": 0}, "sizes"), ({"es": 9}, "overlap"), ({"lse": None}, "null"), ({"entropy": None}, "null"),
                          ({"err": P, "es": 12}, "in their places"), ({"err": C.c_void_p(4100)}, "in their places"),
                          ({"tokens": None}, "which tokens"), ({"V": 100000, "stride": 100000, "es": 100000}, "scratch")):
        _refused(both(**changes), what)
    assert both(N=0, V=100000, stride=100000, es=100000) == 0 and L.cnt_logprob_scratch(0, 100000, 3) == 0
    assert L.cnt_logprob_scratch(-1, 10, 0) == -1 and L.cnt_logprob_scratch(1, 0, 0) == -1 and L.cnt_logprob_scratch(1, 10, 65) == -1


def test_gradients():
    L = load_package().capi.lib()
    h = C.c_void_p()
    ptrs, sizes, types = (C.c_void_p * 1)(4096), (C.c_long * 1)(5), (C.c_int * 1)(0)
    _refused(L.cnt_gradients_create(1, ptrs, None, sizes, types, None), "null")
    _refused(L.cnt_gradients_create(-1, ptrs, None, sizes, types, C.byref(h)), "bad argument")
    _refused(L.cnt_gradients_create(1, None, None, sizes, types, C.byref(h)), "bad argument")
    _refused(L.cnt_gradients_create(1, ptrs, None, sizes, (C.c_int * 1)(4), C.byref(h)), "element type")
    _refused(L.cnt_gradients_create(1, ptrs, None, (C.c_long * 1)(-5), types, C.byref(h)), "negative")
    _refused(L.cnt_gradients_create(1, (C.c_void_p * 1)(None), None, sizes, types, C.byref(h)), "null pointer")
    _refused(L.cnt_gradients_create(1, ptrs, (C.c_void_p * 1)(None), sizes, types, C.byref(h)), "null pointer")
    _refused(L.cnt_gradients_create(1, (C.c_void_p * 1)(4098), None, sizes, types, C.byref(h)), "aligned")
    _refused(L.cnt_gradients_create(1, ptrs, None, (C.c_long * 1)(2 ** 62), types, C.byref(h)), "too many")
    # a tensor twice, or a stretch of another, where it is written
    two, sizes2, types2 = (C.c_void_p * 2), (C.c_long * 2)(5, 5), (C.c_int * 2)(0, 0)
    for grads, clipped in (((4096, 4096), None), ((4096, 4112), None), ((4096, 8192), (16384, 16384)), ((4096, 8192), (16384, 4096)),
                           ((4096, 8192), (4100, 16384)), ((4096, 8192), (16384, 8188))):
        _refused(L.cnt_gradients_create(2, two(*grads), two(*clipped) if clipped else None, sizes2, types2, C.byref(h)), "overlap")
    assert not h
    assert L.cnt_gradients_destroy(None) == 0
    _refused(L.cnt_opt_grad_norm(None, None, 1.0, P), "null")
    _refused(L.cnt_opt_clip(None, None, 1.0, P), "null")
    _refused(L.cnt_opt_step_clipped(None, 0, 4, P, P, P, None, P, None, 1.0, 0.0, 0.0, 0.1, 0.0, None), "null")
    _refused(L.cnt_network_update_clipped(None, None, 0, 0.1, 0.0, 1.0, 1.0, P), "null")


def test_the_binding_checks_tensors():
    capi = load_package().capi
    w, t, out = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="is on cpu"):
        capi.embed_forward(w, t, out)
    with pytest.raises(ValueError, match="is on cpu"):
        capi.logprob_forward(w, lse=torch.zeros(4))
    with pytest.raises(ValueError, match="is on cpu"):
        capi.GradientSet([w])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        capi._element("x", w.double())
    with pytest.raises(ValueError, match="out of range"):
        capi.embed_scratch(0, 1, 1)
    with pytest.raises(ValueError, match="out of range"):
        capi.logprob_scratch(1, 10, 65)


@pytest.mark.gpu
def test_the_binding_checks_tensors_on_the_device():
    capi = load_package().capi
    c = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    w, t, out = c(4, 3), c(2, dtype=torch.int32), c(2, 3)
    for args, what in (((w, t.long(), out), "int32"), ((w, t, c(3, 3)), "2 x 3"), ((w, t, c(3, 2).T), "contiguous"), ((w.double(), t, out), "float32"),
                       ((w, t.cpu(), out), "is on cpu"), ((w, c(4, dtype=torch.int32)[::2], out), "contiguous")):
        with pytest.raises(ValueError, match=what):
            capi.embed_forward(*args)
    with pytest.raises(RuntimeError, match="overlap"):
        capi.embed_forward(w, t, c(1, 3).expand(2, 3))
    with pytest.raises(ValueError, match="logits' type"):
        capi.logprob_backward(out, t, c(2), c(2), c(2), c(2), out.bfloat16())
    with pytest.raises(ValueError, match="row of alternatives"):
        capi.logprob_forward(out, top_logp=c(2, 2), top_tokens=c(2, 3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="alternatives"):
        capi.logprob_forward(out, top_logp=c(2, 4))
    with pytest.raises(ValueError, match="contiguous"):
        capi.GradientSet([c(4, 4).T])
    with pytest.raises(ValueError, match="places"):
        capi.GradientSet([w], [])
    gset = capi.GradientSet([w])
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(RuntimeError, match="positive"):
            capi.opt_clip(gset, bad, c(2))
    with pytest.raises(ValueError, match="2 contiguous values"):
        capi.opt_clip(gset, 1.0, c(3))


class _Elsewhere:
    """what a call looks at of a tensor on a GPU, and nothing behind it"""

    def __init__(self, count):
        self.dtype, self.shape, self.count = torch.float32, (count,), count

    def get_device(self):
        return 0

    def numel(self):
        return self.count

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


def test_clipped_steps_run_where_their_tensors_are():
    # as the other calls with the norm's result: a stream of another device is refused
    capi = load_package().capi
    stream = SimpleNamespace(device_index=1, device="cuda:1", cuda_stream=0)
    none, two = _Elsewhere(0), _Elsewhere(2)
    with pytest.raises(ValueError, match="stream"):
        capi.opt_step_clipped(0, none, none, none, none, none, None, 1.0, 0.0, 0.0, 0.1, 0.0, two, stream=stream)
    net = capi.Network.__new__(capi.Network)
    net.handle, net.loss = capi.VP(), _Elsewhere(1)
    with pytest.raises(ValueError, match="stream"):
        net.update_clipped(0, 0.1, 0.0, 1.0, 1.0, two, stream=stream)


@pytest.mark.parametrize("code,size", [(0, 4), (1, 2), (2, 2)])
def test_rows_that_no_launch_has_threads_for(code, size):
    # (no refused call may touch the addresses; in the logits' place, as rows of this number leave no room for others)
    L = load_package().capi.lib()
    for V, N in ((32641 // size + 1, 1 << 23), (65409 // size + 1, 1 << 22), (131072, 1 << 22)):
        _refused(L.cnt_logprob_error_backward(None, N, V, code, P, V, 1.0, P, P, P, P, P, P, P, V, None, 0), "too many rows")
