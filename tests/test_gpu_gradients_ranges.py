"""Norms at the end of what 32 bits hold, and what clipping makes of them (through the C ABI)."""
import numpy as np
import pytest
import torch

import parity_cases as PC
import symbols as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,value", [(4, 3e38), (100, 2e38), (5001, 3.3e38), (2 ** 20 + 3, 1e36)])
def test_a_norm_beyond_32_bits_counts_as_infinite(n, value, dtype):
    """The factor goes by the norm as it is reported: 0 where that is infinite."""
    capi = PC.pkg().capi
    g, other = torch.full((n,), value, device="cuda", dtype=dtype), torch.ones(70, device="cuda")
    places, result = [torch.full_like(g, 7.0), torch.full_like(other, 7.0)], torch.full((2,), 7.0, device="cuda")
    capi.opt_grad_norm(capi.GradientSet([g, other]), 1e30, result)
    assert result.tolist() == [float("inf"), 0.0]
    result.fill_(7.0)
    capi.opt_clip(capi.GradientSet([g, other], places), 1e30, result)
    assert result.tolist() == [float("inf"), 0.0]
    assert all(torch.all(p == 0) for p in places)


@pytest.mark.parametrize("limit", [1.0, 1e30])
@pytest.mark.parametrize("n,value", [(4, 1e38), (100, 3e37), (5001, 4e36)])
def test_the_largest_norms_of_32_bits(n, value, limit):
    capi = PC.pkg().capi
    g, result = torch.full((n,), value, device="cuda"), torch.zeros(2, device="cuda")
    norm = float(g[0].item()) * np.sqrt(n)
    before = S.f64(g)
    capi.opt_clip(capi.GradientSet([g]), limit, result)
    # the factor is rounded to 32 bits, by at most half of their smallest step, 2^-150, where it is below 2^-126
    S.assert_close(S.f64(result), [norm, limit / norm], [1e-12 * norm, 2.0 ** -150])
    S.assert_close(S.f64(g), before * (limit / norm), before * (2.0 ** -150 + S.U * limit / norm))


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 3.3e38])
def test_a_fraction_without_a_norm_is_a_gradient_of_zeros(bad):
    """Nothing of it comes to the weights; what earlier fractions have left in the momentum does."""
    capi = PC.pkg().capi
    n = 4099
    g, w, delta = torch.randn(n, device="cuda"), torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    g[5:9] = bad
    clip, cur = torch.zeros(2, device="cuda"), torch.zeros(n, device="cuda")
    capi.opt_grad_norm(capi.GradientSet([g]), 1.0, clip)
    for start in (torch.zeros_like(delta), delta):
        weights, deltas = w.clone(), start.clone()
        capi.opt_step_clipped(0, weights, g, cur, None, deltas, None, 1.0, 0.0, 0.0, 0.125, 0.5, clip)
        # products with 0.5 are exact: one rounding, that of the sum
        assert torch.equal(deltas, 0.5 * start) and torch.equal(weights, w + 0.5 * start)
