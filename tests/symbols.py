"""The operators over symbols in 64 bits, from their definitions, and how far fp32 evaluation may be off.  u: half a step of fp32 relative
to the value; a result in 16 bits is off by at most half a step of its own more, plus half its smallest step near zero."""
import numpy as np
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half of the smallest step; fp32 results below 2^-126 may be flushed to zero by the kernels' exp2
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def f64(t):
    return t.detach().cpu().double().numpy()


def embed_rows(table, tokens, scale):
    """table, tokens: numpy"""
    held = (tokens >= 0) & (tokens < len(table))
    return np.where(held[:, None], table[np.where(held, tokens, 0)] * scale, 0.0)


def embed_grad(tokens, err, V, scale):
    """(gradient, sums of absolute values, slots per row)"""
    held = (tokens >= 0) & (tokens < V)
    grad, size, count = np.zeros((V, err.shape[1])), np.zeros((V, err.shape[1])), np.zeros(V, int)
    np.add.at(grad, tokens[held], err[held])
    np.add.at(size, tokens[held], np.abs(err[held]))
    np.add.at(count, tokens[held], 1)
    return grad * scale, size * abs(scale), count


class Rows:
    """Log probabilities and their tolerances for logits x (numpy, 64 bits, exactly what the kernel reads)."""

    def __init__(self, x, scale):
        self.x, self.scale = x, scale
        N, V = x.shape
        with np.errstate(all="ignore"):
            self.m = x.max(1, initial=-np.inf)  # NaN where a row has one
            bad = np.isnan(x).any(1) | np.isposinf(x).any(1)
            empty = ~bad & np.isneginf(self.m)
            self.bad, self.empty = bad, empty
            d = np.where((bad | empty)[:, None], 0.0, scale * (x - np.where(bad | empty, 0.0, self.m)[:, None]))
            e = np.exp(d)
            s = e.sum(1)
            self.p = e / s[:, None]
            self.log_s = np.log(s)
            self.logp = d - self.log_s[:, None]
            d0 = np.where(self.p > 0, d, 0.0)
            self.entropy = self.log_s - (self.p * d0).sum(1)
            self.lse = scale * self.m + self.log_s
        self.lse[bad] = np.nan
        self.entropy[bad] = np.nan
        self.logp[bad] = np.nan
        self.lse[empty] = -np.inf
        self.entropy[empty] = 0.0
        self.logp[empty] = -np.inf
        self.p[empty] = 0.0
        # A lane adds up to 32 logits of a chunk and V / 256 over all chunks one after another; lanes, waves and parts are joined in up
        # to 14 steps, and the sums are brought to a new maximum at most once per join and chunk of 8192: a factor 2^shift whose error,
        # (3 ln 2 |shift| + 2) u, counts with the weight 2^-shift: below 4 u each.
        steps = 40 + V / 256.0 + 4 * (14 + V / 8192.0)
        a1 = (self.p * np.abs(d0)).sum(1)          # mean distance to the maximum
        a2 = (self.p * d0 * d0).sum(1)
        # t = (x - m) * (scale log2 e): three roundings, so 2^t is off by 3 u |d| + 2 u; 4 of each with those of second order
        self.tol_log_s = U * (4 * a1 + steps + 4 + 4 * np.abs(self.log_s))
        self.tol_entropy = self.tol_log_s + U * (4 * a2 + (a1 + 1) * (2 * steps + 12) + 4 * np.abs(self.entropy))
        with np.errstate(all="ignore"):
            self.tol_logp = self.tol_log_s[:, None] + U * 4 * (np.where(np.isfinite(d), np.abs(d), 0.0) + 1)
            self.tol_lse = self.tol_log_s + U * 2 * (np.abs(np.where(np.isfinite(self.m), self.m, 0.0) * scale) + np.abs(self.log_s) + 1)

    def top(self, K):
        order = np.empty((len(self.x), K), int)
        for n, row in enumerate(self.x):
            # (NaN last)
            order[n] = np.lexsort((np.arange(len(row)), -row, np.isnan(row)))[:K]
        return order

    def gradient(self, tokens, g, h, from_saved):
        """(errors of the logits, tolerance in 32 bits); from_saved: from lse and entropy rounded to fp32"""
        N, V = self.x.shape
        held = (tokens >= 0) & (tokens < V)
        gg = np.where(held, g, 0.0)[:, None]
        hh, H = h[:, None], np.where(self.bad, 0.0, self.entropy)[:, None]
        lp = np.where(self.p > 0, self.logp, 0.0)
        err = -gg * self.p - hh * self.p * (lp + H)
        given = np.zeros_like(err)
        rows = np.flatnonzero(held & ~self.empty)
        given[rows, tokens[rows]] = gg[rows, 0]
        lse_off = np.zeros(N)
        if from_saved:
            with np.errstate(all="ignore"):
                # lse is off by its own tolerance, and x * scale, the difference and the factor are rounded
                lse_off = self.tol_lse + U * 4 * (np.where(np.isfinite(self.lse), np.abs(self.lse), 0.0) + np.abs(np.where(np.isfinite(self.m), self.m, 0.0)) * self.scale)
        off_lp = self.tol_logp + lse_off[:, None] + U * 4
        tol = self.p * ((np.abs(gg) + np.abs(hh) * (np.abs(lp) + np.abs(H))) * (off_lp + 16 * U)
                        + np.abs(hh) * (off_lp + self.tol_entropy[:, None])) + 4 * U * np.abs(given)
        out = (err + given) * self.scale
        out[self.bad] = np.nan
        out[self.empty] = 0.0
        return out, tol * self.scale


def assert_close(got, want, tol, dtype=torch.float32):
    """|got - want| <= tol + what rounding to dtype adds; infinities and NaN in the same places"""
    got = np.asarray(got, np.float64)
    want = np.asarray(want, np.float64)
    tol = np.broadcast_to(tol, want.shape)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    ok = np.isfinite(want)
    d = np.abs(got[ok] - want[ok])
    limit = tol[ok] + HALF[dtype] * (np.abs(want[ok]) + tol[ok]) + TINY[dtype]
    worst = np.max(d / limit, initial=0.0)
    assert worst <= 1.0, "%.3g of what is allowed" % worst
