"""What the 4-bit decode makes of small value scales beside dominant tokens, of
value groups of unequal size, and of scores far from zero, against float64 from
the values held.

Bound.  With weights p (float64, sum 1) over tokens, the kernel forms P s in
FP32 relative to a reference and rounds it once to FP16: by 2^-11 of it, or by
half a subnormal step, 2^-25.  The reference is raised to where the largest P of a
pair of pages and their largest value scale s would give 2^12 to 2^13, never
further, so that half a step is at most 2^-37 max(p) max(s).  An output dim is the
sum of (z - 8) times these:
  2^-11 sum p |z - 8| s + 2^-37 max(p) max(s) sum |z - 8|.
The FP32 accumulators hold sum P s (z_d + 16 z_(d+1)) <= 255 sum P s, whose
difference by 16 gives z_(d+1), and sum P s, which counts 8 times; a warp adds at
most 32 pages to each, 2^-23 off at a time (tensor-core accumulators may cut the
rest off), in all
  32 * 2^-23 * (2 * 255 / 16 + 8) sum p s.
A score's FP32 sums (at most 2^5 roundings of partial sums that do not pass
S = scale sum |q| (|z - 8| s + |m|)) move p by the relative e = 2^-19 S; ex2 and
the joins of partial states add 2^-18.  The result is rounded once to the
output type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int4_cases import Held
from oracle import int4_oracle as I

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# An output that is all one token's has a code part of zero where that token's code is
# 8: |x - m| < s / 2.  32 normal values span 4.1 deviations, so s = 0.275 of one, and
# at most erf(0.275 / 2 / sqrt(2)) = 11 % of the dims have it (a midpoint off the middle
# has fewer).  The same again is four standard errors of 128 dims.
MIDDLES = 0.78


def check(a, scale=128 ** -0.5):
    """Bounds of every output; the share of outputs that zeros, or the midpoints
    alone, would put outside them."""
    got, gl = a.run()
    q = a.q[0].double().cpu().numpy()
    group = q.shape[0] // a.hkv
    eps = torch.finfo(a.q.dtype).eps / 2
    tiny = torch.finfo(a.q.dtype).tiny * eps
    zeros, middles = [], []
    for h in range(a.hkv):
        ka, km, va, vm = a.held(h)
        heads = slice(h * group, (h + 1) * group)
        exp, el, p = I.attention(q[heads], ka + km, va + vm, scale)
        size = scale * (np.abs(q[heads]) @ (np.abs(ka) + np.abs(km)).T).max(-1)
        e = (2.0 ** -19 * size + 2.0 ** -18)[:, None]
        s = a.value_scales(h)
        with np.errstate(invalid="ignore"):
            codes = np.where(s > 0, np.abs(va) / s, 8.0).sum(0)
        # (1 + 2^-10: the logarithm and the sums behind the reference)
        floor = 2.0 ** -37 * (1 + 2.0 ** -10) * p.max(-1, keepdims=True) * s.max() * codes
        floor = floor + 2.0 ** -18 * (2 * 255 / 16 + 8) * (p @ s)
        bound = 2.0 ** -11 * (p @ np.abs(va)) + floor + 2 * e * (p @ (np.abs(va) + np.abs(vm)))
        bound = bound + eps * (np.abs(exp) + bound) + tiny + 2.0 ** -23 * np.abs(exp)
        err = np.abs(got[heads] - exp)
        assert (err <= bound).all(), (h, float((err / bound).max()))
        lse_bound = 1.45 * (e[:, 0] + 2.0 ** -20) + 2.0 ** -22 * np.abs(el)
        assert (np.abs(gl[heads] - el) <= lse_bound).all(), h
        zeros.append((np.abs(exp) > bound).mean())
        middles.append((np.abs(p @ va) > bound).mean())
    return min(zeros), min(middles)


def rows(n, hq, hkv, v_std, boost, at, dtype, seed):
    """Scores of deviation about 1.2 nats; token `at` (if any) `boost` nats above
    the rest's largest, by a key along the queries' common direction."""
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(1, 1, 128, generator=g)
    q = base + 0.7 * torch.randn(1, hq, 128, generator=g)
    k = torch.randn(n, hkv, 128, generator=g)
    v = torch.randn(n, hkv, 128, generator=g) * v_std
    if at is not None:
        want = 1.2 * 4.3 + boost  # nats, for the common direction
        k[at] = base[0] * (want * 128 ** 0.5 / float((base * base).sum()))
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [4, 8])
@pytest.mark.parametrize("n,v_std,boost,at", [
    (49152, 0.02, 8.0, 0), (49152, 1e-3, 4.0, 30001), (49152, 5e-3, 8.0, 7), (4099, 1e-3, 8.0, 4098),
    (4099, 0.02, 12.0, 100), (700, 1e-3, 4.0, 0), (20000, 1e-3, 0.0, None), (20000, 1.0, 10.0, 5)])
def test_small_values_beside_a_dominant_token(cuda_lib, n, v_std, boost, at, group, dtype):
    q, k, v = rows(n, 2 * group, 2, v_std, boost, at, dtype, seed=n + int(boost))
    zeros, middles = check(Held(q, k, v, 2, 1))
    assert zeros > 0.9 and middles > MIDDLES


@pytest.mark.parametrize("small", [1e-4, 0.0])
@pytest.mark.parametrize("boost", [8.0, 14.0])
def test_a_dominant_token_of_small_values(cuda_lib, boost, small):
    """An attention sink: most of the weight on a token that adds next to nothing,
    so that the output is the others'."""
    n = 8200
    q, k, v = rows(n, 4, 1, 0.3, boost, 3, F16, seed=11)
    v[3] *= small
    zeros, middles = check(Held(q, k, v, 1, 2))
    assert zeros > 0.9 and middles > MIDDLES


@pytest.mark.parametrize("group", [3, 6])
def test_value_groups_of_unequal_size(cuda_lib, group):
    """A group of dims 2^10 below the token's largest keeps the bound of its own
    weights."""
    q, k, v = rows(6000, group, 1, 1.0, 6.0, 50, F16, seed=5)
    v[:, :, 32:64] *= 2.0 ** -10
    v[:, :, 96:] *= 2.0 ** -5
    zeros, middles = check(Held(q, k, v, 1, 3))
    assert zeros > 0.9 and middles > MIDDLES


@pytest.mark.parametrize("v_std", [1.0, 1e-3, 1e4])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_change_size_along_the_context(cuda_lib, v_std, dtype):
    """Scales that rise, and that fall, by 2^12 along the tokens of one request."""
    for falling in (False, True):
        q, k, v = rows(5000, 4, 1, 1.0, 0.0, None, dtype, seed=9)
        ramp = torch.logspace(-3.6, 0, 5000)[:, None, None] * v_std
        v = (v.float() * (ramp.flip(0) if falling else ramp)).to(dtype)
        zeros, middles = check(Held(q, k, v, 1, 4))
        assert zeros > 0.9 and middles > MIDDLES


def test_repeats_itself(cuda_lib):
    """The same bits from every run of one plan (many items, joined partial
    states, other work in between)."""
    for group, n in ((4, 49152), (8, 9000)):
        q, k, v = rows(n, 2 * group, 2, 1.0, 4.0, 17, F16, seed=6)
        a = Held(q, k, v, 2, 5)
        first = a.wrapper.run(a.q, a.pool, return_lse=True)
        for i in range(20):
            if i % 3 == 0:
                torch.randn(1 << 20, device="cuda").sum()
            again = a.wrapper.run(a.q, a.pool, return_lse=True)
            assert all(torch.equal(x, y) for x, y in zip(first, again)), i
