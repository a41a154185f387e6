"""The 4-bit decode of scores far from zero: FP32 sums of that size have steps of
many units, so a softmax is all on the largest score wherever the others are
steps away.

With q = +-big and keys c_t times the query's signs, the scores are 128 big c_t
scale, and the closest two differ by a tenth of the largest or more, which is
far beyond the relative 2^-16 that rounded sums (2^5 roundings, keys held to
FP16 scales) can move a score.  So the output is the top token's value held, within
the FP16 rounding of its weight (2^-11 of |z - 8| s) and the output's."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from int4_cases import Held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("big,key", [(60000.0, 60000.0), (60000.0, 900.0), (3000.0, 3000.0),
                                     (500.0, 37.0), (60000.0, 5.0)])
@pytest.mark.parametrize("group", [2, 7])
def test_scores_far_from_zero(cuda_lib, group, big, key, sign, dtype):
    g = torch.Generator().manual_seed(int(big) + int(key))
    n = 9
    signs = torch.randint(0, 2, (128,), generator=g) * 2.0 - 1.0
    # The top token is the sixth; with sign -1 every score is negative.
    c = torch.tensor([0.5, 0.3, 0.2, 0.4, 0.1, 1.0, 0.6, 0.05, 0.7]) if sign > 0 else \
        torch.tensor([-0.5, -0.6, -0.7, -0.4, -0.8, -0.1, -0.9, -0.95, -0.3])
    q = (signs * big).expand(1, group, 128).to(dtype)
    k = (c[:, None] * signs * key)[:, None].to(dtype)
    v = (torch.randn(n, 1, 128, generator=g) * torch.logspace(-3, 3, n)[:, None, None]).to(dtype)
    a = Held(q.contiguous(), k, v, 1, 1)
    got, lse = a.run()
    ka, km, va, vm = a.held(0)
    score = (a.q[0].double().cpu().numpy() @ (ka + km).T) * 128 ** -0.5
    assert (score.argmax(-1) == 5).all()
    rest = np.sort(score, -1)[:, ::-1]
    assert (rest[:, 0] - rest[:, 1] > 0.09 * np.abs(rest).max(-1)).all()
    eps = torch.finfo(dtype).eps / 2
    exp = va[5] + vm[5]
    bound = 2.0 ** -11 * np.abs(va[5]) + 2.0 ** -18 * (np.abs(va[5]) + np.abs(vm[5]))
    bound = bound + eps * (np.abs(exp) + bound) + torch.finfo(dtype).tiny * eps
    assert (np.abs(got - exp) <= bound).all()
    el = rest[:, 0] / math.log(2)
    assert (np.abs(lse - el) <= 2.0 ** -16 * np.abs(score).max(-1) / math.log(2)).all()


@pytest.mark.parametrize("exponent", [40, 80, 110, 114])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_queries_of_bfloat16_size(cuda_lib, exponent, sign):
    """Queries past FP16's range up to the documented 2^115: the same one-token
    softmax, and a base-2 LSE of the top score."""
    g = torch.Generator().manual_seed(exponent)
    signs = torch.randint(0, 2, (128,), generator=g) * 2.0 - 1.0
    c = torch.tensor([0.5, 1.0, 0.75]) if sign > 0 else torch.tensor([-0.5, -0.1, -0.75])
    q = (signs * 2.0 ** exponent).expand(1, 4, 128).to(torch.bfloat16)
    k = (c[:, None] * signs)[:, None].to(torch.bfloat16)
    v = torch.randn(3, 1, 128, generator=g).to(torch.bfloat16)
    a = Held(q.contiguous(), k, v, 1, 1)
    got, lse = a.run()
    ka, km, va, vm = a.held(0)
    score = (a.q[0].double().cpu().numpy() @ (ka + km).T) * 128 ** -0.5
    assert (score.argmax(-1) == 1).all()
    exp = va[1] + vm[1]
    bound = 2.0 ** -11 * np.abs(va[1]) + 2.0 ** -18 * (np.abs(va[1]) + np.abs(vm[1]))
    bound = bound + 2.0 ** -8 * (np.abs(exp) + bound)
    assert (np.abs(got - exp) <= bound).all()
    el = score.max(-1) / math.log(2)
    assert (np.abs(lse - el) <= 2.0 ** -16 * np.abs(score).max(-1) / math.log(2)).all()
