"""GPU parity of apply_rotary with the float64 oracle.

Bound per element: the result is rounded once (half a step of its type), and
before that each of the two products and their sum are rounded in FP32, so
the sum is off by at most 2 * 2^-24 (|a c| + |b s|) to first order (3 * is
used)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pagegauge_b200.rotary import RotaryScaling, apply_rotary, rotary_tables
from pagegauge_b200.runtime import read_device_error

pytestmark = pytest.mark.gpu


def rows(tokens, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g) * 2).to(dtype)


def check(got, x, cos, sin, interleaved=False, adjoint=False):
    x64, c, s = (t.double().cpu().numpy() for t in (x, cos, sin))
    exp = I.rotate(x64, c, s, interleaved, adjoint)
    size = I.rotate(np.abs(x64), np.abs(c), -np.abs(s), interleaved)  # |a c| + |b s| at a
    other = I.rotate(np.abs(x64), np.abs(c), np.abs(s), interleaved)  # and at b
    size = np.maximum(np.abs(size), np.abs(other))
    eps = torch.finfo(got.dtype).eps / 2
    tiny = float(torch.finfo(got.dtype).smallest_normal) * 2 * eps
    bound = eps * (np.abs(exp) + 1e-6 * size) + 3 * 2.0 ** -24 * size + tiny
    err = np.abs(got.double().cpu().numpy() - exp)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (128, 64), (80, 80), (80, 34), (64, 62),
                                            (256, 256), (6, 2), (96, 96), (31, 30), (128, 8)])
def test_layouts_and_parts_of_the_head(cuda_lib, dtype, interleaved, dim, rotary_dim):
    tokens, hq, hkv = 37, 5, 2
    q, k = rows(tokens, hq, dim, dtype, 1).cuda(), rows(tokens, hkv, dim, dtype, 2).cuda()
    cos, sin = rotary_tables(4096, rotary_dim, device="cuda")
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 4096, (tokens,), generator=g).int().cuda()
    for adjoint in (False, True):
        qo, ko = apply_rotary(q, k, cos, sin, pos, interleaved=interleaved, adjoint=adjoint)
        at = pos.long()
        check(qo, q, cos[at], sin[at], interleaved, adjoint)
        check(ko, k, cos[at], sin[at], interleaved, adjoint)
    assert read_device_error() == 0


@pytest.mark.parametrize("tokens", [0, 1, 2, 3, 129, 4097])
def test_token_counts(cuda_lib, tokens):
    q, k = rows(tokens, 8, 128, torch.float16, 4).cuda(), rows(tokens, 2, 128, torch.float16,
                                                               5).cuda()
    cos, sin = rotary_tables(70000, 128, scaling=RotaryScaling("parts", 8.0), device="cuda")
    pos = torch.arange(60000, 60000 + tokens, dtype=torch.int32, device="cuda")
    qo, ko = apply_rotary(q, k, cos, sin, pos)
    assert qo.shape == q.shape and ko.shape == k.shape
    if tokens:
        check(qo, q, cos[pos.long()], sin[pos.long()])
        check(ko, k, cos[pos.long()], sin[pos.long()])


@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary_dim", [
    (9473, 2, 1, 64, 26), (9473, 1, 1, 24, 24), (4740, 7, 2, 48, 44), (2369, 20, 4, 80, 34),
    (3, 3, 1, 4096, 4090), (2, 3, 1, 4096, 4096), (3, 2, 1, 1000, 998), (2, 2, 1, 2050, 2050),
    (1, 700, 300, 32, 30), (3, 40, 8, 256, 122), (1, 1, 0, 128, 58)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tiles_of_rows(cuda_lib, tokens, hq, hkv, dim, rotary_dim, interleaved, dtype):
    """Several tokens to a block, a part of a token's rows, rows and pairs
    wider than a block; in place as out of place."""
    q, k = rows(tokens, hq, dim, dtype, 14).cuda(), rows(tokens, hkv, dim, dtype, 15).cuda()
    cos, sin = rotary_tables(300, rotary_dim, device="cuda")
    pos = (torch.arange(tokens, dtype=torch.int32, device="cuda") * 7) % 300
    qo, ko = apply_rotary(q, k, cos, sin, pos, interleaved=interleaved)
    at = pos.long()
    check(qo, q, cos[at], sin[at], interleaved)
    check(ko, k, cos[at], sin[at], interleaved)
    apply_rotary(q, k, cos, sin, pos, interleaved=interleaved, query_out=q, key_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("dim,rotary_dim,dtype", [
    (128, 128, torch.float16), (128, 64, torch.bfloat16), (128, 128, torch.float32),
    (64, 32, torch.float32), (80, 80, torch.float16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_large_calls_equal_small_ones(cuda_lib, dim, rotary_dim, dtype, interleaved):
    """Much data at once, and the same tokens some hundred at a time, bit for
    bit; bad positions are left there too."""
    size = torch.finfo(dtype).bits // 8
    tokens = (105 << 20) // (2 * size * dim * 10) + 5
    g = torch.Generator(device="cuda").manual_seed(16)
    q = torch.randn(tokens, 8, dim, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, 2, dim, generator=g, device="cuda").to(dtype)
    cos, sin = rotary_tables(4096, rotary_dim, device="cuda")
    pos = torch.randint(0, 4096, (tokens,), generator=g, device="cuda").int()
    pos[5] = -1
    pos[tokens - 2] = 4096
    out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    apply_rotary(q, k, cos, sin, pos, interleaved=interleaved, query_out=out[0], key_out=out[1])
    assert read_device_error() == 2
    for t in out:
        assert (t[5] == 7).all() and (t[tokens - 2] == 7).all()
    pos[5] = pos[tokens - 2] = 0
    step = 397
    for t0 in range(0, tokens, step):
        some = slice(t0, t0 + step)
        a, b = apply_rotary(q[some], k[some], cos, sin, pos[some], interleaved=interleaved)
        for got, exp in ((out[0][some], a), (out[1][some], b)):
            for bad in (5, tokens - 2):
                if t0 <= bad < t0 + step:
                    exp[bad - t0] = 7.0
            assert torch.equal(got, exp)
    apply_rotary(q, k, cos, sin, pos, interleaved=interleaved, query_out=q, key_out=k)
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[5] = keep[tokens - 2] = False
    assert torch.equal(q[keep], out[0][keep]) and torch.equal(k[keep], out[1][keep])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_whole_heads_past_256_mb(cuda_lib, dtype):
    tokens = (257 << 20) // (2 * 2 * 128 * 13) + 3
    g = torch.Generator(device="cuda").manual_seed(17)
    q = torch.randn(tokens, 10, 128, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, 3, 128, generator=g, device="cuda").to(dtype)
    cos, sin = rotary_tables(4096, 128, device="cuda")
    pos = torch.randint(0, 4096, (tokens,), generator=g, device="cuda").int()
    for adjoint in (False, True):
        qo, ko = apply_rotary(q, k, cos, sin, pos, adjoint=adjoint)
        for t0 in range(0, tokens, 2999):
            some = slice(t0, t0 + 2999)
            a, b = apply_rotary(q[some], k[some], cos, sin, pos[some], adjoint=adjoint)
            assert torch.equal(qo[some], a) and torch.equal(ko[some], b)
    check(qo[-40:], q[-40:], cos[pos[-40:].long()], sin[pos[-40:].long()], adjoint=True)
    apply_rotary(q, k, cos, sin, pos, adjoint=True, query_out=q, key_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strided_views_in_place_and_out_of_place(cuda_lib, offset, interleaved, dtype):
    """Packed projection rows at odd offsets and strides; the dims and rows
    around the views stay as they were."""
    tokens, hq, hkv, dim = 19, 6, 2, 64
    width = (hq + 2 * hkv) * dim + 2 * offset
    flat = rows(tokens, 1, width, dtype, 6).cuda().view(tokens, width)
    body = flat[:, offset:offset + (hq + 2 * hkv) * dim].unflatten(1, (hq + 2 * hkv, dim))
    q, k = body[:, :hq], body[:, hq:hq + hkv]
    cos, sin = rotary_tables(64, 48, device="cuda")
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda").flip(0).contiguous()
    before = flat.clone()
    qo, ko = apply_rotary(q, k, cos, sin, pos, interleaved=interleaved)
    assert torch.equal(flat, before)
    at = pos.long()
    check(qo, q, cos[at], sin[at], interleaved)
    heads_first = torch.zeros(hkv, tokens, dim, dtype=dtype, device="cuda").transpose(0, 1)
    apply_rotary(q, k, cos, sin, pos, interleaved=interleaved, query_out=q, key_out=heads_first)
    assert torch.equal(q, qo) and torch.equal(heads_first, ko)
    assert torch.equal(flat[:, :offset], before[:, :offset])
    assert torch.equal(flat[:, offset + hq * dim:], before[:, offset + hq * dim:])


def test_query_alone_and_bad_positions_leave_rows(cuda_lib):
    q = rows(5, 3, 128, torch.float16, 7).cuda()
    cos, sin = rotary_tables(16, 128, device="cuda")
    pos = torch.tensor([3, -1, 15, 16, 0], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    got, none = apply_rotary(q, None, cos, sin, pos, query_out=out)
    assert none is None and got is out
    assert read_device_error() == 2
    assert (out[[1, 3]] == 7).all()
    keep = torch.tensor([0, 2, 4], device="cuda")
    check(out[keep], q[keep], cos[pos[keep].long()], sin[pos[keep].long()])


def test_adjoint_is_the_gradient(cuda_lib):
    """<R x, y> = <x, R^T y>, and central differences of <R x, y> in FP32."""
    x, y = rows(4, 2, 32, torch.float32, 8).cuda(), rows(4, 2, 32, torch.float32, 9).cuda()
    cos, sin = rotary_tables(128, 24, scaling=RotaryScaling("parts", 4.0), device="cuda")
    pos = torch.tensor([0, 5, 77, 127], dtype=torch.int32, device="cuda")
    for interleaved in (False, True):
        grad, _ = apply_rotary(y, None, cos, sin, pos, interleaved=interleaved, adjoint=True)
        f = lambda v: float((apply_rotary(v, None, cos, sin, pos,  # noqa: E731
                                          interleaved=interleaved)[0].double() * y).sum())
        for i in ((0, 0, 0), (2, 1, 13), (3, 0, 23), (3, 1, 24), (1, 1, 31)):
            up, down = x.clone(), x.clone()
            up[i] += 1.0
            down[i] -= 1.0
            # The map is linear; each f is off by FP32 rounding of 256 products.
            assert abs((f(up) - f(down)) / 2 - float(grad[i])) < 256 * 2.0 ** -22 * 40


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(cuda_lib, dtype, interleaved):
    """Autograd's gradients are the rotation's transpose applied to those of
    the outputs (one rounding, as a rotation's), for strided rows, expanded
    gradients, either input alone, and twice."""
    flat = rows(9, 7, 64, dtype, 20).cuda().requires_grad_()
    q, k = flat[:, :4], flat[:, 4:6]
    cos, sin = rotary_tables(64, 48, scaling=RotaryScaling("parts", 4.0), device="cuda")
    pos = torch.arange(5, 14, dtype=torch.int32, device="cuda")
    at = pos.long()
    qo, ko = apply_rotary(q, k, cos, sin, pos, interleaved=interleaved)
    check(qo.detach(), q.detach(), cos[at], sin[at], interleaved)
    check(ko.detach(), k.detach(), cos[at], sin[at], interleaved)
    gq, gk = rows(9, 4, 64, dtype, 21).cuda(), rows(9, 2, 64, dtype, 22).cuda()
    (grad,) = torch.autograd.grad((qo, ko), flat, (gq, gk), retain_graph=True)
    check(grad[:, :4], gq, cos[at], sin[at], interleaved, adjoint=True)
    check(grad[:, 4:6], gk, cos[at], sin[at], interleaved, adjoint=True)
    assert (grad[:, 6] == 0).all()
    # The sum's gradient is one expanded value; the key's output is unused.
    (grad,) = torch.autograd.grad(qo.sum(), flat, retain_graph=True)
    check(grad[:, :4], torch.ones_like(gq), cos[at], sin[at], interleaved, adjoint=True)
    assert (grad[:, 4:] == 0).all()
    (grad,) = torch.autograd.grad(ko, flat, gk)
    check(grad[:, 4:6], gk, cos[at], sin[at], interleaved, adjoint=True)
    # Only the key requires a gradient.
    leaf = k.detach().clone().requires_grad_()
    qo, ko = apply_rotary(q.detach(), leaf, cos, sin, pos, interleaved=interleaved)
    assert not qo.requires_grad and ko.requires_grad
    ko.backward(gk)
    check(leaf.grad, gk, cos[at], sin[at], interleaved, adjoint=True)
    # The gradient's gradient is the rotation again.
    leaf = q.detach().clone().requires_grad_()
    qo, none = apply_rotary(leaf, None, cos, sin, pos, interleaved=interleaved)
    assert none is None
    weight = gq.clone().requires_grad_()
    (grad,) = torch.autograd.grad(qo, leaf, weight, create_graph=True)
    (second,) = torch.autograd.grad(grad, weight, gq)
    check(second, gq, cos[at], sin[at], interleaved)


def test_gradients_of_rows_outside_the_tables_are_zero(cuda_lib):
    x = rows(4, 2, 64, torch.float32, 23).cuda().requires_grad_()
    cos, sin = rotary_tables(8, 64, device="cuda")
    pos = torch.tensor([1, -1, 7, 8], dtype=torch.int32, device="cuda")
    y, _ = apply_rotary(x, None, cos, sin, pos)
    (grad,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert read_device_error() == 2
    for t in (y, grad):
        assert (t[[1, 3]] == 0).all() and (t[[0, 2]] != 0).any()


def test_gradient_refusals_and_in_place_writes(cuda_lib):
    q = rows(4, 2, 64, torch.float16, 24).cuda()
    cos, sin = rotary_tables(8, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    leaf = q.clone().requires_grad_()
    for kw in (dict(query_out=torch.empty_like(q)), dict(query_out=leaf)):
        with pytest.raises(ValueError, match="new tensors"):
            apply_rotary(leaf, None, cos, sin, pos, **kw)
    with pytest.raises(ValueError, match="no gradient"):
        apply_rotary(leaf, None, cos.clone().requires_grad_(), sin, pos)
    with pytest.raises(ValueError, match="no gradient"):
        apply_rotary(q, None, cos.clone().requires_grad_(), sin, pos)
    with pytest.raises(ValueError, match="no gradient"):
        apply_rotary(q, None, cos, sin, pos, query_out=leaf)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pos.add_(1)
        with pytest.raises(ValueError, match="captured"):
            apply_rotary(leaf, None, cos, sin, pos)
    with torch.no_grad():
        out, _ = apply_rotary(leaf, None, cos, sin, pos)
    assert not out.requires_grad
    # What a graph saved and a rotation in place then changed is refused.
    hidden = q.float().requires_grad_() * 2
    loss = (hidden * hidden).sum()
    with torch.no_grad():
        apply_rotary(hidden, None, cos, sin, pos, query_out=hidden)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # Tables and positions that changed between forward and backward, too.
    y, _ = apply_rotary(leaf, None, cos, sin, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    with torch.inference_mode():
        x = q.clone()
        apply_rotary(x, None, cos, sin, pos, query_out=x)
    assert torch.equal(x, apply_rotary(q, None, cos, sin, pos)[0])


def test_capture_and_another_stream(cuda_lib):
    q, k = rows(33, 4, 128, torch.bfloat16, 10).cuda(), rows(33, 2, 128, torch.bfloat16,
                                                             11).cuda()
    cos, sin = rotary_tables(256, 128, device="cuda")
    pos = torch.arange(33, dtype=torch.int32, device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    exp = [t.clone() for t in apply_rotary(q, k, cos, sin, pos)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_rotary(q, k, cos, sin, pos, query_out=qo, key_out=ko)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(qo, exp[0]) and torch.equal(ko, exp[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_rotary(q, k, cos, sin, pos, query_out=qo, key_out=ko)
    pos += 100
    graph.replay()
    exp = apply_rotary(q, k, cos, sin, pos)
    assert torch.equal(qo, exp[0]) and torch.equal(ko, exp[1])


def test_refusals(cuda_lib):
    q, k = rows(4, 2, 64, torch.float16, 12).cuda(), rows(4, 1, 64, torch.float16, 13).cuda()
    cos, sin = rotary_tables(8, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    wide = rotary_tables(8, 128, device="cuda")
    for args, kw in (((q, k, *wide, pos), {}), ((q, k, cos.half(), sin.half(), pos), {}),
                     ((q, k, cos, sin[:4], pos), {}), ((q, k, cos, sin, pos.long()), {}),
                     ((q, k, cos, sin, pos[:3]), {}), ((q, k, cos, sin, pos.cpu()), {}),
                     ((q, k, cos.cpu(), sin.cpu(), pos), {}), ((q, k[:3], cos, sin, pos), {}),
                     ((q, k.bfloat16(), cos, sin, pos), {}),
                     ((q.transpose(1, 2), None, cos, sin, pos), {}),
                     ((q, None, cos, sin, pos), dict(key_out=k)),
                     ((q, k, cos, sin, pos), dict(query_out=q[:, :1].expand(4, 2, 64))),
                     ((q, k, cos, sin, pos), dict(query_out=torch.empty_like(q).float())),
                     ((q, k, cos, sin, pos), dict(key_out=torch.empty(4, 2, 64).cuda().half()))):
        with pytest.raises(ValueError):
            apply_rotary(*args, **kw)
    assert math.isfinite(float(q.float().sum()))


def test_a_backward_pass_is_not_captured(cuda_lib):
    """Forward and backward on one stream, the backward pass within a capture: refused
    before it reaches the leaves; the same pass then runs outside the capture."""
    cos, sin = rotary_tables(64, 128, device="cuda")
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    leaf = rows(5, 2, 128, torch.float32, 21).cuda().requires_grad_()
    weight = rows(5, 2, 128, torch.float32, 22).cuda()
    other = torch.zeros(4, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = apply_rotary(leaf, None, cos, sin, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.add_(1)
        with pytest.raises(ValueError, match="captured"):
            torch.autograd.grad(y, leaf, weight, retain_graph=True)
    with torch.cuda.stream(side):
        (grad,) = torch.autograd.grad(y, leaf, weight)
    torch.cuda.synchronize()
    exp, _ = apply_rotary(weight, None, cos, sin, pos, adjoint=True)
    assert torch.equal(grad, exp)
    graph.replay()
    assert (other == 1).all() and read_device_error() == 0


def test_forward_over_reverse_is_refused(cuda_lib):
    """A tangent on the gradient of a differentiable backward pass is not dropped."""
    import torch.autograd.forward_ad as forward

    cos, sin = rotary_tables(64, 128, device="cuda")
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    leaf = rows(5, 2, 128, torch.float32, 23).cuda().requires_grad_()
    weight = rows(5, 2, 128, torch.float32, 24).cuda()
    y, _ = apply_rotary(leaf, None, cos, sin, pos)
    with forward.dual_level():
        dual = forward.make_dual(weight, torch.ones_like(weight))
        for graph in (False, True):
            with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
                torch.autograd.grad(y, leaf, dual, create_graph=graph, retain_graph=True)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="forward-mode"):
                apply_rotary(dual, None, cos, sin, pos)
