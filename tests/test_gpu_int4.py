"""GPU parity of the 4-bit cache: records bit for bit against the oracle's
FP32 steps, decode attention against float64 from the values held.

Attention bound.  With weights p (float64) over tokens, the kernel rounds
P * s to FP16 (2^-11 relative, and half a subnormal step 2^-25) before the
tensor-core products, so an output dim is off by at most
  2^-11 sum p |z - 8| s + 2^-25 sum |z - 8| / l,
l >= 1/4 the sum of the unnormalised weights (a weight of 1/4 is the least
the largest has).  A score's FP32 sums (at most 2^5 roundings of partial sums
that do not pass S = scale sum |q| (|z - 8| s + |m|)) move p by the relative
e = 2^-19 S; ex2 and the joins of partial states add 2^-18.  The result is
rounded once to the output type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pagegauge_b200 import _lib
from pagegauge_b200.int4 import Int4PagePool
from pagegauge_b200.rotary import RotaryScaling, rotary_tables
from pagegauge_b200.runtime import load_append_extension, read_device_error
from pagegauge_b200.wrapper import (BatchDecodeWithPagedKVCacheWrapper, Int4DecodeWrapper,
                                    make_int4_wrapper, merge_state_in_place, plan)

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def cpu(t):
    return t.detach().cpu().numpy() if t.dtype != BF16 else t.detach().float().cpu().numpy()


# ----------------------------------------------------------------- append
class Append:
    """One call's inputs (rows are views of a packed projection)."""

    def __init__(self, tokens, hq=4, hkv=2, dtype=F16, pairs=64, pages=None, seed=1, center=True,
                 pad=0, offset=0, scaling=None):
        g = torch.Generator().manual_seed(seed)
        width = (hq + 2 * hkv) * 128 + offset
        flat = torch.randn(tokens, width, generator=g) * 1.5 + 0.3
        flat = flat.to(dtype).cuda()
        body = flat[:, offset:].unflatten(1, (hq + 2 * hkv, 128))
        self.q, self.k, self.v = body[:, :hq], body[:, hq:hq + hkv], body[:, hq + hkv:]
        self.cos, self.sin = rotary_tables(5000, 2 * pairs, scaling=scaling, device="cuda")
        self.positions = torch.randint(0, 5000, (tokens,), generator=g).int().cuda()
        pages = pages or -(-tokens // 16) + 2
        slots = torch.randperm(pages * 16, generator=g)[:tokens].int()
        if pad:
            slots[torch.randperm(tokens, generator=g)[:pad]] = -1
        self.slots = slots.cuda()
        self.pool = Int4PagePool(pages, hkv)
        self.pool.records.copy_(torch.randint(0, 256, self.pool.records.shape, generator=g,
                                              dtype=torch.uint8))
        self.kw = {}
        if center:
            c = torch.randn(2, 3, hkv, 128, generator=g).to(dtype).cuda()
            rows = torch.randint(0, 3, (tokens,), generator=g).int().cuda()
            self.kw = dict(key_center=c[0], value_center=c[1], center_rows=rows)
        self.rotated = torch.full(self.q.shape, 9.0, dtype=dtype, device="cuda")

    def run(self, **kw):
        load_append_extension().rope_append_int4(
            self.q, self.k, self.v, self.cos, self.sin, self.positions, self.slots,
            kw.pop("rotated_query", self.rotated), self.pool.records, **self.kw, **kw)

    def expected(self, interleaved=False):
        """(rotated q, rotated k, records) by the oracle's FP32 steps."""
        at = self.positions.long()
        cos, sin = cpu(self.cos[at]), cpu(self.sin[at])
        f32 = lambda t: cpu(t.float())  # noqa: E731
        q = I.rotate(f32(self.q), cos, sin, interleaved, dtype=np.float32)
        k = I.rotate(f32(self.k), cos, sin, interleaved, dtype=np.float32)
        kk, vv = k, f32(self.v)
        if self.kw:
            rows = cpu(self.kw["center_rows"])
            kk = kk - f32(self.kw["key_center"])[rows]
            vv = vv - f32(self.kw["value_center"])[rows]
        records = cpu(self.pool.records).copy()
        kq, vq = I.quantise(kk), I.quantise(vv)
        for t, slot in enumerate(cpu(self.slots)):
            if slot < 0:
                continue
            for h in range(self.k.shape[1]):
                I.store_token(records, slot // 16, h, slot % 16, [x[t, h] for x in kq],
                              [x[t, h] for x in vq])
        return q, k, records


def same_rounded(got, exp):
    """Rows equal the FP32 values rounded once."""
    assert torch.equal(got.cpu(), torch.from_numpy(np.ascontiguousarray(exp)).to(got.dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pairs,offset", [(64, 0), (32, 0), (8, 8), (29, 0), (64, 3), (1, 0),
                                          (63, 8), (40, 0), (56, 0), (48, 8), (36, 0), (4, 0)])
def test_append_is_bit_exact(cuda_lib, dtype, interleaved, pairs, offset):
    a = Append(77, hq=5, hkv=3, dtype=dtype, pairs=pairs, pad=5, offset=offset)
    q, k, records = a.expected(interleaved)
    rotated_key = torch.full(a.k.shape, 9.0, dtype=dtype, device="cuda")
    a.run(interleaved=interleaved, rotated_key=rotated_key)
    keep = (a.slots >= 0).cpu()
    same_rounded(a.rotated[keep.cuda()], q[keep.numpy()])
    same_rounded(rotated_key[keep.cuda()], k[keep.numpy()])
    # rows of skipped tokens stay as they were
    assert (a.rotated[~keep.cuda()] == 9).all() and (rotated_key[~keep.cuda()] == 9).all()
    assert np.array_equal(cpu(a.pool.records), records)
    assert read_device_error() == 0


@pytest.mark.parametrize("tokens,hq,hkv", [(0, 4, 1), (1, 1, 1), (1, 32, 8), (35, 32, 8),
                                           (4097, 4, 1), (20000, 3, 1)])
def test_append_sizes(cuda_lib, tokens, hq, hkv):
    a = Append(tokens, hq=hq, hkv=hkv, center=tokens % 2 == 1, seed=tokens + 3,
               scaling=RotaryScaling("parts", 4.0))
    q, _, records = a.expected()
    a.run()
    same_rounded(a.rotated, q)
    assert np.array_equal(cpu(a.pool.records), records)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pairs,offset", [(29, 0), (32, 0), (16, 8), (47, 0), (64, 3), (45, 1)])
def test_append_many_tokens_of_partial_heads(cuda_lib, pairs, offset, interleaved):
    a = Append(1203, hq=5, hkv=3, dtype=BF16, pairs=pairs, pad=7, offset=offset, seed=pairs)
    q, k, records = a.expected(interleaved)
    a.run(interleaved=interleaved, rotated_key=a.k, rotated_query=a.q)
    keep = (a.slots >= 0).cpu()
    same_rounded(a.q[keep.cuda()], q[keep.numpy()])
    same_rounded(a.k[keep.cuda()], k[keep.numpy()])
    assert np.array_equal(cpu(a.pool.records), records)


def test_append_in_place_and_shared_center(cuda_lib):
    for offset in (0, 3):
        a = Append(50, hq=3, hkv=1, offset=offset)
        a.kw.pop("center_rows")
        a.kw["center_rows"] = torch.zeros(50, dtype=torch.int32, device="cuda")
        q, k, records = a.expected()
        a.kw["center_rows"] = None  # row 0 for every token
        a.run(rotated_query=a.q, rotated_key=a.k)
        same_rounded(a.q, q)
        same_rounded(a.k, k)
        assert np.array_equal(cpu(a.pool.records), records)


def test_append_far_pages_and_extreme_values(cuda_lib):
    """Record offsets past 2^31 bytes, values past FP16's range (held as its
    largest), subnormal and constant rows; a NaN stays in its group."""
    pages = 900_000  # 2.3 GB of records of one head
    a = Append(6, hq=1, hkv=1, dtype=BF16, pages=4, center=False)
    a.v[0], a.v[1], a.v[2] = 1e6, -3e38, 1e-7
    a.v[3, 0, ::2] = float("inf")
    a.v[4, 0, 40] = float("nan")
    a.slots = torch.tensor([16 * (pages - 1) + i for i in range(6)], dtype=torch.int32,
                           device="cuda")
    big = torch.zeros(pages, 1, 2560, dtype=torch.uint8, device="cuda")
    a.pool = Int4PagePool(pages, 1, records=big)
    a.run()
    key, value = a.pool.read(a.slots, dtype=torch.float32)
    v = value[:, 0].cpu().numpy()
    assert (v[0] == 65504).all() and (v[1] == -65504).all()
    assert np.abs(v[2] - float(a.v[2, 0, 0])).max() <= 2.0 ** -25
    assert (v[3, ::2] == 65504).all() or np.abs(v[3, ::2] - 65504).max() <= 65504 * 15 / 2 ** 11
    assert np.isnan(v[4, 32:64]).all() and np.isfinite(np.delete(v[4], range(32, 64))).all()
    assert torch.isfinite(key).all()
    assert not big[:pages - 1].any()
    assert read_device_error() == 0


def test_append_reports_bad_tokens_and_skips_them(cuda_lib):
    for field, value, code in (("slots", 16 * 100, 3), ("positions", 5000, 2),
                               ("positions", -1, 2), ("center_rows", 3, 3),
                               ("center_rows", -1, 3)):
        a = Append(9, seed=21)
        q, _, records = a.expected()
        target = a.kw[field] if field in a.kw else getattr(a, field)
        slot = int(a.slots[4])
        target[4] = value
        before = a.pool.records.clone()
        a.run()
        assert read_device_error() == code, field
        assert (a.rotated[4] == 9).all()
        got = a.pool.read(torch.tensor([slot], dtype=torch.int32, device="cuda"))
        a.pool.records, after = before, a.pool.records
        old = a.pool.read(torch.tensor([slot], dtype=torch.int32, device="cuda"))
        for x, y in zip(got, old):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
        keep = [0, 1, 2, 3, 5, 6, 7, 8]
        same_rounded(a.rotated[keep], q[keep])
        a.pool.records = torch.from_numpy(records).cuda()
        others = a.slots[keep]
        exp = a.pool.read(others)
        a.pool.records = after
        for x, y in zip(a.pool.read(others), exp):
            assert torch.equal(x, y)


@pytest.mark.parametrize("tokens,hq,hkv", [(4003, 1, 1), (4001, 7, 1), (3001, 6, 2), (5002, 2, 2),
                                           (3203, 5, 3), (2003, 7, 5), (1201, 8, 8)])
@pytest.mark.parametrize("pairs", [64, 29])
def test_append_and_read_of_many_tokens(cuda_lib, tokens, hq, hkv, pairs):
    """Rows of several tokens in one warp; skipped, refused and last tokens
    leave the others whole.  The read of many tokens is that of few."""
    a = Append(tokens, hq=hq, hkv=hkv, pairs=pairs, pad=9, seed=tokens)
    bad = torch.arange(3, tokens, 331)
    a.positions[bad[0::2].cuda()] = 5000
    a.kw["center_rows"][bad[1::2].cuda()] = -1
    stored = torch.ones(tokens, dtype=torch.bool)
    stored[bad] = False
    given, slots = a.slots, a.slots.clone()
    slots[bad.cuda()] = -1
    safe = a.positions.clamp(max=4999), a.kw["center_rows"].clamp(min=0)
    real = a.positions, a.kw["center_rows"]
    a.slots, a.positions, a.kw["center_rows"] = slots, *safe
    q, _, records = a.expected()
    a.slots, a.positions, a.kw["center_rows"] = given, *real
    a.run()
    assert read_device_error() in (2, 3)
    stored &= (given >= 0).cpu()
    same_rounded(a.rotated[stored.cuda()], q[stored.numpy()])
    assert (a.rotated[~stored.cuda()] == 9).all()
    assert np.array_equal(cpu(a.pool.records), records)
    slots[5] = 16 * a.pool.num_pages
    slots[stored.nonzero()[-1].item()] = -1
    key, value = a.pool.read(slots)
    assert read_device_error() == 3
    for t0 in range(0, tokens, 997):  # few rows each
        few = a.pool.read(slots[t0:t0 + 997])
        read_device_error()
        assert torch.equal(key[t0:t0 + 997], few[0]) and torch.equal(value[t0:t0 + 997], few[1])
    skipped = (slots < 0) | (slots >= 16 * a.pool.num_pages)
    assert (key[skipped] == 0).all() and (value[skipped] == 0).all()


def test_read_matches_the_records(cuda_lib):
    a = Append(40, hkv=3, pad=4)
    a.run()
    (ka, km), (va, vm) = I.load(cpu(a.pool.records))
    slots = a.slots.clone()
    slots[7] = 16 * a.pool.num_pages
    for dtype in (F16, BF16, torch.float32):
        key, value = a.pool.read(slots, dtype=dtype)
        assert read_device_error() == 3
        for got, (z, m) in ((key, (ka, km)), (value, (va, vm))):
            for t, slot in enumerate(cpu(slots)):
                if slot < 0 or slot >= 16 * a.pool.num_pages:
                    assert (got[t] == 0).all()
                    continue
                # (z - 8) s and the sum are rounded in FP32, then to the type
                exp = z[slot // 16, :, slot % 16] + m[slot // 16, :, slot % 16]
                size = np.abs(z[slot // 16, :, slot % 16]) + np.abs(m[slot // 16, :, slot % 16])
                eps = torch.finfo(dtype).eps / 2
                err = np.abs(got[t].double().cpu().numpy() - exp)
                assert (err <= eps * np.abs(exp) * 1.001 + 2.0 ** -23 * size + 2.0 ** -25).all()


def test_append_refusals(cuda_lib):
    a = Append(8)
    good = dict(q=a.q, k=a.k, v=a.v, cos=a.cos, sin=a.sin, pos=a.positions, slots=a.slots,
                rotated=a.rotated, records=a.pool.records)
    bad = [dict(q=a.q.float()), dict(k=a.k.bfloat16()), dict(v=a.v[:, :1]), dict(k=a.k[:7]),
           dict(cos=a.cos.half()), dict(pos=a.positions.long()), dict(slots=a.slots[:7]),
           dict(slots=a.slots.cpu()), dict(rotated=a.rotated[:, :3]),
           dict(rotated=a.rotated[:, :1].expand(a.q.shape)),
           dict(records=a.pool.records[:, :1]), dict(records=a.pool.records[..., :2559]),
           dict(records=a.pool.records.view(torch.int8)), dict(q=a.q.cpu()),
           dict(q=torch.empty(8, 4, 256, device="cuda", dtype=F16)[..., ::2])]
    ext = load_append_extension()
    for kw in bad:
        c = {**good, **kw}
        with pytest.raises((RuntimeError, ValueError)):
            ext.rope_append_int4(c["q"], c["k"], c["v"], c["cos"], c["sin"], c["pos"], c["slots"],
                                 c["rotated"], c["records"])
    for kw in (dict(key_center=a.kw["key_center"]), dict(center_rows=a.kw["center_rows"]),
               {**a.kw, "value_center": a.kw["value_center"][:2]},
               {**a.kw, "key_center": a.kw["key_center"].float()},
               {**a.kw, "center_rows": a.kw["center_rows"].long()}):
        with pytest.raises((RuntimeError, ValueError)):
            ext.rope_append_int4(a.q, a.k, a.v, a.cos, a.sin, a.positions, a.slots, a.rotated,
                                 a.pool.records, **kw)


# -------------------------------------------------------------- attention
class Attend:
    def __init__(self, lengths, hkv=2, group=4, dtype=F16, seed=1, center=True, split=0,
                 loud=1.0, offset=0.0, spare=3, v_scale=1.0):
        self.lengths, self.hkv, self.group = lengths, hkv, group
        rng = np.random.default_rng(seed)
        pages = [-(-n // 16) for n in lengths]
        total = sum(pages) + spare
        x = rng.standard_normal((2, total, hkv, 16, 128)).astype(np.float32)
        x[0, ..., :4] *= loud
        x += offset
        x[1] *= v_scale
        records = rng.integers(0, 256, (total, hkv, I.RECORD)).astype(np.uint8)
        self.order = rng.permutation(total)[:sum(pages)].astype(np.int32)
        kq, vq = I.quantise(x[0]), I.quantise(x[1])
        # Whole pages are stored; slots past a length keep the random bytes,
        # whose scales and midpoints hold NaN and infinities.
        at = 0
        for n in lengths:
            for p in range(-(-n // 16)):
                page = self.order[at]
                at += 1
                for h in range(hkv):
                    for t in range(min(16, n - 16 * p)):
                        I.store_token(records, page, h, t, [y[page, h, t] for y in kq],
                                      [y[page, h, t] for y in vq])
        for part in (2048, 2304):  # make sure of NaN, inf and the lowest value
            meta = records[:, :, part:part + 256].reshape(total, hkv, 16, 8, 2).view(np.uint16)
            at = 0
            for n in lengths:
                for p in range(-(-n // 16)):
                    for t in range(max(0, n - 16 * p), 16):
                        meta[self.order[at], :, t, ::4, 0] = 0x7e00
                        meta[self.order[at], :, t, 1::4, 0] = 0x7c00
                        meta[self.order[at], :, t, 2::4, 0] = 0xfbff
                    at += 1
            records[:, :, part:part + 256] = meta.view(np.uint8).reshape(total, hkv, 256)
        self.host = records
        self.records = torch.from_numpy(records).cuda()
        g = torch.Generator().manual_seed(seed)
        self.q = (torch.randn(len(lengths), hkv * group, 128, generator=g) * 1.2).to(dtype).cuda()
        self.center = None
        if center:
            self.center = torch.randn(len(lengths), hkv, 128, generator=g).to(dtype).cuda()
        self.indptr = torch.tensor([0] + pages).cumsum(0).int()
        self.indices = torch.from_numpy(self.order).cuda()
        self.last = torch.tensor([(n - 1) % 16 + 1 if n else 0 for n in lengths],
                                 dtype=torch.int32, device="cuda")
        self.wrapper = make_int4_wrapper(workspace=torch.empty(64 << 20, dtype=torch.uint8,
                                                               device="cuda"))
        self.split = split
        self.plan()

    def plan(self):
        plan(self.wrapper, self.indptr, self.indices, self.last, torch.uint8, self.split,
             num_qo_heads=self.hkv * self.group, num_kv_heads=self.hkv)

    def run(self, **kw):
        return self.wrapper.run(self.q, self.records, value_center=self.center, return_lse=True,
                                **kw)

    def check(self, out, lse, scale=128 ** -0.5, requests=None):
        eps = torch.finfo(out.dtype).eps / 2
        got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        c = None if self.center is None else self.center.double().cpu().numpy()
        worst = 0.0
        for r, n in enumerate(self.lengths):
            if requests is not None and r not in requests:
                continue
            ids = self.order[self.indptr[r]:self.indptr[r + 1]]
            if n == 0:
                assert (got[r] == 0).all() and np.isneginf(gl[r]).all()
                continue
            for h in range(self.hkv):
                (ka, km), (va, vm) = ([y.reshape(-1, 128)[:n] for y in pair]
                                      for pair in I.load(self.host[ids, h]))
                heads = slice(h * self.group, (h + 1) * self.group)
                exp, el, p = I.attention(q[r, heads], ka + km, va + vm, scale)
                size = scale * (np.abs(q[r, heads]) @ (np.abs(ka) + np.abs(km)).T).max(-1)
                e = 2.0 ** -19 * size + 2.0 ** -18
                big = np.abs(va) + np.abs(vm)
                bound = 2.0 ** -11 * (p @ np.abs(va)) + 2 * e[:, None] * (p @ big)
                # a subnormal step of each weight, over a sum of weights that
                # is at least a quarter of (sum p) / (max p)
                least = 1 / p.max(-1, keepdims=True) / 4
                bound += 2.0 ** -25 * 8 * n / np.maximum(least, 0.25)
                if c is not None:
                    exp = exp + c[r, h]
                bound = bound + eps * (np.abs(exp) + bound) + 2.0 ** -25 + 2.0 ** -23 * np.abs(exp)
                err = np.abs(got[r, heads] - exp)
                worst = max(worst, float((err / bound).max()))
                assert (err <= bound).all(), (r, h, float((err / bound).max()))
                lse_bound = 1.45 * (e + 2.0 ** -20) + 2.0 ** -22 * np.abs(el)
                assert (np.abs(gl[r, heads] - el) <= lse_bound).all(), (r, h)
        return worst


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,split", [
    ([1], 0), ([2], 0), ([15], 0), ([16], 0), ([17], 0), ([33], 1), ([64], 2), ([1000], 7),
    ([0, 5, 0, 300, 16, 1], 0), ([0], 0), ([129, 4097, 2], 128), ([1, 1, 1, 1], 1)])
def test_attention_lengths_and_splits(cuda_lib, dtype, lengths, split):
    a = Attend(lengths, dtype=dtype, split=split, seed=len(lengths) + sum(lengths))
    a.check(*a.run())
    assert read_device_error() == 0


@pytest.mark.parametrize("hkv,group", [(1, 1), (1, 2), (3, 3), (2, 5), (1, 7), (2, 8), (8, 4),
                                       (5, 6)])
def test_attention_head_groups(cuda_lib, hkv, group):
    a = Attend([130, 47], hkv=hkv, group=group, seed=hkv * 10 + group, center=hkv % 2 == 0)
    a.check(*a.run())


@pytest.mark.parametrize("loud,offset,v_scale", [(30.0, 0.0, 1.0), (1.0, 20.0, 1.0),
                                                 (1.0, 0.0, 1e-4), (1.0, 0.0, 2e4),
                                                 (1000.0, 0.0, 1.0)])
def test_attention_value_ranges(cuda_lib, loud, offset, v_scale):
    """Outlier channels, un-centred rows, tiny and huge values."""
    a = Attend([700, 90], loud=loud, offset=offset, v_scale=v_scale, center=False, seed=3)
    a.check(*a.run())


@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 1e-3, 30.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_query_ranges(cuda_lib, q_scale, dtype):
    a = Attend([300], dtype=dtype, seed=4)
    a.q = (a.q.float() * q_scale).to(dtype)
    a.check(*a.run())


def test_attention_long_context(cuda_lib):
    a = Attend([20011], hkv=1, group=4, seed=5)
    a.check(*a.run())
    a.check(*a.run(sm_scale=0.02), scale=float(np.float32(0.02)))


@pytest.mark.parametrize("split,group", [(1, 4), (1, 8), (128, 4)])
def test_attention_more_items_than_blocks(cuda_lib, split, group):
    """More work items than resident blocks: items are handed out by a counter
    that every run leaves at zero (run again, and replayed in a graph)."""
    rng = np.random.default_rng(14)
    lengths = [int(n) for n in rng.integers(1, 129, 70)]
    a = Attend(lengths, hkv=8, group=group, split=split, seed=15)
    assert a.wrapper._plan.num_items > 3 * 148
    assert a.wrapper._plan.single == (split == 128)
    out, lse = a.run()
    a.check(out, lse)
    graph = torch.cuda.CUDAGraph()
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    with torch.cuda.graph(graph):
        for _ in range(3):
            a.run(out=again, lse=lse2)
    for _ in range(2):
        again.zero_()
        graph.replay()
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("rounds", [1.0, 1.01, 1.6, 2.0, 2.01, 2.5, 3.0, 3.01, 4.3])
def test_attention_rounds_of_items(cuda_lib, rounds):
    """Plans of just under and over whole rounds of items; every run leaves the
    counter at zero, and splits agree within their bounds."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    items = int(rounds * 3 * sms)
    rng = np.random.default_rng(items)
    lengths = [int(n) for n in rng.integers(1, 129, 40)]
    while sum(-(-n // 16) for n in lengths) < items:
        lengths.append(int(rng.integers(1, 129)))
    lengths[-1] -= 16 * (sum(-(-n // 16) for n in lengths) - items)
    if lengths[-1] <= 0:
        lengths[-1] = 16
    a = Attend(lengths, hkv=1, group=3, split=1, seed=items)
    assert a.wrapper._plan.num_items in (items, items + 1)
    out, lse = a.run()
    a.check(out, lse)
    for _ in range(3):
        again = a.run()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for split in (0, 3):
        a.split = split
        a.plan()
        a.check(*a.run())
    assert read_device_error() == 0


def test_attention_last_page_without_tokens(cuda_lib):
    a = Attend([33, 16], seed=16)
    a.last[:] = 0  # 32 tokens, and none
    a.lengths = [32, 0]
    a.check(*a.run())


def test_two_wrappers_on_two_streams(cuda_lib):
    both = [Attend([3000, 100], hkv=4, seed=17), Attend([700, 2500], hkv=4, seed=18)]
    exp = [tuple(t.clone() for t in a.run()) for a in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (a, s) in enumerate(zip(both, streams)):
            with torch.cuda.stream(s):
                got[i].append(a.run())
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, exp[i][0]) and torch.equal(lse, exp[i][1])


def test_attention_strides_and_outputs(cuda_lib):
    a = Attend([100, 37, 250], seed=6)
    exp, exp_lse = (t.clone() for t in a.run())
    wide = torch.randn(3, 8, 300, device="cuda").half()
    wide[..., 2:130] = a.q
    a.q = wide[..., 2:130]
    out = torch.full((8, 3, 128), 5.0, dtype=F16, device="cuda").transpose(0, 1)
    lse = torch.empty(3, 8, device="cuda")
    got, got_lse = a.run(out=out, lse=lse)
    assert got is out and got_lse is lse
    assert torch.equal(out, exp) and torch.equal(lse, exp_lse)
    assert torch.equal(a.wrapper.run(a.q, Int4PagePool(a.records.size(0), 2, records=a.records),
                                     value_center=a.center), exp)
    # in place: the output is the query
    a.run(out=a.q)
    assert torch.equal(a.q, exp)


def test_attention_reports_bad_pages(cuda_lib):
    """A page outside the pool is left out: its tokens weigh nothing."""
    for bad in (-1, 10 ** 6):
        a = Attend([64, 40], seed=7)
        a.indices[1] = bad
        out, lse = a.run()
        assert read_device_error() == 3
        keep = np.delete(np.arange(64), range(16, 32))
        q = a.q.double().cpu().numpy()
        for h in range(2):
            (ka, km), (va, vm) = ([y.reshape(-1, 128) for y in pair]
                                  for pair in I.load(a.host[a.order[:4], h]))
            exp, el, _ = I.attention(q[0, 4 * h:4 * h + 4], (ka + km)[keep], (va + vm)[keep],
                                     128 ** -0.5)
            exp = exp + a.center[0, h].double().cpu().numpy()
            assert np.abs(out[0, 4 * h:4 * h + 4].double().cpu().numpy() - exp).max() < 4e-3
            assert np.abs(lse[0, 4 * h:4 * h + 4].double().cpu().numpy() - el).max() < 1e-4
        a.check(out, lse, requests=[1])


def test_attention_cuts_items_past_the_limit(cuda_lib):
    """An item of more pages than the four warps hold (a plan for eight warps)
    is cut at 128 pages and reported; the call ends and the others are whole."""
    import ctypes

    from pagegauge_b200 import _lib
    from pagegauge_b200.wrapper import PagedDecodePlan, _Workspace, plan_items

    a = Attend([16 * 200, 100], hkv=1, seed=19, center=False)
    items, off, info = plan_items(2, 1, a.indptr.numpy(), None, 200, 0, 148, 8)
    assert info.split_pages[0] == 200
    p = PagedDecodePlan(_Workspace(torch.empty(8 << 20, dtype=torch.uint8, device="cuda")), items,
                        off, info, 2, 1, 4)
    out, lse = torch.empty_like(a.q), torch.empty(2, 4, device="cuda")
    x = _lib.PgInt4DecodeArgs(
        q=a.q.data_ptr(), q_stride_b=512, q_stride_h=128, out=out.data_ptr(), out_stride_b=512,
        out_stride_h=128, lse_out=lse.data_ptr(), records=a.records.data_ptr(),
        num_pages=a.records.size(0), indices=a.indices.data_ptr(),
        last_page_len=a.last.data_ptr(), items=p.items_ptr, item_off=p.off_ptr, part_o=p.o_ptr,
        part_lse=p.lse_ptr, work_counter=p.sem_ptr, num_items=p.num_items, batch=2, kv_heads=1,
        group=4, final_mode=int(p.single), sm_scale=128 ** -0.5)
    _lib.check(cuda_lib.pg_decode_int4_run(ctypes.byref(x),
                                           torch.cuda.current_stream().cuda_stream))
    assert read_device_error() == 3
    a.check(out, lse, requests=[1])
    a.lengths = [16 * 128, 100]
    a.check(out, lse)


def test_attention_merges_with_an_exact_tail(cuda_lib):
    """The (out, lse) state joins an FP16 segment's through
    merge_state_in_place, as the INT8 wrapper's does."""
    a = Attend([160], center=False, seed=8)
    out, lse = a.run()
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(2, 16, 2, 128, generator=g).half().cuda() for _ in range(2))
    tail = BatchDecodeWithPagedKVCacheWrapper(torch.empty(8 << 20, dtype=torch.uint8,
                                                          device="cuda"))
    plan(tail, torch.tensor([0, 2], dtype=torch.int32),
         torch.arange(2, dtype=torch.int32, device="cuda"),
         torch.tensor([5], dtype=torch.int32, device="cuda"), F16, num_qo_heads=8, num_kv_heads=2)
    o2, l2 = tail.run(a.q, (k, v), return_lse=True)
    merge_state_in_place(out, lse, o2, l2)
    q = a.q.double().cpu().numpy()
    for h in range(2):
        (ka, km), (va, vm) = ([y.reshape(-1, 128) for y in pair]
                              for pair in I.load(a.host[a.order, h]))
        kk = np.concatenate((ka + km, k[:, :, h].reshape(-1, 128)[:21].double().cpu().numpy()))
        vv = np.concatenate((va + vm, v[:, :, h].reshape(-1, 128)[:21].double().cpu().numpy()))
        exp, el, _ = I.attention(q[0, 4 * h:4 * h + 4], kk, vv, 128 ** -0.5)
        assert np.abs(out[0, 4 * h:4 * h + 4].double().cpu().numpy() - exp).max() < 2e-3
        assert np.abs(lse[0, 4 * h:4 * h + 4].double().cpu().numpy() - el).max() < 2e-4


def test_attention_repeats_bit_for_bit_and_in_graphs(cuda_lib):
    """Same inputs, same bits: eager, again, captured and replayed after the
    lengths grew within their pages, and on another stream."""
    a = Attend([500, 3, 0, 1200], seed=10, split=9)
    out, lse = a.run()
    again, lse2 = a.run()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run(out=again, lse=lse2)
    a.q.mul_(0.5)
    a.last[0] = 2  # 500 = 31 * 16 + 4 tokens become 498
    graph.replay()
    a.lengths = [498, 3, 0, 1200]
    a.check(again, lse2)
    out, lse = a.run()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = a.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_attention_refusals(cuda_lib):
    a = Attend([40, 20], seed=11)
    with pytest.raises(RuntimeError, match="plan"):
        make_int4_wrapper(workspace=torch.empty(1 << 20, dtype=torch.uint8,
                                                device="cuda")).run(a.q, a.records)
    with pytest.raises(ValueError):
        make_int4_wrapper()
    with pytest.raises(ValueError):
        Int4DecodeWrapper(torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), page_gauge=True)
    bad = [dict(q=a.q.float()), dict(q=a.q[:1]), dict(q=a.q[:, :4]), dict(q=a.q.cpu()),
           dict(records=a.records[:, :1]), dict(records=a.records.cpu()),
           dict(records=a.records[..., :1280]), dict(value_center=a.center.float()),
           dict(value_center=a.center[:1]), dict(out=torch.empty_like(a.q).bfloat16()),
           dict(out=a.q[:, :1].expand(a.q.shape)), dict(sm_scale=0.0),
           dict(sm_scale=float("inf")), dict(lse=torch.empty(2, 4, device="cuda")),
           dict(lse=torch.empty(2, 8, device="cuda").half())]
    for kw in bad:
        c = {**dict(q=a.q, records=a.records), **kw}
        with pytest.raises((RuntimeError, ValueError)):
            a.wrapper.run(c.pop("q"), c.pop("records"), **c)
    for args in ((a.indptr, a.indices[:2], a.last), (a.indptr, a.indices.long(), a.last),
                 (a.indptr, a.indices, a.last[:1]),
                 (torch.tensor([0, 3, 2], dtype=torch.int32), a.indices, a.last)):
        with pytest.raises((RuntimeError, ValueError)):
            plan(a.wrapper, *args, torch.uint8, num_qo_heads=8, num_kv_heads=2)
    with pytest.raises(ValueError, match="uint8"):
        plan(a.wrapper, a.indptr, a.indices, a.last, torch.int8, num_qo_heads=8, num_kv_heads=2)
    with pytest.raises(ValueError):
        plan(a.wrapper, a.indptr, a.indices, a.last, torch.uint8, num_qo_heads=18, num_kv_heads=2)


# ------------------------------------------------------------- as one path
def test_inputs_that_require_gradients_are_refused(cuda_lib):
    """And what a call writes carries a new version."""
    a = Attend([33], hkv=2, seed=23)
    w = a.wrapper
    with pytest.raises(ValueError, match="no gradient"):
        w.run(a.q.clone().requires_grad_(), a.records)
    with torch.no_grad():
        got = w.run(a.q.clone().requires_grad_(), a.records)
    assert torch.equal(got, w.run(a.q, a.records)) and not got.requires_grad
    out = torch.zeros_like(a.q)
    version = out._version
    w.run(a.q, a.records, out=out)
    assert out._version > version
    b = Append(3, 4, 2)
    version = b.pool.records._version
    b.run()
    assert b.pool.records._version > version
    b.k = b.k.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        b.run()


def test_prompt_then_decode_steps(cuda_lib):
    """A prompt appended in one call, then tokens one by one, attending after
    each: records equal the oracle's, outputs the attention over them."""
    hq, hkv, prompt, steps = 8, 2, 45, 6
    ext = load_append_extension()
    g = torch.Generator().manual_seed(12)
    lengths = [prompt, 17]
    pool = Int4PagePool(12, hkv)
    table = [[7, 2, 9, 4], [1, 5]]
    cos, sin = rotary_tables(64, 128, device="cuda")
    center = torch.randn(2, 2, hkv, 128, generator=g).half().cuda() * 0.2
    kw = dict(key_center=center[0], value_center=center[1])
    draw = lambda n, h: torch.randn(n, h, 128, generator=g).half().cuda()  # noqa: E731

    def append(rows, q, k, v):
        pos = torch.tensor([p for _, p in rows], dtype=torch.int32, device="cuda")
        slots = torch.tensor([table[r][p // 16] * 16 + p % 16 for r, p in rows],
                             dtype=torch.int32, device="cuda")
        which = torch.tensor([r for r, _ in rows], dtype=torch.int32, device="cuda")
        rotated = torch.empty_like(q)
        ext.rope_append_int4(q, k, v, cos, sin, pos, slots, rotated, pool.records,
                             center_rows=which, **kw)
        return rotated

    rows = [(r, p) for r, n in enumerate(lengths) for p in range(n)]
    append(rows, draw(len(rows), hq), draw(len(rows), hkv), draw(len(rows), hkv))
    wrapper = make_int4_wrapper(workspace=torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    for _ in range(steps):
        rows = [(r, n) for r, n in enumerate(lengths)]
        q = append(rows, draw(2, hq), draw(2, hkv), draw(2, hkv))
        lengths = [n + 1 for n in lengths]
        pages = [-(-n // 16) for n in lengths]
        a = Attend.__new__(Attend)
        a.lengths, a.hkv, a.group, a.q, a.center = lengths, hkv, hq // hkv, q, center[1]
        a.order = np.array(sum((t[:n] for t, n in zip(table, pages)), []), np.int32)
        a.indptr = torch.tensor([0] + pages).cumsum(0).int()
        plan(wrapper, a.indptr, torch.from_numpy(a.order).cuda(),
             torch.tensor([(n - 1) % 16 + 1 for n in lengths], dtype=torch.int32, device="cuda"),
             torch.uint8, num_qo_heads=hq, num_kv_heads=hkv)
        out, lse = wrapper.run(q, pool, value_center=center[1], return_lse=True)
        a.host = cpu(pool.records)
        a.check(out, lse)
    assert read_device_error() == 0


def test_plan_rounds_only_its_own_split(cuda_lib):
    a = Attend([4096], hkv=8, seed=13)
    assert a.wrapper.split_pages == 8
    a.check(*a.run())
    a.split = 5
    a.plan()
    assert a.wrapper.split_pages == 5
    a.check(*a.run())


@pytest.mark.parametrize("lengths", [[5], [300]])
def test_a_workspace_at_an_odd_byte_is_refused(cuda_lib, lengths):
    a = Attend(lengths, seed=2)
    for skip in (1, 2):
        a.wrapper = make_int4_wrapper(workspace=torch.empty(8 << 20, dtype=torch.uint8,
                                                            device="cuda")[skip:])
        a.plan()
        with pytest.raises(RuntimeError, match="aligned"):
            a.run()


@pytest.mark.parametrize("lengths,hkv,group", [
    ([16 * 700] + [3] * 20, 1, 4),  # 88 partials on one head, one on the others
    ([1, 0, 16 * 500 + 5, 17], 3, 8), ([2000] + [9, 0] * 60, 2, 2),
    ([5] * 70 + [16 * 300], 4, 8)])  # joined by a warp per row: many rows
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_skewed_batches(cuda_lib, lengths, hkv, group, dtype):
    """One long request among short ones, joined as the plan's largest head and as the
    mean over the heads would have it: the same within the bound, and the choice is
    the plan's."""
    a = Attend(lengths, hkv=hkv, group=group, dtype=dtype, split=8, seed=7)
    p = a.wrapper._plan
    assert p.most_items == max(np.diff(p.host_off)) == -(-(-(-max(lengths) // 16)) // 8)
    a.check(*a.run())
    field = _lib.PgInt4DecodeArgs.most_items.offset
    block = a.wrapper._block
    for most in (0, 1, 1 << 30):  # the mean, a warp per row, a block per row
        a.wrapper._block = block[:field] + most.to_bytes(4, "little") + block[field + 4:]
        a.check(*a.run())
    assert read_device_error() == 0
