"""The 4-bit cache on the CPU: the record layout and the quantiser's bounds in
the oracle, and the refusals of the C entries and the Python classes."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pagegauge_b200 import _lib
from pagegauge_b200.int4 import Int4PagePool


def test_codes_fill_a_record_once():
    seen = np.zeros((I.RECORD, 2), int)
    for t in range(16):
        for d in range(128):
            seen[I.key_byte(t, d)] += 1
            seen[I.value_byte(t, d)] += 1
    assert (seen[:2048] == 1).all() and (seen[2048:] == 0).all()


def test_store_and_load_round_trip():
    rng = np.random.default_rng(1)
    records = rng.integers(0, 256, (3, 2, I.RECORD), np.uint8)
    x = rng.standard_normal((2, 128)).astype(np.float32)
    k, v = (I.quantise(row) for row in x)
    other = records.copy()
    I.store_token(records, 1, 1, 5, k, v)
    (ka, km), (va, vm) = I.load(records[1, 1])
    for (z, s, m), got in ((k, ka[5] + km[5]), (v, va[5] + vm[5])):
        exp = (z.astype(float) - 8) * np.repeat(s.astype(float), 32) + np.repeat(m.astype(float), 32)
        assert np.array_equal(got, exp)
    touched = np.argwhere(records[1, 1] != other[1, 1])
    assert len(touched) <= 160 and np.array_equal(records[0], other[0])


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 1.0, 300.0, 4e4])
@pytest.mark.parametrize("offset", [0.0, 50.0])
def test_quantiser_error_is_half_a_step(scale, offset):
    """|x - x'| <= s/2 inside the codes' range; beyond it the scale's and the
    midpoint's roundings (2^-11 relative, or half a subnormal step) add."""
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((64, 128)) * scale + offset).astype(np.float32)
    x = np.clip(x, -65504, 65504)
    z, s, m = (t.astype(np.float64) for t in I.quantise(x))
    s, m = np.repeat(s, 32, -1), np.repeat(m, 32, -1)
    err = np.abs((z - 8) * s + m - x)
    slack = 15 * np.maximum(s * 2.0 ** -11, 2.0 ** -25) + np.maximum(np.abs(m) * 2.0 ** -11,
                                                                     2.0 ** -25)
    assert (err <= s * (0.5 + 2.0 ** -20) + slack).all()


def test_constant_groups_are_held_to_one_rounding():
    x = np.repeat(np.float32([3.0, -7.5, 0.0, 1000.25]), 32)[None]
    z, s, m = I.quantise(x)
    assert (s == 0).all() and (z == 8).all()
    assert np.array_equal(np.repeat(m, 32, -1), x.astype(np.float16))


def append_args(**kw):
    a = _lib.PgInt4AppendArgs()
    a.query = a.key = a.value = a.rotated_query = a.records = 0x1000
    a.cosine = a.sine = a.positions = a.slots = 0x1000
    a.table_rows, a.table_stride, a.pairs = 8, 64, 64
    a.num_pages, a.tokens, a.query_heads, a.kv_heads = 4, 1, 4, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def decode_args(**kw):
    a = _lib.PgInt4DecodeArgs()
    a.q = a.out = a.records = a.indices = a.last_page_len = a.items = a.item_off = 0x1000
    a.part_o = a.part_lse = a.work_counter = 0x1000
    a.num_items, a.batch, a.kv_heads, a.group, a.num_pages, a.sm_scale = 2, 1, 1, 4, 4, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry,make,bad", [
    ("pg_rope_append_int4", append_args,
     [dict(dtype=2), dict(tokens=-1), dict(query_heads=0), dict(kv_heads=0), dict(pairs=65),
      dict(pairs=0), dict(table_rows=0), dict(table_stride=63), dict(num_pages=0),
      dict(num_pages=1 << 27), dict(key_center=0x1000), dict(records=0x1008),
      dict(records=None), dict(slots=None), dict(rotated_query=None),
      dict(key_center=0x1000, value_center=0x1000, num_centers=0)]),
    ("pg_decode_int4_run", decode_args,
     [dict(batch=0), dict(group=9), dict(group=0), dict(sm_scale=0.0),
      dict(sm_scale=float("nan")), dict(dtype=2), dict(q=0x1002), dict(q_stride_h=3),
      dict(out=None), dict(num_items=-1), dict(num_pages=0), dict(records=0x1004),
      dict(indices=None), dict(items=None), dict(item_off=None), dict(part_o=None), dict(part_o=0x1004), dict(work_counter=None)]),
])
def test_c_entries_refuse(entry, make, bad):
    fn = getattr(_lib.load(), entry)
    assert fn(None, None) == 1
    for kw in bad:
        assert fn(ctypes.byref(make(**kw)), None) == 1, kw
        assert _lib.load().pg_last_error()
    if entry == "pg_rope_append_int4":
        assert fn(ctypes.byref(make(tokens=0)), None) == 0


def test_read_refuses():
    fn = _lib.load().pg_int4_read
    good = [0x1000, 4, 1, 0x1000, 1, 0x1000, 0x1000, 0, None]
    for i, v in ((0, None), (0, 0x1004), (1, 0), (2, 0), (3, None), (4, -1), (5, 0x1008), (7, 3)):
        bad = list(good)
        bad[i] = v
        assert fn(*bad) == 1, (i, v)
    good[4] = 0
    assert fn(*good) == 0


def test_pool_refuses():
    with pytest.raises(ValueError):
        Int4PagePool(0, 8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        Int4PagePool(2, 8, device="cpu")
    with pytest.raises(ValueError):
        Int4PagePool(2, 8, records=torch.zeros(2, 8, 2559, dtype=torch.uint8))


@pytest.mark.parametrize("structure", [_lib.PgRotaryArgs, _lib.PgInt4AppendArgs,
                                       _lib.PgInt4DecodeArgs])
def test_packed_arguments_have_the_structure_s_layout(structure):
    pack = _lib.packer(structure)
    assert pack.size == ctypes.sizeof(structure)
    count = len(pack.unpack(bytes(pack.size)))
    a = structure.from_buffer_copy(pack.pack(*range(1, count + 1)))
    got = []
    for name, _ in structure._fields_:
        value = getattr(a, name)
        got += list(value) if isinstance(value, ctypes.Array) else [value]
    assert got == list(range(1, count + 1))


def test_automatic_splits_are_whole_pairs_of_four_warps():
    from pagegauge_b200.wrapper import Int4DecodeWrapper, plan_items

    assert Int4DecodeWrapper._split_multiple == 8
    # What plan() does with the planner's automatic split.
    indptr = np.array([0, 256], np.int32)
    _, _, info = plan_items(1, 8, indptr, None, 0, 0, 148)
    split = -(-info.split_pages[0] // 8) * 8
    items, off, info = plan_items(1, 8, indptr, None, split, split, 148)
    assert info.split_pages[0] == split == 8 and off[-1] == 8 * 32


def split_pages(pages, kv_heads, group=4, sms=148, multiple=8):
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    split = ctypes.c_int32()
    _lib.call("pg_int4_split_pages", len(pages), kv_heads, group, indptr.ctypes.data, sms, multiple,
              ctypes.byref(split))
    return split.value


@pytest.mark.parametrize("pages,kv_heads,group,best", [
    # The fastest of measured splits, or one within 3 % of it.
    ([3923] * 4, 4, 4, (72,)), ([3923] * 4, 4, 7, (72,)), ([3000], 8, 4, (56,)),
    ([6250], 8, 4, (120,)), ([8192], 8, 4, (80,)), ([256], 8, 8, (8,)), ([63], 8, 4, (8,)),
    ([53] * 22, 8, 5, (32,)), ([256] * 32, 8, 4, (88,)), ([13] * 64, 8, 4, (16,)),
    ([713] * 12, 1, 8, (24,)), ([128] * 64, 8, 4, (64, 72, 48)), ([512] * 16, 8, 4, (80, 88))])
def test_automatic_split_is_the_measured_one(pages, kv_heads, group, best):
    assert split_pages(pages, kv_heads, group) in best


def test_automatic_split_of_any_plan():
    rng = np.random.default_rng(5)
    assert split_pages([0, 0], 4) == 8
    for _ in range(200):
        pages = rng.integers(0, rng.integers(2, 5000), rng.integers(1, 80))
        split = split_pages(list(pages), int(rng.integers(1, 9)), int(rng.integers(1, 9)),
                            int(rng.integers(1, 200)))
        assert split % 8 == 0 and 8 <= split <= 128
    assert split_pages([100], 1, multiple=500) == 128
    split, bad = ctypes.c_int32(), np.array([0, 4, 2], np.int32)
    for args in ((0, 1, 4, bad.ctypes.data, 148, 8), (2, 0, 4, bad.ctypes.data, 148, 8),
                 (2, 1, 4, bad.ctypes.data, 148, 8), (1, 1, 4, None, 148, 8),
                 (1, 1, 4, bad.ctypes.data, 0, 8), (1, 1, 4, bad.ctypes.data, 148, 0)):
        with pytest.raises((RuntimeError, ValueError)):
            _lib.call("pg_int4_split_pages", *args, ctypes.byref(split))


def test_binding_refuses_what_is_not_a_cuda_tensor():
    ops = _lib.torch_ops()
    q = torch.zeros(2, 4, 128, dtype=torch.float16)
    k = torch.zeros(2, 1, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="query must be a tensor"):
        ops.rope_append_int4(*([None] * 13), False)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_append_int4(q, k, k, q, q, q, q, q, q, None, None, None, None, False)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary(q, k, q, q, q, False, False, None, None)
    with pytest.raises(ValueError, match="dtype"):
        ops.int4_read(q, q, "half", None, None)
    with pytest.raises(ValueError, match="argument block"):
        ops.decode_int4(b"", 0, q, q, 1.0, None, None, None, False)
    with pytest.raises(TypeError, match="arguments"):
        ops.rotary(q)


def test_binding_refuses_forward_mode_duals():
    """A dual tensor does not require a gradient; its tangent would be lost all
    the same, with gradients recorded or not."""
    import torch.autograd.forward_ad as forward

    ops = _lib.torch_ops()
    plain = torch.zeros(2, 4, 128)
    plan = bytes(ctypes.sizeof(_lib.PgInt4DecodeArgs))
    with forward.dual_level():
        dual = forward.make_dual(plain, torch.ones_like(plain))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for at in (0, 1, 2, 3, 7, 8):
                    args = [plain] * 9
                    args[at], args[5], args[6] = dual, False, False
                    with pytest.raises(ValueError, match="forward-mode"):
                        ops.rotary(*args)
                for at in (0, 1, 2, 3, 4, 7, 9, 10, 12):
                    args = [plain] * 14
                    args[at], args[13] = dual, False
                    with pytest.raises(ValueError, match="forward-mode"):
                        ops.rope_append_int4(*args)
                for at in (3, 4):
                    args = [plain, plain, torch.float16, plain, plain]
                    args[at] = dual
                    with pytest.raises(ValueError, match="forward-mode"):
                        ops.int4_read(*args)
                for at in (2, 5, 6, 7):
                    args = [plan, 0, plain, plain, 1.0, plain, plain, plain, False]
                    args[at] = dual
                    with pytest.raises(ValueError, match="forward-mode"):
                        ops.decode_int4(*args)
        rows = forward.make_dual(plain.clone().requires_grad_(), torch.ones_like(plain))
        with pytest.raises(ValueError, match="forward-mode"):
            ops.rotary(rows, None, plain, plain, plain, False, False, None, None)


def test_automatic_split_at_the_ends_of_its_ranges():
    """Page counts whose items pass 32 bits, as many heads as are taken, and a
    multiple that has no second one: an answer within the range, at once."""
    for pages in ([2 ** 31 - 1], [2 ** 30, 0, 2 ** 30 - 1], [2 ** 27 - 1]):
        for kv_heads in (8, 65535):
            for sms in (1, 148, 2 ** 31 - 1):
                split = split_pages(pages, kv_heads, sms=sms)
                assert split % 8 == 0 and 8 <= split <= 128
    assert split_pages([200], 8, multiple=2 ** 31 - 1) == 128
    assert split_pages([200], 8, multiple=127) == 127


@pytest.mark.parametrize("sms,kv_heads,group", [(1, 1, 4), (2, 3, 8), (5, 2, 1)])
def test_automatic_split_counts_rounds_as_handed_out(sms, kv_heads, group):
    """The estimate against one that lists the items and their rounds one by one."""
    rng = np.random.default_rng(sms)
    for _ in range(40):
        pages = [int(n) for n in rng.integers(0, rng.integers(2, 700), rng.integers(1, 12))]
        blocks, costs = 3 * sms, {}
        for s in range(8, 129, 8):
            items = sorted((x for n in pages for x in [s] * (n // s) + [n % s] * (n % s > 0)
                            for _ in range(kv_heads)), reverse=True)
            if not items:
                continue

            def page(k):
                return (1.15 if group > 4 else 1.0) * (
                    0.12 + 0.06 * min(1.0, (len(items) - k * blocks) / blocks))

            cost = items[0] * page(0)
            for i in range(blocks, min(len(items), 2 * blocks)):
                cost = max(cost, items[2 * blocks - 1 - i] * page(0) + items[i] * page(1))
            for k in range(2, -(-len(items) // blocks)):
                cost += items[k * blocks] * page(k)
            cost += 2.6 * ((len(items) - 1) // blocks)
            cost += 2.5 * (0 in pages or len(items) != len(pages) * kv_heads)
            costs[s] = cost
        split = split_pages(pages, kv_heads, group, sms=sms)
        assert split == 8 if not costs else costs[split] <= min(costs.values()) * (1 + 1e-9)


@pytest.mark.parametrize("final_mode", [0, 1])
def test_c_entries_refuse_misaligned_words(final_mode):
    """A workspace that starts at an odd byte puts a plan's words there, and a
    single-item plan needs no partial states whose alignment is looked at."""
    lib = _lib.load()
    for name in ("indices", "last_page_len", "items", "item_slots", "item_off", "part_lse",
                 "work_counter", "lse_out", "out", "value_center"):
        a = decode_args(final_mode=final_mode, **{name: 0x1001})
        assert lib.pg_decode_int4_run(ctypes.byref(a), None) == 1, name
        assert b"aligned" in lib.pg_last_error()
    for name in ("query", "key", "value", "rotated_query", "rotated_key", "cosine", "sine",
                 "positions", "slots"):
        a = append_args(**{name: 0x1001})
        assert lib.pg_rope_append_int4(ctypes.byref(a), None) == 1, name
        assert b"aligned" in lib.pg_last_error()
    assert lib.pg_int4_read(0x1000, 4, 1, 0x1002, 1, 0x1000, 0x1000, 0, None) == 1
    for dtype, at in ((0, 1), (1, 1), (2, 2)):
        for name in ("x", "y", "cosine", "sine", "positions"):
            a = _lib.PgRotaryArgs()
            a.x[0], a.y[0] = 0x1000, 0x2000
            a.heads[0], a.tokens, a.head_dim, a.pairs = 4, 1, 128, 64
            a.table_rows, a.table_stride, a.dtype = 8, 64, dtype
            a.cosine = a.sine = a.positions = 0x3000
            if name in "xy":
                getattr(a, name)[0] += at
            else:
                setattr(a, name, 0x3000 + at)
            assert lib.pg_rotary(ctypes.byref(a), None) == 1, (dtype, name)
            assert b"aligned" in lib.pg_last_error()


@pytest.mark.parametrize("pages,kv_heads,group", [([256], 8, 4), ([3923] * 4, 4, 7), ([0, 5, 300], 2, 8),
                                                  ([1], 1, 1)])
def test_the_wrapper_plans_with_the_split_it_chose(pages, kv_heads, group):
    """What plan() does on the host: the split goes to the planner as it is, and the
    items cover every page of every head once, in items of at most it."""
    from pagegauge_b200.wrapper import Int4DecodeWrapper, plan_items

    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    wrapper = object.__new__(Int4DecodeWrapper)
    split = wrapper._automatic_split(indptr, kv_heads, group, 148)
    assert split == split_pages(pages, kv_heads, group) and split % wrapper._split_multiple == 0
    items, off, info = plan_items(len(pages), kv_heads, indptr, None, split, split, 148)
    assert info.split_pages[0] == split and off[-1] == len(items)
    seen = np.zeros((kv_heads, indptr[-1]), int)
    for request, head, begin, count in items:
        n = count & 0x7FFFFFFF
        assert 1 <= n <= split and indptr[request] <= begin and begin + n <= indptr[request + 1]
        assert (count < 0) == (begin + n == indptr[request + 1])
        seen[head, begin:begin + n] += 1
    assert (seen == 1).all()
