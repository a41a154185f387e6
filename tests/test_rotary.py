"""Rotary tables (CPU): exact angles at far positions, the scalings' formulas,
and the refusals of apply_rotary and of the C entry that need no GPU."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import int4_oracle as I
from pagegauge_b200 import _lib
from pagegauge_b200.rotary import RotaryScaling, apply_rotary, rotary_frequencies, rotary_tables


@pytest.mark.parametrize("rotary_dim", [2, 34, 64, 128])
def test_tables_hold_64_bit_angles(rotary_dim):
    cos, sin = rotary_tables(4, rotary_dim)
    assert cos.shape == sin.shape == (4, rotary_dim // 2) and cos.dtype == torch.float32
    positions = 131072
    cos, sin = rotary_tables(positions, rotary_dim)
    p = positions - 1
    for j in range(rotary_dim // 2):
        angle = p * math.exp(-2 * j / rotary_dim * math.log(1e6))
        # A rounding of the table to FP32, and of the 64-bit angle (2^17 * 2^-52).
        assert abs(float(cos[p, j]) - math.cos(angle)) <= 2 ** -25 + 2 ** -33
        assert abs(float(sin[p, j]) - math.sin(angle)) <= 2 ** -25 + 2 ** -33


def test_scalings():
    base, one = rotary_frequencies(128)
    assert one == 1.0
    inv, scale = rotary_frequencies(128, scaling=RotaryScaling("linear", 4.0))
    assert scale == 1.0 and torch.equal(inv, base / 4)
    inv, scale = rotary_frequencies(128, scaling=RotaryScaling("ntk", 4.0))
    assert scale == 1.0 and inv[0] == 1.0
    assert math.isclose(float(inv[-1]), float(base[-1]) / 4, rel_tol=1e-12)
    s = RotaryScaling("parts", 8.0, trained_positions=8192)
    inv, scale = rotary_frequencies(128, scaling=s)
    assert math.isclose(scale, 0.1 * math.log(8) + 1)
    turns = base * 8192 / (2 * math.pi)
    assert torch.equal(inv[turns > 40], base[turns > 40])
    torch.testing.assert_close(inv[turns < 0.7], base[turns < 0.7] / 8, rtol=1e-12, atol=0)
    between = (inv < base) & (inv > base / 8)
    assert between.any() and (inv[:-1] > inv[1:]).all()
    _, scale = rotary_frequencies(128, scaling=RotaryScaling("parts", 8.0, attention_factor=1.25))
    assert scale == 1.25
    cos, _ = rotary_tables(1, 64, scaling=s)
    assert float(cos[0, 0]) == np.float32(0.1 * math.log(8) + 1)


def test_bad_scalings_and_tables_are_refused():
    for bad in (dict(kind="cubic", factor=2.0), dict(kind="linear", factor=0.5),
                dict(kind="parts", factor=float("inf")),
                dict(kind="parts", factor=2.0, fast_turns=1.0, slow_turns=2.0),
                dict(kind="parts", factor=2.0, trained_positions=0)):
        with pytest.raises(ValueError):
            RotaryScaling(**bad)
    for bad in (dict(positions=0), dict(positions=4, rotary_dim=7),
                dict(positions=4, rotary_dim=0), dict(positions=4, theta=1.0)):
        with pytest.raises(ValueError):
            rotary_tables(**bad)


def test_cpu_rows_are_refused():
    q = torch.zeros(2, 4, 128)
    cos, sin = rotary_tables(8, 128)
    with pytest.raises(ValueError, match="CUDA"):
        apply_rotary(q, None, cos, sin, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="float16"):
        apply_rotary(q.to(torch.int8), None, cos, sin, torch.zeros(2, dtype=torch.int32))


def test_c_entry_refusals_without_gpu():
    lib = _lib.load()

    def call(**kw):
        a = _lib.PgRotaryArgs()
        a.x[0], a.y[0] = 0x1000, 0x2000
        a.heads[0], a.tokens, a.head_dim, a.pairs = 4, 1, 128, 64
        a.table_rows, a.table_stride = 8, 64
        a.cosine = a.sine = a.positions = 0x3000
        for k, v in kw.items():
            setattr(a, k, v)
        rc = lib.pg_rotary(ctypes.byref(a), None)
        return rc, lib.pg_last_error()

    for kw, message in ((dict(dtype=3), b"dtype"), (dict(tokens=-1), b"non-negative"),
                        (dict(pairs=65), b"rotated dims"), (dict(pairs=0), b"rotated dims"),
                        (dict(table_rows=0), b"tables"), (dict(table_stride=63), b"tables"),
                        (dict(cosine=None), b"required"), (dict(positions=None), b"required")):
        rc, error = call(**kw)
        assert rc == 1 and message in error, (kw, error)
    assert call(tokens=0)[0] == 0  # nothing to do
    assert lib.pg_rotary(None, None) == 1


def test_oracle_adjoint_is_the_transpose():
    rng = np.random.default_rng(1)
    x, y = rng.standard_normal((2, 3, 2, 16))
    cos, sin = rng.standard_normal((2, 3, 5))
    for interleaved in (False, True):
        lhs = (I.rotate(x, cos, sin, interleaved) * y).sum()
        rhs = (x * I.rotate(y, cos, sin, interleaved, adjoint=True)).sum()
        assert abs(lhs - rhs) < 1e-12


def test_cpu_rows_that_require_gradients_are_refused_alike():
    q = torch.zeros(2, 4, 128, requires_grad=True)
    k = torch.zeros(2, 2, 128, requires_grad=True)
    cos, sin = rotary_tables(8, 128)
    positions = torch.zeros(2, dtype=torch.int32)
    for key in (None, k, k.detach()):
        with pytest.raises(ValueError, match="CUDA"):
            apply_rotary(q, key, cos, sin, positions)
    with pytest.raises(ValueError, match="CUDA"):
        apply_rotary(q.detach(), k, cos, sin, positions)
