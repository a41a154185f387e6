"""The 4-bit paged cache: a pool of records, one of 2560 bytes per (page of
16 tokens, KV head), that ``AppendExtension.rope_append_int4`` writes and
``wrapper.make_int4_wrapper`` attends over.

A token's key and value are each held as 128 codes z of 4 bits with an FP16
scale s and midpoint m per group of 32 dims, x ~ (z - 8) s + m (160 bytes per
token and KV head for both; the INT8 cache holds 256 and FP16 512).  Scales
belong to one token, so a token is appended in 4 bits at once and no FP16
ring of recent pages is needed.  The record's byte layout is in
include/pagegauge_b200.h.
"""

from __future__ import annotations

import torch

from . import _lib
from .rotary import DTYPES, check_token_index

PAGE = 16
HEAD_DIM = 128
GROUP = 32
RECORD_BYTES = 2560


def check_records(records: torch.Tensor) -> tuple[int, int, int]:
    """(address, pages, KV heads) of a pool's records."""
    shape = records.shape
    address = records.data_ptr()
    if (not records.is_cuda or records.dtype is not torch.uint8 or len(shape) != 3
            or shape[0] == 0 or shape[1] == 0 or shape[2] != RECORD_BYTES
            or not records.is_contiguous() or address % 16):
        raise ValueError(f"records must be contiguous 16-byte aligned CUDA uint8 "
                         f"[pages,Hkv,{RECORD_BYTES}]")
    if shape[0] >= 1 << 27:
        raise ValueError("a pool holds fewer than 2^27 pages")
    return address, shape[0], shape[1]


class Int4PagePool:
    """``num_pages`` pages of ``kv_heads`` records; ``records`` may be a
    caller's uint8 tensor [num_pages, kv_heads, 2560]."""

    def __init__(self, num_pages: int, kv_heads: int, device: torch.device | str = "cuda",
                 records: torch.Tensor | None = None):
        if num_pages <= 0 or kv_heads <= 0:
            raise ValueError("page and head counts must be positive")
        if records is None:
            records = torch.zeros(num_pages, kv_heads, RECORD_BYTES, dtype=torch.uint8,
                                  device=device)
        check_records(records)
        if tuple(records.shape[:2]) != (num_pages, kv_heads):
            raise ValueError(f"records must be [{num_pages},{kv_heads},{RECORD_BYTES}]")
        self.records = records
        self.num_pages, self.kv_heads = num_pages, kv_heads

    @property
    def device(self) -> torch.device:
        return self.records.device

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             key_out: torch.Tensor | None = None, value_out: torch.Tensor | None = None):
        """The (key, value) values held at ``slots`` (device int32 [T], page *
        16 + token), [T, Hkv, 128] each, without the centres that an append
        subtracted.  Negative slots give zeros; slots outside the pool give
        zeros and set the device guard word."""
        if dtype not in DTYPES:
            raise ValueError("values are read as float16, bfloat16 or float32")
        records = self.records
        device, tokens, kv_heads = records.device, slots.numel(), self.kv_heads
        slot_ptr = check_token_index(slots, "slots", tokens, device)
        if key_out is None and value_out is None:
            shape, strides = (tokens, kv_heads, HEAD_DIM), (kv_heads * HEAD_DIM, HEAD_DIM, 1)
            key_out = torch.empty_strided(shape, strides, dtype=dtype, device=device)
            value_out = torch.empty_strided(shape, strides, dtype=dtype, device=device)
        else:
            shape = (tokens, kv_heads, HEAD_DIM)
            for name, t in (("key_out", key_out), ("value_out", value_out)):
                if (t is None or t.shape != shape or t.dtype is not dtype or t.device != device
                        or not t.is_contiguous() or t.data_ptr() % 16):
                    raise ValueError(f"{name} must be contiguous 16-byte aligned "
                                     f"[T,{kv_heads},{HEAD_DIM}] {dtype} (both outputs or none)")
        _lib.launch("pg_int4_read", device, records.data_ptr(), self.num_pages, kv_heads,
                    slot_ptr, tokens, key_out.data_ptr(), value_out.data_ptr(), DTYPES[dtype])
        return key_out, value_out
