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

PAGE = 16
HEAD_DIM = 128
GROUP = 32
RECORD_BYTES = 2560


def check_records(records: torch.Tensor) -> None:
    if (not records.is_cuda or records.dtype != torch.uint8 or records.dim() != 3
            or records.size(0) == 0 or records.size(1) == 0 or records.size(2) != RECORD_BYTES
            or not records.is_contiguous() or records.data_ptr() % 16):
        raise ValueError(f"records must be contiguous 16-byte aligned CUDA uint8 "
                         f"[pages,Hkv,{RECORD_BYTES}]")
    if records.size(0) >= 1 << 27:
        raise ValueError("a pool holds fewer than 2^27 pages")


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
        return (_lib._ops or _lib.torch_ops()).int4_read(self.records, slots, dtype, key_out,
                                                         value_out)
