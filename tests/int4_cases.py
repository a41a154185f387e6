"""One request of the 4-bit cache as tests set it up: appended without rotation,
attended by the decode, with the values held for an expectation."""

from __future__ import annotations

import torch

from oracle import int4_oracle as I
from pagegauge_b200.int4 import Int4PagePool
from pagegauge_b200.runtime import load_append_extension, read_device_error
from pagegauge_b200.wrapper import make_int4_wrapper, plan


class Held:
    """Query rows [1, Hq, 128] and tokens [n, Hkv, 128], on pages in a random order."""

    def __init__(self, q, k, v, hkv, seed):
        n = k.shape[0]
        pages = -(-n // 16)
        self.q, self.hkv, self.n = q.cuda(), hkv, n
        self.pool = Int4PagePool(pages, hkv)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
        at = torch.arange(n, dtype=torch.int32)
        slots = (order[(at // 16).long()] * 16 + at % 16).int().cuda()
        cos, sin = torch.ones(1, 64, device="cuda"), torch.zeros(1, 64, device="cuda")
        dummy = torch.zeros(n, 1, 128, dtype=k.dtype, device="cuda")
        load_append_extension().rope_append_int4(
            dummy, k.cuda(), v.cuda(), cos, sin, torch.zeros(n, dtype=torch.int32, device="cuda"),
            slots, dummy, self.pool.records)
        self.wrapper = make_int4_wrapper(workspace=torch.empty(64 << 20, dtype=torch.uint8,
                                                               device="cuda"))
        plan(self.wrapper, torch.tensor([0, pages], dtype=torch.int32), order.cuda(),
             torch.tensor([(n - 1) % 16 + 1], dtype=torch.int32, device="cuda"), torch.uint8,
             num_qo_heads=q.shape[1], num_kv_heads=hkv)
        self.order = order.long()

    def run(self):
        out, lse = self.wrapper.run(self.q, self.pool, return_lse=True)
        assert read_device_error() == 0
        return out[0].double().cpu().numpy(), lse[0].double().cpu().numpy()

    def held(self, h):
        """Key (z - 8) s and m, value (z - 8) s and m of KV head h, [n, 128] each."""
        records = self.pool.records[self.order.cuda(), h].cpu().numpy()
        (ka, km), (va, vm) = I.load(records)
        return [x.reshape(-1, 128)[:self.n] for x in (ka, km, va, vm)]

    def value_scales(self, h):
        """Value scale of every dim of KV head h, [n, 128]."""
        meta = self.pool.records[self.order.cuda(), h, 2304:].contiguous().view(torch.float16)
        s = meta.double().cpu().numpy().reshape(-1, 16, 2, 4)[:, :, 0].reshape(-1, 4)
        return s.repeat(32, axis=-1)[:self.n]
