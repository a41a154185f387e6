"""The tensor-parallel form of the decoder on the 4-bit cache, as far as one GPU
shows it: a rank's pools and attention hold its own KV heads, and a decoder with a
process group (of one rank) follows the one without."""

from __future__ import annotations

import datetime
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from pagegauge_b200.decoder import (DecoderConfig, PageGaugeDecoder, TensorParallel,
                                    random_decoder_weights)
from pagegauge_b200.runtime import read_device_error

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(layers=2, hidden=512, heads=8, kv_heads=2, intermediate=1024, vocab=512)


def test_ranks_hold_their_heads(cuda_lib):
    """Layer 0 of a prompt, whose input no rank's partial sums change: the pools of two
    ranks' shards side by side are the whole model's, up to FP16 roundings of the
    projection (sums of 512 products in another order: 2^-9 of a row's largest value
    and half a step of the 4-bit group more)."""
    prompt = torch.randint(0, CFG.vocab, (2, 70), generator=torch.Generator().manual_seed(3))
    at = torch.arange(70, dtype=torch.int32, device="cuda")

    def held(tp):
        w = random_decoder_weights(CFG, 43, device="cuda", gen_device="cpu", tp=tp)
        dec = PageGaugeDecoder(w, batch=2, max_context=96, gemm="cublas", kv_cache="int4")
        dec.prefill(prompt.cuda())
        out = []
        for r in range(2):
            rows = dec.pools[0].read(at + r * dec.max_context, dtype=torch.float32)
            out.append([x + c[r].float() for x, c in zip(rows, dec.centers[0])])
        return out

    whole = held(TensorParallel.of(CFG, 0, 1))
    parts = [held(TensorParallel.of(CFG, rank, 2)) for rank in range(2)]
    for r in range(2):
        for kind in range(2):
            both = torch.cat([p[r][kind] for p in parts], 1)
            exp = whole[r][kind]
            assert both.shape == exp.shape == (70, 2, 128)
            spread = exp.unflatten(-1, (4, 32))
            step = (spread.amax(-1) - spread.amin(-1)) / 15
            bound = 1.5 * step + 2 ** -8 * spread.abs().amax(-1) + 2 ** -10
            assert ((both - exp).abs().unflatten(-1, (4, 32)).amax(-1) <= bound).all()
            # The heads are different ones, so that an exchange of them would show.
            assert (exp[:, 0] - exp[:, 1]).abs().mean() > 4 * (both - exp).abs().mean()
    assert read_device_error() == 0


def _one_rank(rank, port):
    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.cuda.set_device(0)
    dist.init_process_group("nccl", rank=0, world_size=1,
                            timeout=datetime.timedelta(seconds=60),
                            device_id=torch.device("cuda", 0))
    try:
        w = random_decoder_weights(CFG, 44, device="cuda", gen_device="cpu")
        prompt = torch.randint(0, CFG.vocab, (2, 30),
                               generator=torch.Generator().manual_seed(4)).cuda()
        alone = PageGaugeDecoder(w, batch=2, max_context=64, gemm="cublas", kv_cache="int4")
        grouped = PageGaugeDecoder(w, batch=2, max_context=64, gemm="cublas", kv_cache="int4",
                                   process_group=dist.group.WORLD, tp_reduce="nccl")
        assert torch.equal(alone.prefill(prompt), grouped.prefill(prompt))
        for i in range(6):  # crosses a page, eager and captured
            grouped.tokens.copy_(alone.tokens)
            alone.step(use_graph=i > 1)
            grouped.step(use_graph=i > 1)
            a, b = alone.logits.float(), grouped.logits.float()
            assert float(torch.nn.functional.cosine_similarity(a, b, dim=-1).min()) >= 0.9999, i
            assert torch.equal(alone.slots, grouped.slots)
        assert read_device_error() == 0
        torch.cuda.synchronize()
        grouped.close()
        del grouped
    finally:
        dist.destroy_process_group()


def test_a_process_group_of_one(cuda_lib):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_one_rank, args=(port,), nprocs=1, join=True)
