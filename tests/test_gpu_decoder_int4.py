"""The decoder on the 4-bit cache, at the benchmark decoder's layer shape
(hidden 4096, 32 query / 8 KV heads, FFN 14336, vocab 32768; two layers).

At every layer of every eager step the 4-bit decode is compared with FP32
torch attention over the values read back from the pool (max-abs 2e-3, cosine
>= 0.9999, the bar of tests/test_gpu_decoder_attention.py), and the appended
token with the layer's own rotated, centred key and value: within half a
step of its group's scale (plus the roundings of the scale and midpoint).
Graph steps must equal the eager ones bit for bit."""

from __future__ import annotations

import math

import pytest
import torch

from pagegauge_b200.decoder import DecoderConfig, PageGaugeDecoder, random_decoder_weights
from pagegauge_b200.rotary import apply_rotary
from pagegauge_b200.runtime import read_device_error

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(layers=2, hidden=4096, heads=32, kv_heads=8, intermediate=14336,
                    vocab=32768)
SMALL = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=1, intermediate=1024, vocab=512)


class Checked:
    """Runs the 4-bit decode and compares it with torch on the same call."""

    def __init__(self, decoder, real, record):
        self.decoder, self.real, self.record = decoder, real, record

    def __getattr__(self, name):
        return getattr(self.real, name)

    def run(self, q, pool, value_center=None, out=None):
        self.real.run(q, pool, value_center=value_center, out=out)
        d = self.decoder
        group = q.shape[1] // pool.kv_heads
        kv_of_q = torch.arange(q.shape[1], device=q.device) // group
        for r, p in enumerate(int(x) for x in d.host_positions):
            slots = torch.arange(p + 1, dtype=torch.int32, device=q.device) + r * d.max_context
            k, v = pool.read(slots, dtype=torch.float32)
            s = torch.einsum("hd,thd->ht", q[r].float(), k[:, kv_of_q]) / math.sqrt(128)
            o = torch.einsum("ht,thd->hd", torch.softmax(s, dim=1), v[:, kv_of_q])
            exp = (o + value_center[r].float()[kv_of_q]).half().float()
            got = out[r].float()
            self.record.append((float((got - exp).abs().max()),
                                float(torch.nn.functional.cosine_similarity(
                                    got.flatten(), exp.flatten(), dim=0))))
        return out


def checked(dec, record):
    entry = dec._entry

    def wrapped(positions):
        e = entry(positions)
        if not isinstance(e["dec"], Checked):
            e["dec"] = Checked(dec, e["dec"], record)
        return e

    dec._entry = wrapped


@pytest.mark.parametrize("cfg,batch,prompt_len,gemm", [(CFG, 2, 4090, "auto"),
                                                       (SMALL, 3, 31, "cublas"),
                                                       (SMALL, 1, 16, "pg")])
def test_attention_and_graphs(cuda_lib, cfg, batch, prompt_len, gemm):
    weights = random_decoder_weights(cfg, 20261004, device="cuda")
    prompt = torch.randint(0, cfg.vocab, (batch, prompt_len),
                           generator=torch.Generator().manual_seed(41)).cuda()
    a, b = (PageGaugeDecoder(weights, batch=batch, max_context=prompt_len + 48, gemm=gemm,
                             kv_cache="int4") for _ in range(2))
    la, lb = a.prefill(prompt), b.prefill(prompt)
    assert torch.equal(la, lb)
    record: list = []
    checked(a, record)
    steps = 20  # crosses a page
    for i in range(steps):
        a.step(use_graph=False)
        b.step(use_graph=True)
        assert torch.equal(a.logits, b.logits) and torch.equal(a.tokens, b.tokens), i
    assert len(record) == steps * cfg.layers * batch
    assert max(e for e, _ in record) <= 2e-3 and min(c for _, c in record) >= 0.9999
    assert int(a.positions[0]) == prompt_len + steps
    assert a.slots.tolist() == [r * a.max_context + prompt_len + steps for r in range(batch)]
    assert b.replans >= 2 and read_device_error() == 0
    assert b.launches_per_step() == a.launches_per_step() > 0


def test_prompt_pages_hold_the_rotated_centred_rows(cuda_lib):
    weights = random_decoder_weights(SMALL, 5, device="cuda")
    prompt = torch.randint(0, SMALL.vocab, (2, 77), generator=torch.Generator().manual_seed(2))
    dec = PageGaugeDecoder(weights, batch=2, max_context=128, kv_cache="int4")
    dec.prefill(prompt.cuda())
    at = torch.arange(77, dtype=torch.int32, device="cuda")
    for r in range(2):
        # Layer 0's rows, recomputed from the embedding.
        h = weights.embed[prompt[r].cuda()].contiguous()
        x = torch.empty_like(h)
        dec._norm(h, None, weights.layers[0].attn_norm, x)
        qkv = torch.matmul(x, weights.layers[0].qkv.t())
        k = qkv[:, 512:640].view(77, 1, 128)
        v = qkv[:, 640:].view(77, 1, 128)
        rk, _ = apply_rotary(k, None, dec.cos, dec.sin, at)
        key, value = dec.pools[0].read(at + r * dec.max_context, dtype=torch.float32)
        for got, rows, c in ((key, rk, dec.centers[0][0, r]), (value, v, dec.centers[0][1, r])):
            assert torch.equal(c, rows.float().mean(0).half())
            exp = rows.float() - c.float()
            spread = exp.unflatten(-1, (4, 32))
            step = (spread.amax(-1) - spread.amin(-1)) / 15
            # half a step, the FP16 roundings of the scale (15 steps of it) and
            # the midpoint, and of the rotated key compared with
            bound = step * (0.5 + 15 * 2 ** -11) + spread.abs().amax(-1) * 2 ** -10 + 2 ** -13
            err = (got - exp).abs().unflatten(-1, (4, 32)).amax(-1)
            assert (err <= bound).all()


def test_close_to_the_page_gauge_decoder(cuda_lib):
    """Same weights and prompt: prefills differ by the rotation's rounding
    alone (FP32 against FP16 steps), decode steps by the caches' precision."""
    weights = random_decoder_weights(SMALL, 6, device="cuda")
    prompt = torch.randint(0, SMALL.vocab, (2, 200),
                           generator=torch.Generator().manual_seed(3)).cuda()
    a = PageGaugeDecoder(weights, batch=2, max_context=512)
    b = PageGaugeDecoder(weights, batch=2, max_context=512, kv_cache="int4")
    la, lb = a.prefill(prompt).float(), b.prefill(prompt).float()
    cos = torch.nn.functional.cosine_similarity
    assert float(cos(la.flatten(), lb.flatten(), dim=0)) >= 0.9999
    b.tokens.copy_(a.tokens)
    a.step(use_graph=False)
    b.step(use_graph=False)
    assert float(cos(a.logits.float().flatten(), b.logits.float().flatten(), dim=0)) >= 0.99


def test_refusals(cuda_lib):
    weights = random_decoder_weights(SMALL, 7, device="cuda")
    for kw in (dict(kv_cache="int2"), dict(kv_cache="int4", sink_pages=1),
               dict(kv_cache="int4", ring_pages=4), dict(kv_cache="int4", suffix_pages=1)):
        with pytest.raises(ValueError):
            PageGaugeDecoder(weights, batch=1, max_context=64, **kw)


def test_steps_without_a_prompt(cuda_lib):
    """Decoding from an empty cache: every request appends to its own pages, so
    each follows a decoder that runs it alone.  Their logits differ by the FP16
    roundings of the projections' sums alone."""
    weights = random_decoder_weights(SMALL, 8, device="cuda")
    first = torch.tensor([3, 77, 400], device="cuda")
    alone = []
    steps = 18  # crosses a page
    feed = torch.randint(0, SMALL.vocab, (steps, 3),
                         generator=torch.Generator().manual_seed(9)).cuda()
    feed[0] = first
    for batch in (slice(0, 3), slice(0, 1), slice(1, 2), slice(2, 3)):
        n = batch.stop - batch.start
        dec = PageGaugeDecoder(weights, batch=n, max_context=40, kv_cache="int4", gemm="cublas")
        logits = []
        for i in range(steps):
            dec.tokens.copy_(feed[i, batch])
            dec.step(use_graph=i > 2)
            logits.append(dec.logits.float().clone())
        assert dec.slots.tolist() == [r * dec.max_context + steps for r in range(n)]
        # Every request's pages hold its tokens.
        for r in range(n):
            at = torch.arange(steps, dtype=torch.int32, device="cuda") + r * dec.max_context
            key, value = dec.pools[0].read(at, dtype=torch.float32)
            assert (key.abs().amax((1, 2)) > 0).all() and (value.abs().amax((1, 2)) > 0).all()
        alone.append(torch.stack(logits, 1))
    together, single = alone[0], torch.cat(alone[1:])
    cos = torch.nn.functional.cosine_similarity(together, single, dim=-1)
    assert float(cos.min()) >= 0.999 and read_device_error() == 0
