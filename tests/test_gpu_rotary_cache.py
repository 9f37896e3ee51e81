"""GPU: the paged cache with rotary positions and masked attention, as a model's layers use it: prompt chunks, decode and verify
steps, eager and captured, each step's stored keys and outputs against the float64 oracles over all rows written so far.

Tolerances: the pools as in test_gpu_rotary.py (half a step of the codes, and the rotation's 24 * 2^-24); the output against the
oracle over the pool's own values and the float64 rotation of q, rounded to q's type by the kernel (half a step of q moves a score
by at most |scale| sum |q k| eps / 2, a weight by twice that), as in test_gpu_masked_attention.py beyond.
"""

import numpy as np
import pytest
import torch

from bpt_amd import PagedQuantKVCache
from oracle import masked as omask
from oracle import rotary as orot

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV, D = 8, 2, 128
SCALE = D**-0.5
DTYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "bf16": torch.bfloat16}
MASKS = {
    "none": None,
    "cap and window": dict(softcap=20.0, window=37),
    "bias and prefix": lambda b: dict(slopes=2.0 ** -torch.arange(1, HQ + 1, device=DEV, dtype=torch.float32),
                                      prefix_lens=torch.full((b,), 9, dtype=torch.int32, device=DEV), max_prefix=9),
}


def rows(g, b, h, n):
    return torch.randn((b, h, n, D), generator=g, device=DEV).to(torch.bfloat16)


class Model:
    """One layer's cache, its rotary set-up, and every sequence's rows in float64."""

    def __init__(self, fmt, axes):
        kw = dict(k_scale=torch.full((1, HKV), 0.05), v_scale=torch.full((1, HKV), 0.02)) if fmt == "fp8" else {}
        self.cache = PagedQuantKVCache(num_layers=1, num_kv_heads=HKV, head_dim=D, num_blocks=64, block_size=16, kv_dtype=DTYPES[fmt],
                                       device=DEV, **kw)
        self.fmt, self.axes = fmt, axes
        self.inv_freq = (1e4 ** (-torch.arange(48, dtype=torch.float64) / 48)).float().to(DEV)  # 96 of 128 channels
        self.sections = None if axes == 1 else (20, 14, 14)
        self.which = [0] * 48 if axes == 1 else [0] * 20 + [1] * 14 + [2] * 14
        g = torch.Generator(device=DEV).manual_seed(99)
        self.q_norm, self.k_norm = (1 + 0.1 * torch.randn((2, D), generator=g, device=DEV)).to(torch.bfloat16)
        self.keys, self.values = {}, {}

    def positions(self, pos):
        return pos if self.axes == 1 else torch.stack([pos, pos // 3 + 5, pos % 7])

    def rotary(self, pos):
        return dict(positions=self.positions(pos), inv_freq=self.inv_freq, sections=self.sections, q_norm=self.q_norm, k_norm=self.k_norm)

    def rotated(self, x, pos, weight):  # [B, H, Q, D] -> float64 [B, Q, H, D]
        p = self.positions(pos).cpu().numpy().reshape(self.axes, *pos.shape)
        x = x.transpose(1, 2).double().cpu().numpy()
        return orot.rotate(x, p, self.inv_freq.cpu().numpy(), self.which, weight=weight.double().cpu().numpy()), x

    def pool(self):
        out = []
        for codes, scale in ((self.cache.k[0], self.cache.k_scale[0]), (self.cache.v[0], self.cache.v_scale[0])):
            x = codes.float().double()
            if self.fmt == "fp8":
                x = x * scale.double()[:, None]
            elif self.fmt == "int8":
                x = x * scale.double()[..., None]
            out.append(x.cpu().numpy())
        return out

    def check(self, seqs, pos, q, k, v, out, mask):
        b, n = pos.shape
        want_k, raw_k = self.rotated(k, pos, self.k_norm)
        spread = orot.spread(raw_k, self.inv_freq.cpu().numpy(), weight=self.k_norm.double().cpu().numpy())
        pool_k, pool_v = self.pool()
        for i, s in enumerate(seqs):
            for j in range(n):
                p = int(pos[i, j])
                page, off = self.cache.tables[s][p // 16], p % 16
                for got, want, size in ((pool_k[page, off], want_k[i, j], spread[i, j]),
                                        (pool_v[page, off], v[i, :, j].double().cpu().numpy(), np.abs(v[i, :, j].double().cpu().numpy()))):
                    if self.fmt == "bf16":
                        half = 2.0**-8 * np.abs(want)
                    elif self.fmt == "fp8":
                        half = np.maximum(2.0**-4 * np.abs(want), 2.0**-10 * 0.05)
                    else:
                        half = 0.5 * np.abs(want).max(-1, keepdims=True) / 127 * (1 + 2.0**-10)
                    assert (np.abs(got - want) <= half * (1 + 2.0**-10) + 24 * 2.0**-24 * size + 2.0**-20 * np.abs(want)).all()
        want_q, _ = self.rotated(q, pos, self.q_norm)
        lens = (pos[:, -1] + 1).cpu().numpy()
        tables = [self.cache.tables[s] for s in seqs]
        how = {n_: t.cpu().numpy() if torch.is_tensor(t) else t for n_, t in (mask or {}).items() if n_ != "max_prefix"}
        how["prefix"] = how.pop("prefix_lens", None)
        want, _, mean, slack = omask.attend(want_q, pool_k, pool_v, tables, lens, SCALE, **how)
        # Half a step of q's rounding: of the largest sum of |q k|, which 130 * 2^-24 of is part of the slack.
        slack = slack * (1 + 2.0**-8 / (130 * 2.0**-24))
        got = out.transpose(1, 2).double().cpu().numpy()
        bound = (2 * slack + 2.0**-15)[..., None] * mean * 1.01 + 2.0**-8 * np.abs(want) + 2.0**-25
        assert (np.abs(got - want) <= bound).all(), f"{(np.abs(got - want) - bound).max():.3e} over the bound"


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("fmt, axes", [("fp8", 1), ("int8", 3), ("bf16", 1), ("fp8", 3)])
def test_chunks_decode_and_verify(fmt, axes, mask):
    m, g = Model(fmt, axes), torch.Generator(device=DEV).manual_seed(7)
    seqs, lens = ["a", "b", "c"], [70, 33, 1]
    of = (lambda b: MASKS[mask](b)) if callable(MASKS[mask]) else (lambda b: MASKS[mask])

    def step(which, pos):
        q, k, v = rows(g, len(which), HQ, pos.shape[1]), rows(g, len(which), HKV, pos.shape[1]), rows(g, len(which), HKV, pos.shape[1])
        meta = m.cache.prepare(which, pos)
        out = m.cache.attend(0, q, k, v, meta, SCALE, rotary=m.rotary(pos), mask=of(len(which)))
        torch.cuda.synchronize()
        m.check(which, pos, q, k, v, out, of(len(which)))

    for s, n in zip(seqs, lens):  # prompts in two chunks
        m.cache.reserve(s, 120)
        for lo, hi in ((0, n // 2), (n // 2, n)):
            if hi > lo:
                step([s], torch.arange(lo, hi, device=DEV, dtype=torch.int32)[None])
    at = torch.tensor(lens, device=DEV, dtype=torch.int32)
    for _ in range(2):  # decode
        step(seqs, at[:, None])
        at = at + 1
    step(seqs, at[:, None] + torch.arange(4, device=DEV, dtype=torch.int32))  # verify


def test_masks_without_rotation_and_rotation_without_masks_agree_with_the_single_calls():
    from bpt_amd import paged_decode_attention, paged_masked_attention, quantize_append, rotary_append

    for mask in (dict(softcap=5.0), None):
        g = torch.Generator(device=DEV).manual_seed(3)
        one, two = Model("int8", 1), Model("int8", 1)
        pos = torch.arange(0, 21, device=DEV, dtype=torch.int32)[None]
        q, k, v = rows(g, 1, HQ, 21), rows(g, 1, HKV, 21), rows(g, 1, HKV, 21)
        for m in (one, two):
            m.cache.reserve("s", 40)
        meta = one.cache.prepare(["s"], pos)
        rotary = None if mask else one.rotary(pos)
        got = one.cache.attend(0, q, k, v, meta, SCALE, rotary=rotary, mask=mask)
        c = two.cache
        pools, slots = (c.k[0], c.v[0], c.k_scale[0], c.v_scale[0]), (meta.write_blocks, meta.write_offsets)
        qt, kt, vt = (x.transpose(1, 2) for x in (q, k, v))
        if mask:
            quantize_append(kt, vt, *pools, *slots)
            want = paged_masked_attention(qt, *pools[:2], meta.block_table, meta.context_lens, *pools[2:], scale=SCALE,
                                          max_context=meta.kv_len, **mask)
        else:
            turned = rotary_append(qt, kt, vt, pos, one.inv_freq, *pools, *slots, q_norm=one.q_norm, k_norm=one.k_norm)
            want = paged_decode_attention(turned, *pools[:2], meta.block_table, meta.context_lens, *pools[2:], scale=SCALE,
                                          max_context=meta.kv_len)
        assert torch.equal(got, want.transpose(1, 2))
        assert torch.equal(one.cache.k[0], c.k[0]) and torch.equal(one.cache.v_scale[0], c.v_scale[0])


def test_a_captured_step_replays():
    """prepare and attend with rotation and mask in one graph, replayed over a few steps against the eager calls on a second cache."""
    g = torch.Generator(device=DEV).manual_seed(5)
    one, two = Model("fp8", 3), Model("fp8", 3)
    seqs = ["a", "b"]
    for m in (one, two):
        for s in seqs:
            m.cache.reserve(s, 100)
    mask = dict(softcap=9.0, window=30)
    pos = torch.tensor([[0], [0]], device=DEV, dtype=torch.int32)
    axes = one.positions(pos).clone()
    q, k, v = rows(g, 2, HQ, 1), rows(g, 2, HKV, 1), rows(g, 2, HKV, 1)

    def step(m):
        how = {**m.rotary(pos), "positions": axes}
        return m.cache.attend(0, q, k, v, m.cache.prepare(seqs, pos), SCALE, rotary=how, mask=mask)

    step(two)  # the second cache's warm-up, overwritten by its first step
    step(one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(one)
    for i in range(40):
        pos.copy_(torch.tensor([[i], [i + 20]], device=DEV))
        axes.copy_(one.positions(pos))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV).to(x.dtype))
        graph.replay()
        want = step(two)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    assert torch.equal(one.cache.k[0].view(torch.uint8), two.cache.k[0].view(torch.uint8))


def test_a_refused_step_stores_nothing():
    m, g = Model("bf16", 1), torch.Generator(device=DEV).manual_seed(5)
    m.cache.reserve("s", 40)
    pos = torch.arange(0, 3, device=DEV, dtype=torch.int32)[None]
    q, k, v = rows(g, 1, HQ, 3), rows(g, 1, HKV, 3), rows(g, 1, HKV, 3)
    meta = m.cache.prepare(["s"], pos)
    for bad in (dict(mask=dict(softcap=-1.0)), dict(mask=dict(window=0), rotary=m.rotary(pos)), dict(rotary=m.rotary(pos), mask=dict(softcap=1e-45)),
                dict(rotary={**m.rotary(pos), "sections": (1, 2)}), dict(rotary=m.rotary(pos), scale=float("nan")),
                dict(mask=dict(softcap=2.0), scale=float("nan"))):
        with pytest.raises(ValueError):
            m.cache.attend(0, q, k, v, meta, **{"scale": SCALE, **bad})
    with pytest.raises(ValueError, match="bf16 or f16"):
        m.cache.attend(0, q.float(), k.float(), v.float(), meta, SCALE, mask=dict(window=3))
    torch.cuda.synchronize()
    assert not m.cache.k[0].any() and not m.cache.v[0].any()
