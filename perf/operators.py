"""Measured operators: rotary positions on their way into a paged KV cache, and masked attention over it.

Three operators, each in a plain form (torch operations in 32 bits) and as this framework's entry point:

  embed    `rotary_embed`: queries and keys normalised per head (optional) and rotated by their positions on one or
           several axes (text: one; images: height and width; video: time, height and width)
  append   `rotary_append`: the same rotation of a step's new queries and keys, the keys and values quantized into
           their slots of the paged cache on the way
  attend   `paged_masked_attention`: attention over the paged cache with scores capped by a tanh, a bias that falls with
           distance, a sliding window, a prefix that every query sees and documents that do not see one another

Lengths, positions' ranges and masks come from the case alone, values from the seed. Caches hold what serving puts
there: keys with a few outlier channels, quantized with the formulas of their format, pages scattered over a pool.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
_FLOATS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_PACKAGE = str(Path(__file__).resolve().parent.parent / "bytes-per-token_amd")


# ---- the cases ----------------------------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # One decode step's queries and keys of a small batch: the smallest call, where latency counts.
        _embed("embed bf16 8x1", 8, 1, norm=True),
        # The patches of a few images on their way through a vision encoder: two axes, heads of 80 channels, no cache.
        _embed("embed bf16 4x4097 images", 4, 4097, hq=16, hkv=16, d=80, axes=2),
        # A serving batch's decode step: per-head norm, rotation and FP8 store of 32 new tokens.
        _append("append fp8 32x1", "fp8", 32, 1, norm=True),
        # A speculative verify of five tokens per sequence into a BF16 cache, pairs of neighbouring channels.
        _append("append bf16 64x5", "bf16", 64, 5, interleaved=True),
        # A prompt chunk with video in it: three axes, INT8 with a scale per token and head.
        _append("append int8 1x2048 video", "int8", 1, 2048, hq=32, axes=3, norm=True),
        # The largest prompt chunk of a batch into an FP8 cache, half of the channels rotated.
        _append("append fp8 4x4096", "fp8", 4, 4096, hq=32, rot=64),
        # One short chat on an unquantized cache with capped scores: latency counts.
        _attend("attend bf16 1x512 cap", "bf16", 1, 1, 512, 512, cap=50.0),
        # A serving batch in the middle of its conversations: ragged lengths, capped scores, FP8 with per-head scales.
        _attend("attend fp8 32x256-4096 cap", "fp8", 32, 1, 256, 4096, cap=30.0),
        # Long conversations on an INT8 cache with a bias that falls with distance.
        _attend("attend int8 16x1000-9001 bias", "int8", 16, 1, 1000, 9001, hq=32, bias=True),
        # Long documents read through a window of 4096 tokens and 64 first tokens that stay visible.
        _attend("attend fp8 8x32768 window", "fp8", 8, 1, 32768, 32768, hq=32, window=4096, prefix=64),
        # A verify of several queries over packed documents behind a prefix that all of them see.
        _attend("attend fp8 16x5 documents", "fp8", 16, 5, 1024, 2900, hq=32, prefix=300, docs=3),
        # A long prompt's chunk: 2048 new tokens on 2049 cached ones, capped scores, a window.
        _attend("attend bf16 2048+2049 cap", "bf16", 1, 2048, 4097, 4097, cap=50.0, window=2500),
    ]


def _embed(name, batch, queries, hq=16, hkv=8, d=128, rot=0, axes=1, cyclic=False, interleaved=False, norm=False,
           q="bf16", far=4096):
    return {"name": name, "kind": "embed", "batch": batch, "queries": queries, "hq": hq, "hkv": hkv, "d": d, "rot": rot or d,
            "axes": axes, "cyclic": cyclic, "interleaved": interleaved, "norm": norm, "q": q, "far": far}


def _append(name, fmt, batch, queries, page=16, **more):
    return {**_embed(name, batch, queries, **more), "kind": "append", "fmt": fmt, "page": page}


def _attend(name, fmt, batch, queries, lo, hi, hq=16, hkv=8, cap=0.0, bias=False, window=0, prefix=0, docs=0, q="bf16",
            page=16):
    return {"name": name, "kind": "attend", "fmt": fmt, "batch": batch, "queries": queries, "lo": lo, "hi": hi, "hq": hq,
            "hkv": hkv, "cap": cap, "bias": bias, "window": window, "prefix": prefix, "docs": docs, "q": q, "page": page}


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    """One more case of the listed kinds, over their whole ranges, and no dearer than the dearest listed one."""
    top = [(c["kind"], _cost(c)) for c in listed()]
    while True:
        case = _draw_any(rng)
        most = [cost for kind, cost in top if kind == case["kind"]]
        if all(x <= max(of) for x, of in zip(_cost(case), zip(*most))):
            return case


def _cost(c: dict) -> tuple[float, ...]:
    """Bytes and operations, the cache's tokens and the pairs of a query and a token, seen or not."""
    w = work(c)
    if c["kind"] != "attend":
        return w["bytes"], w["flops"]
    return w["bytes"], w["flops"], c["batch"] * c["hi"] * c["hkv"], c["batch"] * c["hi"] * c["queries"] * c["hq"]


def _draw_any(rng: random.Random) -> dict:
    kind = rng.choice(["embed", "append", "append", "attend", "attend", "attend"])
    hq, hkv = rng.choice([(16, 8), (16, 8), (32, 8), (32, 8), (64, 8), (8, 8), (12, 4), (5, 1), (9, 3)])
    fmt = rng.choice(["fp8", "fp8", "int8", "bf16"])
    q = rng.choice(["bf16", "bf16", "bf16", "f16"])
    if kind == "attend":
        queries = rng.choice([1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 2048)])
        hi = _log_int(rng, max(queries, 16), 32768)
        lo = hi if rng.random() < 0.25 else _log_int(rng, max(queries, hi // 16, 1), hi)
        case = _attend("", fmt, _log_int(rng, 1, 96 if queries < 10 else 4), queries, lo, hi, hq=hq, hkv=hkv, q=q,
                       page=rng.choice([16, 16, 32, 64]))
        for what in rng.sample(["cap", "bias", "window", "prefix", "docs"], rng.randint(1, 3)):
            case[what] = {"cap": rng.choice([5.0, 20.0, 30.0, 50.0]), "bias": True, "window": _log_int(rng, 1, hi),
                          "prefix": _log_int(rng, 1, hi), "docs": rng.randint(2, 9)}[what]
    else:
        d = rng.choice([128, 128, 128, 64, 256])
        if kind == "embed":
            d = rng.choice([d, 80, 96, 72])
        axes = rng.choice([1, 1, 2, 3])
        more = dict(hq=hq, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2]), axes=axes, cyclic=axes > 1 and rng.random() < 0.5,
                    interleaved=rng.random() < 0.3, norm=rng.random() < 0.5, far=_log_int(rng, 4096, 1 << 20))
        batch = _log_int(rng, 1, 128)
        queries = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
        if kind == "embed":
            case = _embed("", batch, queries, q=rng.choice([q, q, "f32"]), **more)
        else:
            case = _append("", fmt, batch, queries, q=q, page=rng.choice([16, 16, 32]), **more)
    case.pop("name")
    return case


# ---- lengths, masks and sizes, from the case alone ---------------------------------------------------------


def _lengths(c: dict) -> np.ndarray:
    """Tokens of each sequence, the new ones included: spread evenly from lo to hi, neighbours in the batch unlike."""
    b = c["batch"]
    lens = np.linspace(c["lo"], c["hi"], b).round().astype(np.int64) if b > 1 else np.array([c["hi"]], dtype=np.int64)
    return lens[(np.arange(b) * 7 + 3) % b] if b % 7 else lens


def _masks(c: dict) -> dict:
    """Each sequence's length, prefix and each query's position and first token behind the prefix, as numpy arrays."""
    lens = _lengths(c)
    pos = lens[:, None] - c["queries"] + np.arange(c["queries"])[None, :]
    prefix = np.zeros_like(lens) if not c["prefix"] else np.maximum(1, c["prefix"] * (1 + np.arange(len(lens))) // len(lens))
    starts = np.zeros_like(pos)
    if c["docs"]:  # equally long documents: a query's first token is its own document's
        size = np.maximum(1, -(-lens // c["docs"]))[:, None]
        starts = np.maximum(pos, 0) // size * size
    return {"lens": lens, "pos": pos, "prefix": np.minimum(prefix, lens), "starts": starts}


def _seen(c: dict) -> tuple[int, int]:
    """(tokens that some query of their sequence sees, pairs of a query and a token that it sees)."""
    m = _masks(c)
    lo = m["starts"] if not c["window"] else np.maximum(m["starts"], m["pos"] - c["window"] + 1)
    lo, hi, prefix = np.maximum(lo, m["prefix"][:, None]), m["pos"] + 1, m["prefix"]  # the prefix, and what is behind it
    pairs = prefix[:, None] + np.maximum(hi - lo, 0)
    tokens = prefix + np.maximum(hi.max(1) - lo.min(1), 0)
    return int(tokens.sum()), int(pairs.sum())


def work(case: dict) -> dict:
    c, elem = case, 4 if case["q"] == "f32" else 2
    if c["kind"] == "attend":
        tokens, pairs = _seen(c)
        per = c["hkv"] * 2 * (128 * (2 if c["fmt"] == "bf16" else 1) + (4 if c["fmt"] == "int8" else 0))
        rows = c["batch"] * c["queries"] * c["hq"]
        return {"bytes": tokens * per + rows * 128 * 2 * elem, "flops": pairs * c["hq"] * 128 * 4}
    tokens = c["batch"] * c["queries"]
    moved = tokens * c["d"] * elem * (2 * c["hq"] + (2 if c["kind"] == "embed" else 1) * c["hkv"])
    if c["kind"] == "append":
        moved += tokens * c["hkv"] * (c["d"] * elem + 2 * c["d"] * (2 if c["fmt"] == "bf16" else 1) + (8 if c["fmt"] == "int8" else 0))
    return {"bytes": moved + tokens * 4 * c["axes"], "flops": tokens * (c["hq"] + c["hkv"]) * (3 * c["rot"] + (4 * c["d"] if c["norm"] else 0))}


# ---- inputs --------------------------------------------------------------------------------------------------


def _sections(c: dict) -> tuple[int, ...] | None:
    """How many of the rotated pairs follow each axis: as even as they go, the first axis the most."""
    if c["axes"] == 1:
        return None
    half, n = c["rot"] // 2, c["axes"]
    rest = [half // (n + 1) if n == 3 else half // 2] * (n - 1)
    return (half - sum(rest), *rest)


def _random(g, shape, dtype=torch.float32, amp=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * amp).to(dtype)


def _rows(g, b, n, h, d, dtype):
    """Keys of a projection: a few channels are larger than the others."""
    x = torch.randn((b, n, h, d), generator=g, device=DEV)
    x[..., :: d // 4] *= 6.0
    return x.to(dtype)


def _quantized(x, fmt):
    """A pool [..., Hkv, D] of float values in its format, and its scales."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    if fmt == "fp8":
        scale = (x.abs().amax(dim=(0, 1, 3)) / 448).contiguous()
        return (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale
    scale = (x.abs().amax(dim=-1) / 127).clamp_min(1e-12)
    return (x / scale[..., None]).round().clamp(-128, 127).to(torch.int8), scale.contiguous()


def prepare(case: dict, seed: int) -> dict:
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    b, n, hq, hkv, dtype = c["batch"], c["queries"], c["hq"], c["hkv"], _FLOATS[c["q"]]
    s = dict(c)
    if c["kind"] == "attend":
        m, page = _masks(c), c["page"]
        per_seq = -(-int(m["lens"].max()) // page)
        blocks = [-(-int(t) // page) for t in m["lens"]]
        pool = sum(blocks) + max(8, sum(blocks) // 4)
        ids = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
        table, at = torch.zeros((b, per_seq), dtype=torch.int32, device=DEV), 0
        for i, k in enumerate(blocks):
            table[i, :k], at = ids[at : at + k], at + k
        s["k_cache"], s["k_scale"] = _quantized(_rows(g, pool, page, hkv, 128, torch.float32), c["fmt"])
        s["v_cache"], s["v_scale"] = _quantized(_random(g, (pool, page, hkv, 128)), c["fmt"])
        s |= {"query": _random(g, (b, n, hq, 128), dtype, 1.5), "block_table": table, "max_context": int(m["lens"].max()),
              "context_lens": torch.from_numpy(m["lens"]).to(DEV, torch.int32), "scale": 128**-0.5,
              "slopes": None, "prefix_lens": None, "starts": None}
        if c["bias"]:
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq)
        if c["prefix"]:
            s["prefix_lens"] = torch.from_numpy(m["prefix"]).to(DEV, torch.int32)
            s["max_prefix"] = int(m["prefix"].max())
        if c["docs"]:
            s["starts"] = torch.from_numpy(m["starts"]).to(DEV, torch.int32)
        return s
    d, rot = c["d"], c["rot"]
    base = torch.randint(0, c["far"], (b, 1), generator=g, device=DEV) + torch.arange(n, device=DEV)
    if c["axes"] == 1:
        positions = base
    else:  # a picture's rows and columns (and a film's frames before them), 64 wide, behind some text
        cell = torch.arange(n, device=DEV).expand(b, n)
        grid = [cell // 4096, cell // 64 % 64, cell % 64][3 - c["axes"] :]
        positions = torch.stack([base[:, :1] + x for x in grid])
    s |= {"query": _random(g, (b, n, hq, d), dtype), "key": _rows(g, b, n, hkv, d, dtype), "positions": positions.to(torch.int32).contiguous(),
          "inv_freq": (1e6 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)).float(),
          "sections": _sections(c), "q_norm": None, "k_norm": None}
    if c["norm"]:
        s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype), (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype)
    if c["kind"] == "append":  # the new tokens' slots in a pool with as much again in it
        page = c["page"]
        pool = -(-2 * b * n // page) + 1
        slots = torch.randperm(pool * page, generator=g, device=DEV)[: b * n].reshape(b, n)
        s["value"] = _random(g, (b, n, hkv, d), dtype)
        s["k_cache"], s["k_scale"] = _quantized(_rows(g, pool, page, hkv, d, torch.float32), c["fmt"])
        s["v_cache"], s["v_scale"] = _quantized(_random(g, (pool, page, hkv, d)), c["fmt"])
        s["write_blocks"], s["write_offsets"] = (slots // page).to(torch.int32), (slots % page).to(torch.int32)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return _run_own(state)
    return {"embed": _plain_embed, "append": _plain_append, "attend": _plain_attend}[state["kind"]](state)


def _run_own(s: dict):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import bpt_amd

    if s["kind"] == "attend":
        return bpt_amd.paged_masked_attention(
            s["query"], s["k_cache"], s["v_cache"], s["block_table"], s["context_lens"], s["k_scale"], s["v_scale"],
            scale=s["scale"], max_context=s["max_context"], softcap=s["cap"] or None, slopes=s["slopes"],
            window=s["window"] or None, prefix_lens=s["prefix_lens"], max_prefix=s.get("max_prefix"), starts=s["starts"],
            out_dtype=s["query"].dtype)
    how = dict(sections=s["sections"], cyclic=s["cyclic"], interleaved=s["interleaved"], q_norm=s["q_norm"],
               k_norm=s["k_norm"], eps=1e-6)
    if s["kind"] == "embed":
        return bpt_amd.rotary_embed(s["query"], s["key"], s["positions"], s["inv_freq"], **how)
    q = bpt_amd.rotary_append(s["query"], s["key"], s["value"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"],
                              s["k_scale"], s["v_scale"], s["write_blocks"], s["write_offsets"], **how)
    return q, *_pools(s)


def _pools(s: dict):
    """The pools as the values that they stand for (FP8 codes as they are: a type of values, under constant scales)."""
    if s["fmt"] != "int8":
        return s["k_cache"], s["v_cache"]
    return ((s["k_cache"] * s["k_scale"][..., None]).to(torch.bfloat16), (s["v_cache"] * s["v_scale"][..., None]).to(torch.bfloat16),
            s["k_scale"], s["v_scale"])


def _axis_of_pair(half: int, axes: int, sections, cyclic: bool) -> list[int]:
    """The axis that turns each pair of channels: in stretches of sections[a] pairs, or (cyclic) dealt out in turn, axis 0
    taking what the others leave."""
    if axes == 1:
        return [0] * half
    if not cyclic:
        return [a for a, k in enumerate(sections) for _ in range(k)]
    return [i % axes if i // axes < sections[i % axes] else 0 for i in range(half)]


def _plain_rotated(s: dict, x, weight):
    """x [B, Q, H, D] normalised per head and rotated, in 32 bits; angles in 64."""
    x, rot = x.float(), s["rot"]
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    pos = s["positions"].double()
    if s["axes"] > 1:
        pos = pos[_axis_of_pair(rot // 2, s["axes"], s["sections"], s["cyclic"])].permute(1, 2, 0)  # [B, Q, rot / 2]
    else:
        pos = pos[..., None]
    angle = (pos * s["inv_freq"].double())[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    if s["interleaved"]:
        x1, x2 = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1).flatten(-2)
    else:
        x1, x2 = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_embed(s: dict):
    return (_plain_rotated(s, s["query"], s["q_norm"]).to(s["query"].dtype), _plain_rotated(s, s["key"], s["k_norm"]).to(s["key"].dtype))


def _plain_append(s: dict):
    at = (s["write_blocks"].long(), s["write_offsets"].long())
    for what, x in (("k", _plain_rotated(s, s["key"], s["k_norm"])), ("v", s["value"].float())):
        cache, scale = s[what + "_cache"], s[what + "_scale"]
        if s["fmt"] == "bf16":
            cache[at] = x.to(torch.bfloat16)
        elif s["fmt"] == "fp8":
            cache.view(torch.uint8)[at] = (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            fresh = (x.abs().amax(-1) / 127).clamp_min(1e-12)
            cache[at] = (x / fresh[..., None]).round().clamp(-128, 127).to(torch.int8)
            scale[at] = fresh
    return _plain_rotated(s, s["query"], s["q_norm"]).to(s["query"].dtype), *_pools(s)


def _visible(s: dict, tokens):
    """[B, Q, T]: which of the tokens each query sees, and how far they are from it."""
    lens = s["context_lens"].long()[:, None, None]
    pos = lens - s["queries"] + torch.arange(s["queries"], device=DEV)[None, :, None]
    near = tokens <= pos
    if s["window"]:
        near &= pos - tokens < s["window"]
    if s["starts"] is not None:
        near &= tokens >= s["starts"].long()[:, :, None]
    if s["prefix_lens"] is not None:
        near = near | (tokens < s["prefix_lens"].long()[:, None, None])
    return near & (tokens < lens), (pos - tokens).abs()


def _plain_attend(s: dict):
    b, n, hq, d = s["query"].shape
    hkv, page, tokens = s["hkv"], s["page"], torch.arange(s["max_context"], device=DEV)
    blocks, offsets = s["block_table"].long()[:, tokens // page], (tokens % page).expand(b, -1)

    def gathered(cache, scale):  # [B, Hkv, T, D]
        if s["fmt"] == "fp8":
            x = cache.view(torch.uint8)[blocks, offsets].view(torch.float8_e4m3fn).float() * scale[:, None]
        else:
            x = cache[blocks, offsets].float()
            if s["fmt"] == "int8":
                x = x * scale[blocks, offsets][..., None]
        return x.transpose(1, 2).contiguous()

    q = s["query"].float().reshape(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = torch.matmul(q, gathered(s["k_cache"], s["k_scale"]).transpose(2, 3).contiguous()) * s["scale"]
    score = score.reshape(b, hkv, hq // hkv, n, -1)
    if s["cap"]:
        score = s["cap"] * torch.tanh(score / s["cap"])
    seen, far = _visible(s, tokens)
    if s["slopes"] is not None:
        score = score - s["slopes"].reshape(hkv, -1, 1, 1) * far[:, None, None].float()
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.reshape(b, hkv, -1, tokens.numel()), gathered(s["v_cache"], s["v_scale"]))
    out = out.reshape(b, hkv, hq // hkv, n, d) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(s["query"].dtype)


# ---- 64 bits -----------------------------------------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s["kind"] == "attend":
        return _exact_attend(s)
    q, k = _exact_rotated(s, s["query"], s["q_norm"]), _exact_rotated(s, s["key"], s["k_norm"])
    if s["kind"] == "embed":
        return q, k
    pools, scales = [], []
    where = s["write_blocks"].long() * s["page"] + s["write_offsets"].long()
    for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (s["value"].double(), s["v_cache"], s["v_scale"])):
        flat = cache.double().flatten(0, 1)
        if s["fmt"] == "int8":  # the nearest code of the row's own scale, and the value it stands for
            step = (x.abs().amax(-1) / 127).clamp_min(1e-12)
            x = (x / step[..., None]).round().clamp(-128, 127) * step[..., None]
            all_steps = scale.double().flatten()
            flat = flat * all_steps.reshape(-1, s["hkv"], 1)
            steps = all_steps.reshape(-1, s["hkv"]).index_copy(0, where.flatten(), step.flatten(0, 1))
            scales.append(steps.reshape(scale.shape))
        elif s["fmt"] == "fp8":  # the value itself in units of the scale: a code is off it by its rounding
            x = (x / scale.double()[:, None]).clamp(-448, 448)
        pools.append(flat.index_copy(0, where.flatten(), x.flatten(0, 1)).reshape(cache.shape))
    return q, *pools, *scales


def _exact_rotated(s: dict, x, weight):
    """Pairs of channels as complex numbers, multiplied by exp(i angle)."""
    x, half = x.double(), s["rot"] // 2
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / s["d"] + 1e-6).sqrt() * weight.double()
    first = torch.arange(half, device=DEV) * (2 if s["interleaved"] else 1)
    second = first + (1 if s["interleaved"] else half)
    pos = s["positions"].reshape(s["axes"], s["batch"], s["queries"])
    axis = _axis_of_pair(half, s["axes"], s["sections"], s["cyclic"])
    angle = torch.stack([pos[axis[i]].double() * s["inv_freq"][i].double() for i in range(half)], -1)[:, :, None]
    turned = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)
    out = x.clone()
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _exact_attend(s: dict):
    b, n, hq, d = s["query"].shape
    group, page, out = hq // s["hkv"], s["page"], torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for i in range(b):
        length = int(s["context_lens"][i])
        pages = s["block_table"][i, : -(-length // page)].long()
        j = torch.arange(length, device=DEV)
        p = torch.arange(length - n, length, device=DEV)[:, None]
        ok = (j <= p) & (j > p - s["window"]) if s["window"] else j <= p
        if s["starts"] is not None:
            ok = ok & (j >= s["starts"][i][:, None])
        if s["prefix_lens"] is not None:
            ok = ok | (j < s["prefix_lens"][i])
        for h in range(s["hkv"]):
            k, v = (s[w].view(torch.uint8)[pages, :, h].view(s[w].dtype).double().flatten(0, 1)[:length] if s["fmt"] != "bf16"
                    else s[w][pages, :, h].double().flatten(0, 1)[:length] for w in ("k_cache", "v_cache"))
            if s["fmt"] == "fp8":
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            elif s["fmt"] == "int8":
                k, v = (x * s[w][pages, :, h].double().flatten()[:length, None] for x, w in ((k, "k_scale"), (v, "v_scale")))
            for r in range(h * group, (h + 1) * group):
                a = s["query"][i, :, r].double() @ k.T * s["scale"]
                a = s["cap"] * torch.tanh(a / s["cap"]) if s["cap"] else a
                if s["slopes"] is not None:
                    a = a - s["slopes"][r].double() * (p - j).abs()
                a = torch.softmax(a.masked_fill(~ok, -math.inf), -1).nan_to_num(0.0)
                out[i, :, r] = a @ v
    return out
