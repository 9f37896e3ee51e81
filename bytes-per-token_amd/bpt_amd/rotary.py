"""Rotary positions on HIP: queries and keys normalised per head and rotated, the keys on their way into the paged cache.

What a model does between its projections and the cache's attend (fastserve's engine/rope.py and the per-head norms of
engine/model.py:52-74) as one launch: `rotary_embed` writes rotated queries and keys, `rotary_append` writes rotated
queries and stores the rotated keys and the values into their pages, as `quantize_append` does.

With `inv_freq` [rotary_dim / 2] and t = position * inv_freq[i] (computed in float64), pair i of a row's channels becomes
scaling * (a cos t - b sin t, a sin t + b cos t); the pairs are channels (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with
`interleaved`, and channels past rotary_dim stay. Positions may have several axes (time, height, width): each pair then
follows one of them, in stretches of `sections[a]` pairs, or dealt out in turn with `cyclic` (pair i follows axis i % A
while i // A < sections[i % A], else axis 0). Arithmetic is float32, rounded once. These are inference operators: they
record no gradient.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .paged_attention import _FLOAT_CODES, _INDEX_CODES, _append_args, _on_device, _stream

MAX_AXES = 8


@functools.lru_cache(maxsize=256)
def pair_axes(half: int, axes: int, sections: tuple[int, ...] | None, cyclic: bool) -> bytes:
    """The axis that each of the `half` pairs follows, one byte each."""
    if axes == 1:
        if sections is not None and sections != (half,):
            raise ValueError(f"sections {sections} given for positions with one axis and {half} pairs")
        return bytes(half)
    if not 1 <= axes <= MAX_AXES:
        raise ValueError(f"positions must have 1 to {MAX_AXES} axes, got {axes}")
    if sections is None or len(sections) != axes or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"sections must be {axes} numbers of pairs with the sum {half}, got {sections}")
    if not cyclic:
        return b"".join(bytes([a]) * n for a, n in enumerate(sections))
    out = bytes(i % axes if i // axes < sections[i % axes] else 0 for i in range(half))
    if any(out.count(a) != n for a, n in enumerate(sections)):
        raise ValueError(f"cyclic sections {sections} do not fit: axis a's last pair {axes} * (sections[a] - 1) + a must be "
                         f"below {half}, and axis 0 takes the rest")
    return out


def _check_rows(name: str, x: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if x.dim() != 4 or x.stride(3) != 1:
        raise ValueError(f"{name} must be [B, Q, H, D] with contiguous channels, got {tuple(x.shape)}")
    if x.dtype not in _FLOAT_CODES:
        raise ValueError(f"{name} must be bf16, f16 or f32, got {x.dtype}")
    if like is not None:
        if x.dtype != like.dtype or x.device != like.device:
            raise ValueError(f"{name} must have q's dtype and device")
        if x.shape[:2] != like.shape[:2] or x.shape[3] != like.shape[3]:
            raise ValueError(f"{name} must be [{like.shape[0]}, {like.shape[1]}, H, {like.shape[3]}], got {tuple(x.shape)}")


def _out_like(name: str, out: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor:
    if out is None:
        return x.new_empty(x.shape)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(-1) != 1:
        raise ValueError(f"{name} must be {tuple(x.shape)} in {x.dtype} on {x.device}, channels contiguous")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not be an expanded view")
    return out


def _rotary_args(q, k, q_out, k_out, positions, inv_freq, sections, cyclic, interleaved, scaling, q_norm, k_norm, eps):
    """The checked bpt_rotary_args."""
    b, n, hq, d = q.shape
    pos_shape, pos_code = positions.shape, _INDEX_CODES.get(positions.dtype)
    if len(pos_shape) not in (2, 3) or pos_shape[-2:] != (b, n) or pos_code is None:
        raise ValueError(f"positions must be int32 / int64 [{b}, {n}] or [axes, {b}, {n}], got {tuple(positions.shape)}")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 [rotary_dim / 2]")
    half = inv_freq.shape[0]
    if not 1 <= half <= d // 2 or d % 2 or d > 256:
        raise ValueError(f"{half} pairs do not fit into head_dim {d} (even, at most 256)")
    norm_code = 0
    for w in (q_norm, k_norm):
        if w is not None:
            if w.shape != (d,) or w.dtype not in _FLOAT_CODES or not w.is_contiguous():
                raise ValueError(f"q_norm and k_norm must be contiguous bf16 / f16 / f32 [{d}]")
            norm_code = _FLOAT_CODES[w.dtype]
    if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
        raise ValueError("q_norm and k_norm must share a dtype")
    dev = q.device
    if not q.is_cuda:
        raise ValueError("rotary positions are applied on a GPU: q must be a cuda tensor")
    if positions.device != dev or inv_freq.device != dev or (q_norm is not None and q_norm.device != dev) or (
            k_norm is not None and k_norm.device != dev):
        raise ValueError(f"positions, inv_freq and norm weights must be on q's device {dev}")
    axes = 1 if len(pos_shape) == 2 else pos_shape[0]
    which = pair_axes(half, axes, None if sections is None else tuple(sections), bool(cyclic))
    pos_sa, pos_sb, pos_sq = (0, *positions.stride()) if len(pos_shape) == 2 else positions.stride()
    q_sb, q_sq, q_sh, _ = q.stride()
    qo_sb, qo_sq, qo_sh, _ = q_out.stride()
    k_ptr = ko_ptr = None
    k_sb = k_sq = k_sh = ko_sb = ko_sq = ko_sh = hk = 0
    if k is not None:
        k_ptr, hk = k.data_ptr(), k.shape[2]
        k_sb, k_sq, k_sh, _ = k.stride()
    if k_out is not None:
        ko_ptr = k_out.data_ptr()
        ko_sb, ko_sq, ko_sh, _ = k_out.stride()
    # The fields of bpt_rotary_args in order, up to pair_axis.
    a = _lib.RotaryArgs(
        _lib.ROTARY_ARGS_SIZE, _FLOAT_CODES[q.dtype], norm_code, pos_code, b, n, hq, hk, d, 2 * half, axes, bool(interleaved), scaling,
        eps, q.data_ptr(), q_sb, q_sq, q_sh, k_ptr, k_sb, k_sq, k_sh, q_out.data_ptr(), qo_sb, qo_sq, qo_sh, ko_ptr, ko_sb, ko_sq, ko_sh,
        None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), inv_freq.data_ptr(),
        positions.data_ptr(), pos_sa, pos_sb, pos_sq,
    )
    ctypes.memmove(a.pair_axis, which, half)
    return a


def rotary_embed(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    sections: tuple[int, ...] | None = None,
    cyclic: bool = False,
    interleaved: bool = False,
    scaling: float = 1.0,
    q_norm: torch.Tensor | None = None,
    k_norm: torch.Tensor | None = None,
    eps: float = 1e-6,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [B, Q, Hq, D] and k [B, Q, Hk, D] (or None) rotated by their positions; returns both in their dtype.

    positions   [B, Q] or [axes, B, Q], int32 or int64: any integers
    inv_freq    float32 [rotary_dim / 2]
    sections    with several axes: how many pairs follow each (see the module's description); `cyclic`: dealt out in turn
    scaling     factor on the rotated channels (a length-extension's attention factor)
    q/k_norm    optional [D] weights: x * rsqrt(mean(x^2) + eps) * weight per head, ahead of the rotation
    q/k_out     optional outputs; the inputs themselves are allowed (in place), other overlaps are not
    """
    _check_rows("q", q)
    if k is not None:
        _check_rows("k", k, q)
    elif k_norm is not None or k_out is not None:
        raise ValueError("k_norm and k_out go with k")
    q_out = _out_like("q_out", q_out, q)
    k_out = None if k is None else _out_like("k_out", k_out, k)
    a = _rotary_args(q, k, q_out, k_out, positions, inv_freq, sections, cyclic, interleaved, scaling, q_norm, k_norm, eps)
    with _on_device(q.device):
        _lib.check(_lib.lib().bpt_rotary_embed(a, _stream(q.device)))
    return q_out, k_out


def rotary_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor | None,
    v_scale: torch.Tensor | None,
    write_blocks: torch.Tensor,
    write_offsets: torch.Tensor,
    *,
    sections: tuple[int, ...] | None = None,
    cyclic: bool = False,
    interleaved: bool = False,
    scaling: float = 1.0,
    q_norm: torch.Tensor | None = None,
    k_norm: torch.Tensor | None = None,
    eps: float = 1e-6,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """rotary_embed of q and k whose keys go into the paged pools, with the values, as quantize_append stores them: one
    launch, and the keys are quantized from float32 (rotary_embed, then quantize_append, would round them to their dtype in
    between). Returns the rotated q.

    k, v [B, Q, Hkv, D] are stored at slot write_offsets[b, i] of page write_blocks[b, i]; rows whose page or offset lies
    outside the pool are skipped (their q is rotated all the same). The slots of a call must be distinct. Pools, scales and
    slots as quantize_append's, head_dim 64, 128 or 256; the other arguments as rotary_embed's.
    """
    _check_rows("q", q)
    w, dev = _append_args(k, v, k_cache, v_cache, k_scale, v_scale, write_blocks, write_offsets)
    if k.dtype != q.dtype or q.device != dev or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q must have k's dtype, device, batch, queries and head_dim, got {q.dtype} {tuple(q.shape)}, k {tuple(k.shape)}")
    q_out = _out_like("q_out", q_out, q)
    a = _rotary_args(q, k, q_out, None, positions, inv_freq, sections, cyclic, interleaved, scaling, q_norm, k_norm, eps)
    with _on_device(q.device):
        _lib.check(_lib.lib().bpt_rotary_append(a, w, _stream(q.device)))
    return q_out
