"""Paged attention with masked and shaped scores on HIP, over the same BF16 / FP8 / INT8 caches as paged_decode_attention.

Query i of sequence b sits at position p = context_lens[b] - Q + i and sees cache slot j if

    j < context_lens[b]  and  (j < prefix_lens[b]  or  (starts[b, i] <= j <= p  and  p - j < window))

and its score for head h is t = scale * q.k, then softcap * tanh(t / softcap), then minus slopes[h] * |p - j|. Prefixes make
prefix language models (and, with a window, first tokens that stay visible), starts keep documents packed into one sequence
apart, slopes are a linear bias by distance. What is not given does not apply. A query that sees nothing gets zeros. Any number of
queries, one launch; no gradient is recorded.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .paged_attention import _decode_args, _on_device, _stream, cached_buffer


def _mask_args(b, nq, hq, max_context, softcap, slopes, window, prefix_lens, max_prefix, starts) -> _lib.MaskArgs:
    """The checked bpt_mask_args."""
    if softcap is not None and not ctypes.c_float(softcap).value > 0:
        raise ValueError(f"softcap must be positive as a float32, got {softcap}")
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if slopes is not None and not (slopes.dtype == torch.float32 and tuple(slopes.shape) == (hq,) and slopes.is_contiguous()):
        raise ValueError(f"slopes must be a contiguous float32 [{hq}]")
    if prefix_lens is None:
        if max_prefix is not None:
            raise ValueError("max_prefix goes with prefix_lens")
        max_prefix = 0
    else:
        if not (prefix_lens.dtype == torch.int32 and tuple(prefix_lens.shape) == (b,) and prefix_lens.is_contiguous()):
            raise ValueError(f"prefix_lens must be a contiguous int32 [{b}]")
        max_prefix = max_context if max_prefix is None else max_prefix
        if max_prefix < 0:
            raise ValueError(f"max_prefix must not be negative, got {max_prefix}")
    if starts is not None and not (starts.dtype == torch.int32 and tuple(starts.shape) == (b, nq)):
        raise ValueError(f"starts must be int32 [{b}, {nq}]")
    st_sb, st_sq = (0, 0) if starts is None else starts.stride()
    top = 2**31 - 1
    return _lib.MaskArgs(
        _lib.MASK_ARGS_SIZE, 0.0 if softcap is None else float(softcap), 0 if window is None else min(int(window), top),
        min(int(max_prefix), top), None if slopes is None else slopes.data_ptr(),
        None if prefix_lens is None else prefix_lens.data_ptr(), None if starts is None else starts.data_ptr(), st_sb, st_sq,
    )


def paged_masked_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    *,
    scale: float,
    max_context: int,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    window: int | None = None,
    prefix_lens: torch.Tensor | None = None,
    max_prefix: int | None = None,
    starts: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    lse: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    counters: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention over the paged cache with the masks and scores of the module's description.

    q, caches, block_table, context_lens, scales, max_context, out, out_dtype, lse as paged_decode_attention's (q in bf16 or
    f16 only; head_dim 128)
    softcap      positive float: scores are softcap * tanh(score / softcap)
    slopes       float32 [Hq]: scores fall by slopes[h] per token of distance
    window       a query sees its own position and the window - 1 before it
    prefix_lens  int32 [B]: the tokens of each sequence that all of its queries see, later ones included
    max_prefix   upper bound on prefix_lens, known on the host (larger ones are cut to it); sizes the launch. Default: max_context
    starts       int32 [B, Q]: each query's first token behind the prefix
    workspace, counters  optional device buffers of at least masked_plan(...) bytes, the counters zero-filled before their first
                 use and not shared by calls that may run at once; default: cached per (device, stream), or the graph's own while
                 one is captured

    Returns [B, Q, Hq, D] (or [B, Hq, D] for a 3-D q with one query per sequence) in out_dtype.
    """
    call = _checked(q, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, scale, max_context, softcap, slopes, window,
                    prefix_lens, max_prefix, starts, out, out_dtype, lse)
    result = _launch(*call, workspace, counters)
    return result[:, 0] if (q.dim() == 3 and result.dim() == 4) else result


def _checked(q, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, scale, max_context, softcap=None, slopes=None, window=None,
             prefix_lens=None, max_prefix=None, starts=None, out=None, out_dtype=torch.bfloat16, lse=None):
    """Everything of a call that can be refused, apart from its buffers: (decode args, mask args, device, result)."""
    q4 = q[:, None] if q.dim() == 3 else q
    a, (b, nq, hq, d) = _decode_args(q4, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, scale, max_context, None,
                                     out.dtype if out is not None else out_dtype)
    m = _mask_args(b, nq, hq, int(max_context), softcap, slopes, window, prefix_lens, max_prefix, starts)
    if q.dtype == torch.float32:
        raise ValueError("q must be bf16 or f16")
    dev = q.device
    if not q.is_cuda:
        raise ValueError("paged_masked_attention runs on a GPU: q must be a cuda tensor")
    for t in (k_cache, v_cache, block_table, context_lens, k_scale, v_scale, slopes, prefix_lens, starts):
        if t is not None and t.device != dev:
            raise ValueError(f"a tensor of the call is on {t.device}, q on {dev}")
    if out is None:
        out4 = q.new_empty((b, nq, hq, d), dtype=out_dtype)
    else:
        out4 = out[:, None] if out.dim() == 3 else out
        if tuple(out4.shape) != (b, nq, hq, d):
            raise ValueError(f"out must be [{b}, {nq}, {hq}, {d}]")
        if not (out4.stride(-1) == 1 and out4.device == dev):
            raise ValueError("out must be a cuda tensor with contiguous channels")
        if any(n > 1 and s == 0 for n, s in zip(out4.shape, out4.stride())):
            raise ValueError("out must not be an expanded view")
    a.out = out4.data_ptr()
    a.out_stride_b, a.out_stride_q, a.out_stride_h, _ = out4.stride()
    if lse is not None:
        if not (lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() == b * nq * hq and lse.device == dev):
            raise ValueError(f"lse must be a contiguous float32 tensor of {b} x {nq} x {hq} on q's device")
        a.lse_out = lse.data_ptr()
    return a, m, dev, out if out is not None else out4


def _launch(a, m, dev, result, workspace=None, counters=None) -> torch.Tensor:
    lib = _lib.lib()
    with _on_device(dev):
        stream = _stream(dev)
        if workspace is None or counters is None:
            ws_bytes, cnt_bytes = ctypes.c_size_t(), ctypes.c_size_t()
            _lib.check(lib.bpt_masked_plan(a, m, ws_bytes, cnt_bytes))
            if torch._C._cuda_isCurrentStreamCapturing():
                # Captures share one stream, but their graphs may be replayed at once: each call gets buffers of its own, from
                # its graph's pool, and the counters' clearing is part of the graph.
                workspace = torch.empty(ws_bytes.value, dtype=torch.uint8, device=dev) if workspace is None else workspace
                counters = torch.zeros(cnt_bytes.value // 4, dtype=torch.int32, device=dev) if counters is None else counters
            else:
                workspace = cached_buffer("partials", dev, stream, ws_bytes.value) if workspace is None else workspace
                counters = cached_buffer("counters", dev, stream, cnt_bytes.value) if counters is None else counters
        for name, t in (("workspace", workspace), ("counters", counters)):
            if t.device != dev or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous tensor on q's device")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.nbytes
        a.counters, a.counters_bytes = counters.data_ptr(), counters.nbytes
        _lib.check(lib.bpt_paged_masked(a, m, stream))
    return result


def masked_plan(q, k_cache, v_cache, block_table, context_lens, k_scale=None, v_scale=None, *, scale, max_context, softcap=None,
                slopes=None, window=None, prefix_lens=None, max_prefix=None, starts=None) -> tuple[int, int]:
    """(workspace bytes, counter bytes) that paged_masked_attention would use. Host only."""
    q4 = q[:, None] if q.dim() == 3 else q
    a, (b, nq, hq, _) = _decode_args(q4, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, scale, max_context, None,
                                     torch.bfloat16)
    m = _mask_args(b, nq, hq, int(max_context), softcap, slopes, window, prefix_lens, max_prefix, starts)
    ws, cnt = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.check(_lib.lib().bpt_masked_plan(a, m, ws, cnt))
    return ws.value, cnt.value
