"""CPU: paged_masked_attention's refusals, its plan, and the oracle's masks."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import masked as omask

BF = torch.bfloat16


def args(**change):
    a = dict(q=torch.zeros(2, 3, 4, 128, dtype=BF), k_cache=torch.zeros(4, 16, 2, 128, dtype=BF),
             v_cache=torch.zeros(4, 16, 2, 128, dtype=BF), block_table=torch.zeros(2, 2, dtype=torch.int32),
             context_lens=torch.zeros(2, dtype=torch.int32), scale=0.1, max_context=32)
    a.update(change)
    return a


@pytest.mark.parametrize("change, said", [
    (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(window=0), "window"),
    (dict(slopes=torch.ones(3)), "slopes"), (dict(slopes=torch.ones(4, dtype=torch.float64)), "slopes"),
    (dict(slopes=torch.ones(8)[::2]), "slopes"), (dict(max_prefix=3), "max_prefix"),
    (dict(prefix_lens=torch.zeros(3, dtype=torch.int32)), "prefix_lens"), (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), "prefix_lens"),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int32), max_prefix=-1), "max_prefix"),
    (dict(starts=torch.zeros(2, 2, dtype=torch.int32)), "starts"), (dict(starts=torch.zeros(2, 3)), "starts"),
    (dict(q=torch.zeros(2, 3, 4, 128)), "bf16 or f16"), (dict(q=torch.zeros(2, 3, 4, 64, dtype=BF)), "head_dim"), ({}, "GPU"),
    (dict(softcap=1e-50), "softcap"),
])
def test_bad_arguments_are_refused(change, said):
    from bpt_amd import paged_masked_attention

    with pytest.raises(ValueError, match=said):
        paged_masked_attention(**args(**change))


def c_args(**change):
    from bpt_amd import _lib

    a = _lib.DecodeArgs(struct_size=_lib.DECODE_ARGS_SIZE, batch=2, num_queries=1, num_q_heads=4, num_kv_heads=2, head_dim=128, page_size=16,
                        num_blocks=8, max_blocks_per_seq=64, max_context=1000, sm_scale=0.1, kv_stride_block=4096, kv_stride_token=256,
                        kv_stride_head=128)
    m = _lib.MaskArgs(struct_size=_lib.MASK_ARGS_SIZE)
    for name, value in change.items():
        setattr(m if hasattr(m, name) and name != "struct_size" else a, name, value)
    return a, m


@pytest.mark.parametrize("change, said", [
    (dict(q_dtype=2), "bf16 or f16"), (dict(num_splits=3), "num_splits"), (dict(flags=1), "flags"), (dict(len_offset=1), "len_offset"),
    (dict(merge_out=16), "merge"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"), (dict(window=-1), "window"),
    (dict(max_prefix=-1), "max_prefix"), (dict(head_dim=64), "head_dim"), (dict(page_size=24), "page_size"),
    (dict(sm_scale=float("nan")), "sm_scale"), (dict(softcap=1e-38, sm_scale=1e30), "out of range"),
    (dict(kv_stride_token=1 << 27), "2 GiB"), (dict(struct_size=1), "stale"),
    (dict(max_context=2**31 - 1, max_blocks_per_seq=2**27), "max_context"),
])
def test_the_c_entry_refuses(built_lib, change, said):
    from bpt_amd import _lib

    a, m = c_args(**change)
    ws, cnt = ctypes.c_size_t(), ctypes.c_size_t()
    for rc in (built_lib.bpt_masked_plan(a, m, ws, cnt), built_lib.bpt_paged_masked(a, m, None)):
        assert rc == _lib.BPT_ERR_INVALID_ARGUMENT
        assert said in built_lib.bpt_last_error().decode()


def test_the_c_entry_refuses_a_stale_mask_missing_tensors_and_small_buffers(built_lib):
    from bpt_amd import _lib

    a, m = c_args()
    m.struct_size = 8
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_ERR_INVALID_ARGUMENT and "stale" in built_lib.bpt_last_error().decode()
    assert built_lib.bpt_paged_masked(a, None, None) == _lib.BPT_ERR_INVALID_ARGUMENT
    a, m = c_args()
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_ERR_INVALID_ARGUMENT and "non-NULL" in built_lib.bpt_last_error().decode()
    a, m = c_args(q=16, k_cache=16, v_cache=16, block_table=16, out=16)
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_ERR_INVALID_ARGUMENT and "workspace" in built_lib.bpt_last_error().decode()
    a.workspace, a.workspace_bytes = 256, 1 << 40
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_ERR_INVALID_ARGUMENT and "counter" in built_lib.bpt_last_error().decode()
    a.k_cache = 8
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_ERR_INVALID_ARGUMENT and "aligned" in built_lib.bpt_last_error().decode()
    a.batch = 0
    assert built_lib.bpt_paged_masked(a, m, None) == _lib.BPT_OK


@pytest.mark.parametrize("change", [dict(), dict(window=64), dict(num_queries=700), dict(batch=4096), dict(max_context=0),
                                    dict(window=2**31 - 1), dict(prefix_lens=16, max_prefix=2**31 - 1, window=5)])
def test_plans(built_lib, change):
    """A plan's buffers hold its partials; a window shrinks them to what it leaves to read."""
    a, m = c_args(**change)
    ws, cnt = ctypes.c_size_t(), ctypes.c_size_t()
    assert built_lib.bpt_masked_plan(a, m, ws, cnt) == 0
    assert (ws.value == 0) == (cnt.value == 0) and ws.value % 256 == 0 and ws.value < 1 << 33
    if change == dict(window=64):
        assert ws.value == 0  # four steps: one piece
    if not change:
        assert ws.value > 0


def test_oracle_masks():
    seen, far = omask.visible(6, 2, prefix=1, starts=[3, 0], window=2)
    assert np.array_equal(seen, np.array([[1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]], dtype=bool))
    assert np.array_equal(far[0], [4, 3, 2, 1, 0, 1])
