"""CPU: rotary positions' host side (axes of pairs, refusals) and the oracle against its derivative's definition."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import rotary as orot


def test_pairs_follow_their_sections():
    from bpt_amd.rotary import pair_axes

    assert pair_axes(4, 1, None, False) == bytes(4)
    assert pair_axes(4, 1, (4,), True) == bytes(4)
    assert list(pair_axes(8, 3, (4, 2, 2), False)) == [0, 0, 0, 0, 1, 1, 2, 2]
    assert list(pair_axes(8, 3, (4, 2, 2), True)) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert list(pair_axes(5, 2, (0, 5), False)) == [1] * 5


@pytest.mark.parametrize("half, axes, sections, cyclic", [
    (8, 2, None, False), (8, 2, (4, 3), False), (8, 2, (9, -1), False), (8, 3, (4, 4), False), (8, 1, (4,), False),
    (8, 3, (2, 3, 3), True), (6, 9, (1,) * 9, False), (8, 0, (), False),
])
def test_sections_that_do_not_fit_are_refused(half, axes, sections, cyclic):
    from bpt_amd.rotary import pair_axes

    with pytest.raises(ValueError):
        pair_axes(half, axes, sections, cyclic)


def args(**change):
    """rotary_append's arguments on the CPU, some of them changed."""
    bf = torch.bfloat16
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=bf), k=torch.zeros(2, 3, 2, 64, dtype=bf), v=torch.zeros(2, 3, 2, 64, dtype=bf),
             positions=torch.zeros(2, 3, dtype=torch.int32), inv_freq=torch.ones(32),
             k_cache=torch.zeros(4, 16, 2, 64, dtype=bf), v_cache=torch.zeros(4, 16, 2, 64, dtype=bf), k_scale=None, v_scale=None,
             write_blocks=torch.zeros(2, 3, dtype=torch.int32), write_offsets=torch.zeros(2, 3, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(positions=torch.zeros(3, 2, dtype=torch.int32)), dict(positions=torch.zeros(2, 3)),
    dict(positions=torch.zeros(2, 2, 3, dtype=torch.int32)), dict(inv_freq=torch.ones(33)), dict(inv_freq=torch.ones(0)),
    dict(inv_freq=torch.ones(32, dtype=torch.float64)), dict(inv_freq=torch.ones(64)[::2]), dict(q_norm=torch.ones(32)),
    dict(q_norm=torch.ones(64), k_norm=torch.ones(64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 4, 64)),
    dict(q=torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.int32)),
    dict(q_out=torch.zeros(2, 3, 4, 64)), dict(q_out=torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16).expand(2, 3, 4, 64)),
    dict(k=torch.zeros(2, 3, 2, 32, dtype=torch.bfloat16)), dict(sections=(16, 15)), dict(sections=(16, 16)),
    {},  # nothing is wrong but that the tensors are on the CPU
])
def test_bad_arguments_are_refused(change):
    from bpt_amd import rotary_append, rotary_embed

    a = args(**change)
    with pytest.raises(ValueError):
        rotary_append(**a)
    if "q_out" not in change and "k" not in change and "q" not in change:
        for name in ("v", "k_cache", "v_cache", "k_scale", "v_scale", "write_blocks", "write_offsets"):
            a.pop(name)
        with pytest.raises(ValueError):
            rotary_embed(**a)


def test_embed_without_keys_refuses_what_goes_with_them():
    from bpt_amd import rotary_embed

    a = args()
    with pytest.raises(ValueError, match="go with k"):
        rotary_embed(a["q"], None, a["positions"], a["inv_freq"], k_norm=torch.ones(64))


@pytest.mark.parametrize("field, value, said", [
    ("struct_size", 8, "stale binding"), ("x_dtype", 3, "bf16, f16 or f32"), ("positions_dtype", 2, "int32 or int64"),
    ("batch", -1, ">= 0"), ("head_dim", 258, "head_dim"), ("head_dim", 63, "head_dim"), ("rotary_dim", 66, "rotary_dim"),
    ("rotary_dim", 0, "rotary_dim"), ("rotary_dim", 31, "rotary_dim"), ("num_axes", 0, "num_axes"), ("num_axes", 9, "num_axes"),
    ("scaling", float("inf"), "scaling"), ("eps", -1.0, "eps"), ("eps", float("nan"), "eps"), ("q", None, "non-NULL"),
    ("k_out", None, "non-NULL"), ("inv_freq", None, "non-NULL"), ("positions", None, "non-NULL"), ("pair_axis", 1, "axis"),
])
def test_the_c_entry_refuses(built_lib, field, value, said):
    from bpt_amd import _lib

    a = _lib.RotaryArgs(struct_size=_lib.ROTARY_ARGS_SIZE, batch=1, num_queries=1, num_q_heads=1, num_k_heads=1, head_dim=64,
                        rotary_dim=64, num_axes=1, scaling=1.0, eps=1e-6, q=16, k=16, q_out=16, k_out=16, inv_freq=16, positions=16)
    if field == "pair_axis":
        a.pair_axis[31] = value
    else:
        setattr(a, field, value)
    assert built_lib.bpt_rotary_embed(ctypes.byref(a), None) == _lib.BPT_ERR_INVALID_ARGUMENT
    assert said in built_lib.bpt_last_error().decode()


@pytest.mark.parametrize("change", [dict(batch=2), dict(num_queries=2), dict(num_kv_heads=2), dict(head_dim=128), dict(src_dtype=2),
                                    dict(k=32), dict(new_stride_h=8)])
def test_the_halves_of_an_append_must_agree(built_lib, change):
    from bpt_amd import _lib

    a = _lib.RotaryArgs(struct_size=_lib.ROTARY_ARGS_SIZE, batch=1, num_queries=1, num_q_heads=1, num_k_heads=1, head_dim=64,
                        rotary_dim=64, num_axes=1, scaling=1.0, eps=1e-6, q=16, k=16, q_out=16, inv_freq=16, positions=16)
    w = _lib.AppendArgs(struct_size=_lib.APPEND_ARGS_SIZE, batch=1, num_queries=1, num_kv_heads=1, head_dim=64, page_size=16,
                        num_blocks=1, k=16, v=16, write_blocks=16, write_offsets=16, k_cache=16, v_cache=16)
    for name, value in change.items():
        setattr(w, name, value)
    assert built_lib.bpt_rotary_append(ctypes.byref(a), ctypes.byref(w), None) == _lib.BPT_ERR_INVALID_ARGUMENT
    assert "same keys" in built_lib.bpt_last_error().decode()


def test_calls_with_no_rows_do_nothing(built_lib):
    from bpt_amd import _lib

    a = _lib.RotaryArgs(struct_size=_lib.ROTARY_ARGS_SIZE, batch=0, num_queries=1, num_q_heads=1, num_k_heads=1, head_dim=64,
                        rotary_dim=64, num_axes=1, scaling=1.0, eps=1e-6)
    assert built_lib.bpt_rotary_embed(ctypes.byref(a), None) == _lib.BPT_OK
    a.batch, a.num_q_heads, a.num_k_heads = 4, 0, 0
    assert built_lib.bpt_rotary_embed(ctypes.byref(a), None) == _lib.BPT_OK


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_turns_by_the_angle(interleaved):
    """d/dt (a cos t - b sin t, a sin t + b cos t) = (-second, first): by differences of a fractional frequency."""
    g = np.random.default_rng(0)
    x, pos, f, h = g.standard_normal((1, 2, 1, 8)), np.array([[[3, 5]]]), np.array([0.5, 0.25, 0.125]), 1e-6
    at = lambda d: orot.rotate(x, pos, f + d, interleaved=interleaved)  # noqa: E731
    slope, mid = (at(h) - at(-h)) / (2 * h), at(0.0)
    for i in range(3):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, 3 + i)
        assert np.allclose(slope[..., a], -mid[..., b] * pos[0][..., None], atol=1e-7)
        assert np.allclose(slope[..., b], mid[..., a] * pos[0][..., None], atol=1e-7)
    assert np.array_equal(mid[..., 6:], x[..., 6:])
