"""GPU: rotary positions (rotary_embed, rotary_append) against the float64 oracle.

Tolerances, from the arithmetic: a float32 result is a sum of two products. The angle's float64 error is below 2^-22 at
2^31 positions (2^-40 at 2^13); cosine and sine are off by at most 2^-23 (the reduced angle's rounding, the polynomial's last
two steps), each product and sum by 2^-24, the norm's root mean square by (21 + 4) / 2 roundings of 2^-24 (16 terms in a lane,
5 exchanges, then division, square root, reciprocal), its two products by two. Together below 24 * 2^-24 = 1.5e-6 of the pair's
magnitudes; rounding to 16 bits adds half a step, `eps / 2` of the value (and half of the least subnormal for f16, 2^-25).
"""

import numpy as np
import pytest
import torch

from oracle import rotary as orot

pytestmark = pytest.mark.gpu

DEV = "cuda"
EXACT = 24 * 2.0**-24


def within(got, want, spread, far=0.0):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    bound = (EXACT + far) * spread * (1 + half) + half * np.abs(want) + (2.0**-25 if got.dtype == torch.float16 else 1e-30)
    assert (err <= bound).all(), f"{(err - bound).max():.3e} over the bound, at {np.argwhere(err > bound)[:4]}"


def rows(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def freqs(half):
    return (1e4 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(DEV)


def sections_of(half, axes):
    rest = [half // (axes + 1)] * (axes - 1)
    return None if axes == 1 else (half - sum(rest), *rest)


def positions_of(axes, b, n, dtype, seed, most=5000):
    g = torch.Generator(device=DEV).manual_seed(seed)
    p = torch.randint(-10, most, (axes, b, n), generator=g, device=DEV).to(dtype)
    return (p[0] if axes == 1 else p), p.cpu().numpy()


CASES = [  # b, n, hq, hk, d, rot, axes, cyclic, interleaved, norm, dtype, index
    (1, 1, 16, 8, 128, 128, 1, False, False, True, torch.bfloat16, torch.int32),
    (3, 5, 32, 8, 128, 128, 3, True, False, False, torch.float16, torch.int64),
    (2, 7, 4, 2, 128, 64, 1, False, True, True, torch.float32, torch.int32),
    (2, 33, 5, 1, 64, 64, 2, False, True, False, torch.bfloat16, torch.int64),
    (1, 130, 3, 3, 256, 256, 3, False, False, True, torch.float32, torch.int32),
    (1, 9, 16, 16, 80, 80, 2, False, False, False, torch.bfloat16, torch.int32),
    (2, 3, 2, 1, 72, 36, 3, True, False, True, torch.float32, torch.int32),  # 18 pairs: no whole units
    (2, 3, 2, 2, 256, 2, 1, False, False, True, torch.float32, torch.int32),  # 17 units in 32 lanes
    (1, 4, 1, 1, 2, 2, 1, False, True, True, torch.float32, torch.int32),
    (1, 4, 3, 0, 96, 48, 2, True, True, False, torch.bfloat16, torch.int32),  # no keys
    (1, 2, 1, 1, 20, 14, 1, False, True, True, torch.float16, torch.int64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_embed(case):
    from bpt_amd import rotary_embed
    from bpt_amd.rotary import pair_axes

    b, n, hq, hk, d, rot, axes, cyclic, inter, norm, dtype, index = case
    q, k = rows((b, n, hq, d), dtype, 1), rows((b, n, hk, d), dtype, 2) if hk else None
    pos, pos_h = positions_of(axes, b, n, index, 3)
    wq, wk = (rows((d,), dtype, 4), rows((d,), dtype, 5) if hk else None) if norm else (None, None)
    sections, inv = sections_of(rot // 2, axes), freqs(rot // 2)
    got = rotary_embed(q, k, pos, inv, sections=sections, cyclic=cyclic, interleaved=inter, scaling=1.25, q_norm=wq, k_norm=wk, eps=1e-5)
    torch.cuda.synchronize()
    which = list(pair_axes(rot // 2, axes, sections, cyclic))
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        if x is None:
            assert y is None
            continue
        host = (x.double().cpu().numpy(), inv.cpu().numpy())
        weight = None if w is None else w.double().cpu().numpy()
        want = orot.rotate(host[0], pos_h, host[1], which, inter, 1.25, weight, 1e-5)
        assert y.dtype == dtype and y.shape == x.shape
        within(y, want, orot.spread(host[0], host[1], inter, 1.25, weight, 1e-5))


def test_far_positions():
    """Angles of positions up to 2^31: the turns are held in float64, 2^31 * 2^-52 turns of error at most."""
    from bpt_amd import rotary_embed

    q = rows((1, 6, 2, 64), torch.float32, 0)
    pos = torch.tensor([[0, 1 << 20, 123456789, (1 << 31) - 1, -(1 << 31), -7]], dtype=torch.int64, device=DEV)
    got, _ = rotary_embed(q, None, pos, freqs(32))
    torch.cuda.synchronize()
    x = q.double().cpu().numpy()
    want = orot.rotate(x, pos.cpu().numpy()[None], freqs(32).cpu().numpy())
    within(got, want, orot.spread(x, freqs(32).cpu().numpy()), far=2.0**-20 * 6.3)
    near = [0, 1, 5]
    assert np.abs(got.double().cpu().numpy() - want)[:, near].max() < 24 * 2.0**-24 * 8


@pytest.mark.parametrize("how", ["views", "unaligned", "in place", "expanded positions"])
def test_strides(how):
    from bpt_amd import rotary_embed

    b, n, hq, hk, d = 2, 5, 4, 2, 64
    fused = rows((b, n, hq + 2 * hk, d + (1 if how == "unaligned" else 0)), torch.bfloat16, 6)
    before = fused.clone()
    q, k = fused[:, :, :hq, :d], fused[:, :, hq : hq + hk, :d]
    pos, pos_h = positions_of(1, b, n, torch.int32, 7)
    if how == "expanded positions":
        pos = pos[:1].expand(b, n)
        pos_h = pos.cpu().numpy()[None]
    inv = freqs(16)
    more = dict(q_out=q, k_out=k) if how == "in place" else {}
    if how == "views":  # head-major inputs and outputs
        q, k = q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2)
        more = dict(q_out=torch.empty((b, hq, n, d), dtype=q.dtype, device=DEV).transpose(1, 2))
    x = [t.double().cpu().numpy() for t in (q, k)]
    got = rotary_embed(q, k, pos, inv, **more)
    torch.cuda.synchronize()
    for y, host in zip(got, x):
        within(y, orot.rotate(host, pos_h, inv.cpu().numpy()), orot.spread(host, inv.cpu().numpy()))
    if how == "in place":
        assert got[0].data_ptr() == fused.data_ptr()
        assert torch.equal(fused[:, :, hq + hk :], before[:, :, hq + hk :])
    else:
        assert torch.equal(fused, before)


def pools(fmt, nb, page, hkv, d, per_token):
    g = torch.Generator(device=DEV).manual_seed(11)
    dtype = {"bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}[fmt]
    raw = torch.randint(0, 100, (2, nb, page, hkv, d * (2 if fmt == "bf16" else 1)), generator=g, device=DEV, dtype=torch.uint8)
    k, v = raw[0].view(dtype), raw[1].view(dtype)
    if fmt == "bf16":
        return k, v, None, None
    shape = (nb, page, hkv) if per_token else (hkv,)
    ks, vs = (torch.rand(shape, generator=g, device=DEV) * 0.02 + 0.01 for _ in range(2))
    return k, v, ks, vs


@pytest.mark.parametrize("fmt, per_token", [("bf16", False), ("fp8", False), ("fp8", True), ("int8", False), ("int8", True)])
@pytest.mark.parametrize("d, hkv, dtype, inter", [(128, 8, torch.bfloat16, False), (64, 1, torch.float16, True), (256, 3, torch.float32, False),
                                                  (128, 2, torch.bfloat16, True)])
def test_append(fmt, per_token, d, hkv, dtype, inter):
    """Queries as embed's; the pool holds the rotated keys and the values to half a step of its codes, in their slots and
    nowhere else; rows with no slot leave nothing."""
    from bpt_amd import rotary_append

    b, n, hq, page, nb, rot = 3, 4, 2 * hkv, 16, 6, d // 2
    q, k, v = rows((b, n, hq, d), dtype, 1), rows((b, n, hkv, d), dtype, 2), rows((b, n, hkv, d), dtype, 3)
    kc, vc, ks, vs = pools(fmt, nb, page, hkv, d, per_token)
    was = [None if t is None else t.clone() for t in (kc, vc, ks, vs)]
    slots = torch.randperm(nb * page, generator=torch.Generator().manual_seed(5))[: b * n].reshape(b, n)
    wb, wo = slots // page, slots % page
    wb[0, 1], wb[1, 2], wo[2, 3], wb[2, 0] = -1, nb, page, 1 << 30
    pos, pos_h = positions_of(2, b, n, torch.int32, 3)
    wk = rows((d,), torch.float32, 9)
    got = rotary_append(q, k, v, pos, freqs(rot // 2), kc, vc, ks, vs, wb.to(DEV), wo.to(DEV), sections=(rot // 2 - 5, 5), interleaved=inter,
                        k_norm=wk, eps=1e-6)
    torch.cuda.synchronize()
    inv = freqs(rot // 2).cpu().numpy()
    which = [0] * (rot // 2 - 5) + [1] * 5
    xq, xk, xv = (t.double().cpu().numpy() for t in (q, k, v))
    within(got, orot.rotate(xq, pos_h, inv, which, inter), orot.spread(xq, inv, inter))
    weight = wk.double().cpu().numpy()
    want_k = orot.rotate(xk, pos_h, inv, which, inter, 1.0, weight)
    spread_k = orot.spread(xk, inv, inter, 1.0, weight)
    live = ((wb >= 0) & (wb < nb) & (wo >= 0) & (wo < page)).numpy()
    at = (wb.numpy()[live], wo.numpy()[live])
    for cache, scale, old, old_scale, want, spread in ((kc, ks, was[0], was[2], want_k, spread_k), (vc, vs, was[1], was[3], xv, np.abs(xv))):
        want, spread = want[live], spread[live]
        stored = cache.float().cpu().double().numpy()[at]
        if fmt == "bf16":
            bound = EXACT * spread * 1.01 + 2.0**-8 * np.abs(want)
            step = np.ones_like(want[..., :1])
        else:
            step = scale.cpu().double().numpy()[at][..., None] if per_token else scale.cpu().double().numpy()[:, None]
            if per_token:  # the row's own scale: its largest magnitude over the code range
                amax = np.abs(want).max(-1, keepdims=True) / (448 if fmt == "fp8" else 127)
                assert (np.abs(step - amax) <= (EXACT + 2.0**-23) * spread.max(-1, keepdims=True) / 100 + 2.0**-23 * amax).all()
            top = 448 if fmt == "fp8" else 127
            want = np.clip(want, -top * step if fmt == "fp8" else -128 * step, top * step)
            half = np.maximum(2.0**-4 * np.abs(want), 2.0**-10 * step) if fmt == "fp8" else 0.5 * step
            bound = half * (1 + 2.0**-20) + (EXACT + 2.0**-22) * spread + 2.0**-22 * np.abs(want)
        err = np.abs(stored * step - want)
        assert (err <= bound).all(), f"{(err - bound).max():.3e} over the bound"
        keep = np.ones((nb, page), dtype=bool)
        keep[at] = False
        raw = lambda t: t.contiguous().view(torch.uint8).cpu().numpy()  # noqa: E731
        assert np.array_equal(raw(cache)[keep], raw(old)[keep])
        if per_token:
            assert np.array_equal(scale.cpu().numpy()[keep], old_scale.cpu().numpy()[keep])
        elif scale is not None:
            assert torch.equal(scale, old_scale)


def test_append_matches_quantize_append_on_unrotated_rows():
    """Position 0 turns nothing: the stored codes and scales are quantize_append's, bit for bit."""
    from bpt_amd import quantize_append, rotary_append

    for fmt, per_token in (("bf16", False), ("fp8", False), ("fp8", True), ("int8", True)):
        b, n, hkv, d = 2, 9, 4, 128
        q, k, v = (rows((b, n, hkv, d), torch.bfloat16, s) for s in (1, 2, 3))
        one, two = pools(fmt, 3, 16, hkv, d, per_token), pools(fmt, 3, 16, hkv, d, per_token)
        slots = torch.randperm(48, generator=torch.Generator().manual_seed(1))[: b * n].reshape(b, n).to(DEV, torch.int32)
        zero = torch.zeros((b, n), dtype=torch.int64, device=DEV)
        out = rotary_append(q, k, v, zero, freqs(64), *one, slots // 16, slots % 16)
        quantize_append(k, v, *two, slots // 16, slots % 16)
        torch.cuda.synchronize()
        assert torch.equal(out, q)
        for x, y in zip(one, two):
            assert (x is None and y is None) or torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


SCALES = [1.0, 0.0137, 3e-5, 7.7, 2.0**-10, 1e-12, 2.0**101, 2.0**127, 3e38, 2.0**-101, 1e-39, 0.0, -0.25, float("inf"), float("nan")]


def stored_alike(fmt, per_token, x, scales):
    """rotary_append stores the values x [N, D] under every scale as quantize_append does, bit for bit (any NaN as any other)."""
    from bpt_amd import quantize_append, rotary_append

    heads = 1 if per_token else len(scales)
    n, d = x.shape
    v = x[None, :, None].expand(1, n, heads, d).contiguous()
    q, nb = torch.zeros_like(v), -(-n // 16)
    at = torch.arange(n, device=DEV, dtype=torch.int32)[None]
    got, want = [], []
    for out in (got, want):
        k_cache, v_cache, ks, vs = pools(fmt, nb, 16, heads, d, per_token)
        if fmt != "bf16" and not per_token:
            ks, vs = torch.ones(heads, device=DEV), torch.tensor(scales, device=DEV)
        if out is got:
            rotary_append(q, torch.zeros_like(v), v, at, freqs(d // 2), k_cache, v_cache, ks, vs, at // 16, at % 16)
        else:
            quantize_append(torch.zeros_like(v), v, k_cache, v_cache, ks, vs, at // 16, at % 16)
        torch.cuda.synchronize()
        out += [v_cache.float(), v_cache.view(torch.uint8)] + ([vs] if per_token else [])
    if per_token:
        # The maximum of a row with a signalling NaN depends on the order it is taken in: max(x, sNaN) is a NaN, which max(NaN, y)
        # then drops. Such rows are left out.
        bits, top = (x.view(torch.int16).int() & 0x7FFF), {torch.bfloat16: (0x7F80, 0x40), torch.float16: (0x7C00, 0x200)}[x.dtype]
        keep = torch.ones(nb * 16, dtype=torch.bool, device=DEV)
        keep[:n] = ~((bits > top[0]) & (bits & top[1] == 0)).any(-1)
        for out in (got, want):
            out[:] = [t.flatten(0, 1)[keep] for t in out]
    nan = torch.isnan(got[0])
    assert torch.equal(nan, torch.isnan(want[0]))
    each = nan.repeat_interleave(got[1].shape[-1] // d, -1)
    bad = (got[1] != want[1]) & ~each
    assert not bad.any(), f"{int(bad.sum())} codes differ, first at {bad.nonzero()[0].tolist()}"
    assert all(torch.equal(a, b) for a, b in zip(got[2:], want[2:]))


@pytest.mark.parametrize("fmt, per_token", [("bf16", False), ("fp8", False), ("fp8", True), ("int8", False), ("int8", True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_is_stored_as_quantize_append_stores_it(fmt, per_token, dtype):
    bits = torch.arange(65536, dtype=torch.int32, device=DEV).to(torch.int16).view(dtype)
    stored_alike(fmt, per_token, bits.reshape(512, 128), SCALES)
    stored_alike(fmt, per_token, bits.reshape(128, 512).T.reshape(512, 128), SCALES)  # magnitudes far apart in a row


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_values_next_to_the_midpoints_of_codes(fmt):
    """Where a product with the scale's reciprocal and the division could round apart."""
    if fmt == "fp8":
        codes = torch.arange(127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
        mid = (codes[1:] + codes[:-1]) / 2
    else:
        mid = torch.arange(127, device=DEV).double() + 0.5
    scales = [s for s in SCALES if 0 < s < 2.0**100] + [0.3 + 0.0007 * i for i in range(24)]
    for s in scales:
        near = (mid * float(np.float32(s))).float()
        up = torch.nextafter(near, torch.full_like(near, float("inf")))
        down = torch.nextafter(near, torch.zeros_like(near))
        x = torch.cat([near, up, down, -near, -up, -down, torch.zeros(24 if len(mid) == 126 else 6, device=DEV)])
        x = torch.cat([x, torch.zeros(-len(x) % 128, device=DEV)]).reshape(-1, 128)
        stored_alike(fmt, False, x, [s])


def test_nan_and_infinity_stay_in_their_pair():
    from bpt_amd import rotary_embed

    q = rows((1, 2, 2, 64), torch.float32, 0)
    q[0, 0, 0, 3], q[0, 1, 1, 40] = float("nan"), float("inf")
    pos = torch.tensor([[5, 9]], dtype=torch.int32, device=DEV)
    got, _ = rotary_embed(q, None, pos, freqs(16))
    torch.cuda.synchronize()
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 0, 0, [3, 19]] = True
    want[0, 1, 1, 40] = True  # past rotary_dim: as it is
    assert torch.equal(bad, want) and got[0, 1, 1, 40] == float("inf")


def test_empty_calls():
    from bpt_amd import rotary_append, rotary_embed

    q, k = rows((0, 3, 4, 64), torch.bfloat16, 0), rows((0, 3, 2, 64), torch.bfloat16, 0)
    pos = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    a, b = rotary_embed(q, k, pos, freqs(32))
    assert a.shape == q.shape and b.shape == k.shape
    cache = torch.zeros((1, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    assert rotary_append(q, k, k, pos, freqs(32), cache, cache.clone(), None, None, slots, slots).shape == q.shape


def test_on_a_stream_and_in_a_graph():
    from bpt_amd import rotary_append, rotary_embed

    b, n, hq, hkv, d = 4, 1, 16, 8, 128
    q, k, v = rows((b, n, hq, d), torch.bfloat16, 1), rows((b, n, hkv, d), torch.bfloat16, 2), rows((b, n, hkv, d), torch.bfloat16, 3)
    pos = torch.tensor([[7], [1], [900], [31]], dtype=torch.int64, device=DEV)
    inv = freqs(64)
    wb, wo = torch.arange(b, device=DEV, dtype=torch.int32)[:, None], torch.zeros((b, 1), device=DEV, dtype=torch.int32)
    kc, vc, ks, vs = pools("int8", b, 16, hkv, d, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = rotary_embed(q, k, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_append(q, k, v, pos, inv, kc, vc, ks, vs, wb, wo)
    for step in range(3):
        pos += step
        q.copy_(rows((b, n, hq, d), torch.bfloat16, 20 + step))
        graph.replay()
        want, _ = rotary_embed(q, k, pos, inv)
        other = pools("int8", b, 16, hkv, d, True)
        rotary_append(q, k, v, pos, inv, *other, wb, wo)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(kc[:, 0], other[0][:, 0]) and torch.equal(ks[:, 0], other[2][:, 0]) and torch.equal(vc[:, 0], other[1][:, 0])
    want = orot.rotate(k.double().cpu().numpy(), np.array([[[7], [1], [900], [31]]]), inv.cpu().numpy())
    within(eager[1], want, orot.spread(k.double().cpu().numpy(), inv.cpu().numpy()))


def test_pools_past_2_to_31_bytes():
    """A slot whose byte offset passes 32 bits is written where it lies."""
    from bpt_amd import rotary_append

    nb, page, hkv, d = 2300, 1024, 8, 128
    kc = torch.zeros((nb, page, hkv, d), dtype=torch.int8, device=DEV).view(torch.float8_e4m3fn)
    vc = kc.clone()
    scale = torch.ones(hkv, device=DEV)
    q, k = rows((1, 1, 8, d), torch.bfloat16, 1), rows((1, 1, hkv, d), torch.bfloat16, 2)
    zero = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    rotary_append(q, k, k, zero, freqs(64), kc, vc, scale, scale, zero + nb - 1, zero + page - 1)
    torch.cuda.synchronize()
    assert kc.numel() > 1 << 31
    assert torch.equal(kc[-1, -1].view(torch.uint8), k[0, 0].float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert int(kc.view(torch.uint8).view(torch.int64).ne(0).sum()) <= hkv * d // 8
