"""GPU: paged_masked_attention against the float64 oracle.

Tolerances: a score is off by `slack` (oracle/masked.py: float32 products and sums, the cap, the bias); a weight then by that
and by 2^-16 (two bf16 parts, each rounded to 8 bits: 2^-9 twice, 2^-18, and the float32 exponential), the sums of T terms by
T 2^-24 each, numerator and denominator alike. So an output is off by at most (2 slack + 2^-15 + T 2^-23) of the weighted mean of
|v|, and by half a step of its type.
"""

import numpy as np
import pytest
import torch

from oracle import masked as omask

pytestmark = pytest.mark.gpu

DEV = "cuda"
D = 128
FORMATS = [("bf16", False), ("fp8", False), ("fp8", True), ("int8", False), ("int8", True)]


class Case:
    """A paged cache of random values and one call over it."""

    def __init__(self, fmt, per_token, lens, nq=1, hq=4, hkv=2, page=16, q_dtype=torch.bfloat16, seed=0, head_major=False,
                 table=torch.int32, spare=1, amp=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        b, per_seq = len(lens), max(1, -(-max(lens, default=0) // page)) + spare
        nb = b * per_seq + 3
        shape = (nb, hkv, page, D) if head_major else (nb, page, hkv, D)
        x = [torch.randn(shape, generator=g, device=DEV) * amp for _ in range(2)]
        x = [t.transpose(1, 2) if head_major else t for t in x]
        self.k_scale = self.v_scale = None
        if fmt == "bf16":
            self.k, self.v = (t.to(torch.bfloat16) for t in x)
        else:
            top, dtype = (448.0, torch.float8_e4m3fn) if fmt == "fp8" else (127.0, torch.int8)
            scales = [(t.abs().amax(-1) if per_token else t.abs().amax(dim=(0, 1, 3))) / top for t in x]
            self.k_scale, self.v_scale = (s.contiguous() for s in scales)
            codes = [t / (s[..., None] if per_token else s[:, None]) for t, s in zip(x, (self.k_scale, self.v_scale))]
            self.k, self.v = (c.clamp(-top, top).to(dtype) if fmt == "fp8" else c.round().clamp(-127, 127).to(dtype) for c in codes)
        ids = torch.randperm(nb, generator=g, device=DEV)
        self.table = ids[: b * per_seq].reshape(b, per_seq).to(table)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.q = torch.randn((b, nq, hq, D), generator=g, device=DEV).to(q_dtype)
        self.fmt, self.per_token, self.max_context = fmt, per_token, max(max(lens, default=0), 1)

    def values(self):
        out = []
        for codes, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = codes.float().double()
            if scale is not None:
                x = x * (scale.double()[..., None] if self.per_token else scale.double()[:, None])
            out.append(x.cpu().numpy())
        return out

    def call(self, scale=0.11, **how):
        from bpt_amd import paged_masked_attention

        how.setdefault("max_context", self.max_context)
        return paged_masked_attention(self.q, self.k, self.v, self.table, self.lens, self.k_scale, self.v_scale, scale=scale, **how)

    def oracle(self, scale=0.11, lens=None, **how):
        k, v = self.values()
        host = {n: t.cpu().numpy() if torch.is_tensor(t) else t for n, t in how.items()}
        host["prefix"] = host.pop("prefix_lens", None)
        lens = self.lens.cpu().numpy() if lens is None else lens
        return omask.attend(self.q.double().cpu().numpy(), k, v, self.table.cpu().numpy(), lens, np.float64(np.float32(scale)), **host)

    def check(self, scale=0.11, out_dtype=torch.bfloat16, **how):
        lse = torch.full(self.q.shape[:3], 7.0, device=DEV)
        got = self.call(scale, out_dtype=out_dtype, lse=lse, **how)
        torch.cuda.synchronize()
        compare(got, lse, *self.oracle(scale, **{k: v for k, v in how.items() if k not in ("max_context", "max_prefix")}), self.max_context)


def compare(got, lse, want, want_lse, spread, slack, tokens):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    rel = (2 * slack + 2.0**-15 + tokens * 2.0**-23)[..., None]
    bound = rel * spread * (1 + half) + half * np.abs(want) + 2.0**-25
    with np.errstate(invalid="ignore"):
        err = np.where((got == want) | np.isnan(want), 0.0, np.abs(got - want))
    assert (err <= np.where(np.isnan(bound), np.inf, bound)).all(), f"{np.nanmax(err - bound):.3e} over the bound"
    if lse is not None:
        lse = lse.double().cpu().numpy()
        seen = np.isfinite(want_lse)
        assert np.array_equal(np.isneginf(lse), np.isneginf(want_lse))
        off = np.abs(lse[seen] - want_lse[seen])
        assert (off <= slack[seen] + 2.0**-18 + tokens * 2.0**-24 + np.abs(want_lse[seen]) * 2.0**-22).all()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slopes_of(hq):
    return 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq)


MASKS = {
    "causal": lambda c: {},
    "cap": lambda c: dict(softcap=3.0),
    "bias": lambda c: dict(slopes=slopes_of(c.q.shape[2])),
    "window": lambda c: dict(window=20),
    "prefix": lambda c: dict(prefix_lens=i32([(7 + 29 * i) % (c.max_context + 5) for i in range(len(c.lens))])),
    "documents": lambda c: dict(starts=(c.lens[:, None] - c.q.shape[1] + torch.arange(c.q.shape[1], device=DEV, dtype=torch.int32)) // 37 * 37),
    "all": lambda c: dict(softcap=2.0, slopes=slopes_of(c.q.shape[2]), window=45, prefix_lens=i32([3] * len(c.lens)), max_prefix=33,
                          starts=torch.full(c.q.shape[:2], 11, device=DEV, dtype=torch.int32)),
}


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("fmt, per_token", FORMATS)
@pytest.mark.parametrize("nq, hq, hkv, q_dtype, out", [
    (1, 2, 2, torch.bfloat16, torch.bfloat16),   # one row
    (5, 6, 2, torch.float16, torch.float32),     # 15 rows of 16
    (4, 10, 2, torch.bfloat16, torch.float16),   # 20 rows: two row tiles in a wave
    (11, 3, 1, torch.bfloat16, torch.float32),   # 33 rows: four waves, 64-row tiles
    (67, 2, 1, torch.float16, torch.float16),    # 134 rows: two 128-row tiles, the second nearly empty
])
def test_masks(mask, fmt, per_token, nq, hq, hkv, q_dtype, out):
    c = Case(fmt, per_token, [150, 0, 1, 33, 67, 300], nq, hq, hkv, q_dtype=q_dtype, seed=nq)
    c.check(out_dtype=out, **MASKS[mask](c))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 127, 129, 260])
def test_rows_and_lengths(rows, length):
    c = Case("fp8", False, [length], rows, 1, 1, seed=rows + length)
    c.check(softcap=5.0, window=max(length // 2, 1))


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 128, 1024])
@pytest.mark.parametrize("fmt, per_token", [("bf16", False), ("fp8", True), ("int8", True)])
@pytest.mark.parametrize("nq", [1, 40])
def test_pages_and_layouts(page, fmt, per_token, nq):
    for head_major, table in ((False, torch.int64), (True, torch.int32)):
        c = Case(fmt, per_token, [75, 300, 31], nq, 4, 2, page=page, head_major=head_major, table=table, seed=page)
        c.check(prefix_lens=i32([10, 40, 99]), window=50, slopes=slopes_of(4))


@pytest.mark.parametrize("fmt, per_token", FORMATS)
@pytest.mark.parametrize("nq, hq", [(1, 8), (3, 8), (90, 2)])
def test_split_over_many_pieces(fmt, per_token, nq, hq):
    """A few long sequences: every tile is cut into pieces that meet in the workspace."""
    c = Case(fmt, per_token, [5003, 129, 2600], nq, hq, 2, seed=3)
    c.check(softcap=4.0, slopes=slopes_of(hq) / 64)
    c.check(window=700, prefix_lens=i32([130, 1, 2000]))


@pytest.mark.parametrize("nq, hq", [(1, 2), (1, 4), (1, 6), (1, 10), (1, 16), (1, 18), (2, 20), (100, 2)])
@pytest.mark.parametrize("mask", ["causal", "steep", "prefix"])
def test_long_sequences_of_few_heads(nq, hq, mask):
    """Dozens of pieces a row, shared out among the threads that combine them where there are few rows."""
    c = Case("fp8", False, [9000, 2100], nq, hq, 2, seed=hq)
    how = {"causal": {}, "steep": dict(slopes=torch.full((hq,), 0.3, device=DEV)),
           "prefix": dict(prefix_lens=i32([100, 2100]), starts=torch.full((2, nq), 8500, device=DEV, dtype=torch.int32))}[mask]
    c.check(out_dtype=torch.float32, **how)
    once = c.call(**how)
    assert torch.equal(once, c.call(**how))


def test_nan_reaches_its_row_through_many_pieces():
    for hq in (2, 10):
        c = Case("bf16", False, [9000], 1, hq, 2, seed=2)
        clean = c.call()
        c.q[0, 0, 1, 7] = float("nan")
        got = c.call()
        assert torch.isnan(got[0, 0, 1]).all()
        got[0, 0, 1] = clean[0, 0, 1]
        assert torch.equal(got, clean)


def test_pieces_are_combined_in_order():
    """The same call gives the same bits, whichever piece comes last."""
    c = Case("fp8", False, [9000, 8000, 77], 2, 8, 2)
    first = c.call(softcap=4.0)
    for _ in range(20):
        assert torch.equal(c.call(softcap=4.0), first)


def test_rows_that_see_nothing():
    """Starts past the position, and queries before the sequence: zeros and -inf, whatever the other rows see."""
    for nq, hq in ((4, 4), (70, 2)):
        c = Case("bf16", False, [40, 2, 0, 90], nq, hq, 2, seed=1)
        starts = torch.zeros((4, nq), dtype=torch.int32, device=DEV)
        starts[0, ::2], starts[3] = 1000, 2**31 - 1
        c.check(starts=starts)
        c.check(starts=starts, prefix_lens=i32([0, 5, 5, -3]), window=1)
        lse = torch.zeros((4, nq, hq), device=DEV)
        out = c.call(starts=starts, lse=lse)
        assert (out[3] == 0).all() and torch.isneginf(lse[3]).all() and (out[2] == 0).all()


def test_lengths_past_the_bounds_are_cut():
    c = Case("bf16", False, [100, 100], 2, 2, 1)
    c.lens = i32([64, 90])
    want = c.call(max_context=64)
    c.lens = i32([100, 90])
    got = c.call(max_context=64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.lens = i32([-5, 64])
    assert (c.call(max_context=64)[0] == 0).all()
    c.lens = i32([100, 100])  # a prefix past max_prefix is cut to it
    assert torch.equal(c.call(prefix_lens=i32([99, 20]), max_prefix=20, window=3), c.call(prefix_lens=i32([20, 20]), window=3))


@pytest.mark.parametrize("fmt, per_token", FORMATS)
@pytest.mark.parametrize("nq, hq", [(2, 4), (3, 16), (40, 2)])
def test_what_is_not_seen_adds_nothing(fmt, per_token, nq, hq):
    """NaN and infinities in slots that no query sees change no bit; one that only later queries see reaches only them."""
    c = Case(fmt, per_token, [120, 61], nq, hq, 2, seed=9)
    how = dict(window=30, prefix_lens=i32([5, 0]), softcap=6.0)
    clean = c.call(**how)
    hidden = [(0, j) for j in (5, 20, 119 - nq - 30)] + [(1, 61), (1, 63)]  # (sequence, token), unseen

    def poison(where, bad):
        for b, j in where:
            e, off = int(c.table[b, j // 16]), j % 16
            for cache, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
                if fmt == "int8":
                    if per_token:
                        scale[e, off] = bad
                elif fmt == "fp8":
                    cache.view(torch.uint8)[e, off] = 0x7F
                else:
                    cache[e, off] = bad

    poison(hidden, float("nan"))
    assert torch.equal(c.call(**how), clean)
    if fmt == "bf16" or per_token:
        poison(hidden, float("inf"))
        assert torch.equal(c.call(**how), clean)
    if fmt == "int8" and not per_token:
        return
    poison([(0, 119)], float("nan"))  # the last token: the last query alone sees it
    got = c.call(**how)
    assert torch.equal(got[0, :-1], clean[0, :-1]) and torch.equal(got[1], clean[1])
    assert torch.isnan(got[0, -1]).all()


@pytest.mark.parametrize("nq, hq", [(2, 4), (40, 2)])
def test_infinite_values_reach_the_rows_that_see_them(nq, hq):
    c = Case("bf16", False, [70], nq, hq, 2, seed=2)
    clean = c.call(softcap=6.0)
    e, off = int(c.table[0, 69 // 16]), 69 % 16
    c.v[e, off, 0, 5], c.v[e, off, 1, 77] = float("inf"), float("-inf")
    got = c.call(softcap=6.0)
    want = clean.clone()
    want[0, -1, : hq // 2, 5], want[0, -1, hq // 2 :, 77] = float("inf"), float("-inf")
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite) and torch.equal(got[~finite], want[~finite])
    assert torch.allclose(got[finite].float(), want[finite].float(), rtol=2**-7, atol=2**-10)
    c.check(softcap=6.0)


def test_nan_queries_stay_in_their_row():
    for nq, hq in ((3, 4), (40, 4)):
        c = Case("fp8", False, [90], nq, hq, 2, seed=2)
        clean = c.call()
        c.q[0, 1, 2, 7] = float("nan")
        got = c.call()
        assert torch.isnan(got[0, 1, 2]).all()
        got[0, 1, 2] = clean[0, 1, 2]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_queries_meet_the_cap(dtype):
    """Scores of plus and minus infinity are the cap and its negative."""
    for nq, hq in ((2, 4), (40, 4)):
        c = Case("bf16", False, [90], nq, hq, 2, seed=2, q_dtype=dtype)
        c.q[0, 1, 2, 7] = float("inf")
        c.check(softcap=2.0, out_dtype=torch.float32)


@pytest.mark.parametrize("cap", [1e-3, 0.5, 200.0, 300.0, 1e4, 1e30])
def test_caps_of_every_size(cap):
    """Caps past 256 take the other form of tanh; a cap far above the scores changes nothing but rounding."""
    c = Case("bf16", False, [200], 2, 4, 2, seed=4, amp=3.0)
    c.check(scale=0.7, softcap=cap, out_dtype=torch.float32)


def test_scores_far_apart_and_negative_scales():
    c = Case("bf16", False, [400], 1, 4, 2, seed=4, amp=20.0)
    c.check(scale=3.0, out_dtype=torch.float32)
    c.check(scale=-0.2, softcap=30.0, out_dtype=torch.float32)
    c.check(scale=0.0, slopes=slopes_of(4), out_dtype=torch.float32)


@pytest.mark.parametrize("big", [2.0**70, 2.0**-70])
def test_value_scales_of_every_size(big):
    c = Case("int8", True, [100], 2, 4, 2, seed=4)
    c.v_scale *= big
    k, v = c.values()
    got = c.call(out_dtype=torch.float32).double().cpu().numpy()
    want, _, spread, slack = c.oracle()
    assert (np.abs(got - want) <= (2 * slack + 2.0**-15 + 2.0**-16)[..., None] * spread).all()


def test_views_and_outputs():
    """3-D q, strided q and out; what lies around out is left alone."""
    c = Case("bf16", False, [50, 60], 1, 4, 2)
    want = c.call()
    wide = torch.zeros((2, 1, 4, 3 * D), dtype=torch.bfloat16, device=DEV)
    wide[..., D : 2 * D] = c.q
    c.q = wide[..., D : 2 * D]
    buf = torch.full((2, 1, 4, D + 6), 9.0, dtype=torch.bfloat16, device=DEV)
    out = buf[..., 3 : 3 + D]
    assert c.call(out=out) is out
    assert torch.equal(out, want) and (buf[..., :3] == 9).all() and (buf[..., 3 + D :] == 9).all()
    c.q = c.q[:, 0]
    assert torch.equal(c.call(), want[:, 0])
    m = Case("fp8", False, [300], 80, 2, 1)
    want = m.call(window=9)
    buf = torch.full((1, 2, 80, D + 6), 9.0, dtype=torch.bfloat16, device=DEV)
    out = buf.transpose(1, 2)[..., 3 : 3 + D]
    m.call(window=9, out=out)
    assert torch.equal(out, want) and (buf[..., :3] == 9).all() and (buf[..., 3 + D :] == 9).all()


def test_an_expanded_output_is_refused():
    c = Case("bf16", False, [40, 7])
    with pytest.raises(ValueError, match="expanded"):
        c.call(out=torch.zeros((1, *c.q.shape[1:]), device=DEV, dtype=torch.bfloat16).expand(c.q.shape))


def test_empty_batch_and_no_context():
    c = Case("bf16", False, [], 3, 4, 2)
    assert c.call().shape == (0, 3, 4, D)
    c = Case("fp8", False, [0, 0], 3, 4, 2)
    assert (c.call(max_context=0) == 0).all()


def test_pools_past_2_to_31_bytes():
    c = Case("fp8", False, [200], 1, 4, 2)
    nb, page = 9000, 1024
    big = [torch.zeros((nb, page, 2, D), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    for x, small in zip(big, (c.k, c.v)):
        pages = torch.cat([small.view(torch.uint8)[int(e)] for e in c.table[0]])[:page]
        x.view(torch.uint8)[nb - 1, : pages.shape[0]] = pages
    want = c.call(softcap=4.0)
    c.k, c.v, c.table = *big, i32([[nb - 1]])
    assert c.k.numel() > 1 << 31
    assert torch.equal(c.call(softcap=4.0), want)


def test_two_streams_at_once():
    c, d = Case("fp8", False, [4000] * 4, 1, 8, 2), Case("int8", True, [3000] * 4, 1, 8, 2)
    want = c.call(softcap=4.0), d.call(window=999)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s):
            a = c.call(softcap=4.0)
        with torch.cuda.stream(t):
            b = d.call(window=999)
        got.append((a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_two_graphs_replayed_at_once():
    """Each captured call has partials and counters of its own, so graphs of one capture stream may overlap."""
    c, d = Case("fp8", False, [4000] * 4, 1, 8, 2), Case("bf16", False, [3000] * 4, 2, 8, 2)
    c.call(softcap=4.0), d.call(window=999)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, case, how in zip(graphs, (c, d), (dict(softcap=4.0), dict(window=999))):
        with torch.cuda.graph(graph):
            outs.append(case.call(**how))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        for case, length in ((c, 4000 - 100 * step), (d, 3000 - 10 * step)):
            case.lens.fill_(length)
            case.q.copy_(torch.randn(case.q.shape, device=DEV).to(case.q.dtype))
        want = c.call(softcap=4.0), d.call(window=999)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_callers_own_buffers():
    from bpt_amd import masked_plan

    c = Case("fp8", False, [4000] * 2, 1, 8, 2)
    ws, cnt = masked_plan(c.q, c.k, c.v, c.table, c.lens, c.k_scale, c.v_scale, scale=0.11, max_context=4000, softcap=4.0)
    assert ws > 0 and cnt > 0
    workspace, counters = torch.empty(ws, dtype=torch.uint8, device=DEV), torch.zeros(cnt, dtype=torch.uint8, device=DEV)
    want = c.call(softcap=4.0)
    for _ in range(3):
        assert torch.equal(c.call(softcap=4.0, workspace=workspace, counters=counters), want)
    torch.cuda.synchronize()
    assert int(counters.sum()) == 0
    with pytest.raises(ValueError, match="workspace"):
        c.call(softcap=4.0, workspace=workspace[:-256], counters=counters)
    with pytest.raises(ValueError, match="counter"):
        c.call(softcap=4.0, workspace=workspace, counters=counters[:0])


def test_unmasked_calls_agree_with_paged_decode_attention():
    from bpt_amd import paged_decode_attention

    for fmt, per_token in FORMATS:
        c = Case(fmt, per_token, [500, 77], 3, 8, 2)
        a = c.call(out_dtype=torch.float32)
        b = paged_decode_attention(c.q, c.k, c.v, c.table, c.lens, c.k_scale, c.v_scale, scale=0.11, max_context=500, out_dtype=torch.float32)
        _, _, spread, slack = c.oracle()
        assert ((a - b).abs().double().cpu().numpy() <= 2 * (2 * slack + 2.0**-15 + 2.0**-14)[..., None] * spread).all()
