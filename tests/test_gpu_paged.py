"""Paged-cache operators against plain 64-bit forms, on the GPU.

Tolerances come from counting roundings (u = eps / 2 of the output type, 2^-24
for f32 arithmetic) and are computed from each case's own values:

* append: the angle is reduced in 64 bits and rounded to f32 in turns (at most
  2^-25 of a turn, 2 pi 2^-25 < 2^-22 rad), sin and cos add 2^-23 each, the two
  products and their sum 3 * 2^-24, so a rotated element is off by at most
  2^-21 (|x1| + |x2|) scale before its own rounding.  Copies are exact.
* attend: a score is off by at most (head_dim + 8) 2^-24 sum |q k| scale (an f32
  sum in any order, the scale, the cap), which moves a weight by as much
  relatively; the weight itself is off by 2^-16 (exp2, and its split into two
  16-bit parts), the two sums by 2^-24 per position.  Numerator and denominator
  both carry it: twice that times max |v|, plus the output's rounding.
* verify: token choices must be equal (the oracle asserts that no choice of
  these inputs is nearer to its border than 1e-5); a log-probability is off by
  2^-18 (the sum of exponentials) and 2^-22 of itself.
"""
import math

import pytest
import torch

from conftest import has_gpu

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


@pytest.fixture(scope="module")
def paged():
    if not has_gpu():
        pytest.skip("no CUDA device")
    from cljxla_b200.host import paged as m
    return m


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    """A cache with random pages, a step's packed rows, and the plain forms."""

    def __init__(self, lens, counts, nkv, group, hd, page, dtype, width=None, seed=0, behind=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.counts, self.nkv, self.group, self.hd, self.page = lens, counts, nkv, group, hd, page
        self.dtype = TYPES[dtype]
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        need = [-(-n // page) for n in lens]
        self.width = max(need + [1]) if width is None else width
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            m = min(n, self.width)
            self.table[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
            at += n
        rows = self.starts[-1] + behind
        rnd = lambda *s: torch.randn(s, generator=g)
        self.k = rnd(self.pages, nkv, page, hd).to(self.dtype)
        self.v = rnd(self.pages, nkv, page, hd).to(self.dtype)
        self.q = (rnd(rows, nkv * group, hd) * spread).to(self.dtype)
        self.kn = rnd(rows, nkv, hd).to(self.dtype)
        self.vn = rnd(rows, nkv, hd).to(self.dtype)

    def cache(self, paged, k=None, v=None):
        self.dk = self.k.cuda() if k is None else k
        self.dv = self.v.cuda() if v is None else v
        self.dtable, self.dlens = self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.dstarts = torch.tensor(self.starts, dtype=torch.int32).cuda()
        return paged.PagedKV(self.dk, self.dv, self.dtable, self.dlens)

    def page_at(self, b, j):
        if not 0 <= j < self.width * self.page:
            return None
        p = int(self.table[b, j // self.page])
        return p if 0 <= p < self.pages else None

    def rows(self):
        """(row, sequence, position) of every packed row."""
        for b, c in enumerate(self.counts):
            for i in range(c):
                yield self.starts[b] + i, b, self.lens[b] - c + i

    def attend(self, scale, softcap, window, most=None):
        """(value, tolerance before the output's rounding), None for rows that are not computed."""
        want, tol = [None] * self.q.shape[0], [None] * self.q.shape[0]
        k, v, q = self.k.double(), self.v.double(), self.q.double()
        for r, b, pos in self.rows():
            if most is not None and r - self.starts[b] >= most:
                continue
            lo = 0 if window < 0 else max(0, pos - window)
            seen = [(self.page_at(b, j), j % self.page) for j in range(lo, pos + 1)]
            seen = [(p, o) for p, o in seen if p is not None]
            if not seen:
                want[r] = torch.zeros(self.nkv * self.group, self.hd, dtype=torch.float64)
                tol[r] = torch.zeros(self.nkv * self.group, 1, dtype=torch.float64)
                continue
            ps, os = (torch.tensor(x) for x in zip(*seen))
            kk, vv = k[ps, :, os], v[ps, :, os]  # [n, nkv, hd]
            qq = q[r].view(self.nkv, self.group, self.hd)
            s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
            size = torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()).amax(-1) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                size = size + 4 * softcap
            w = torch.softmax(s, -1)
            want[r] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(-1, self.hd)
            one = (self.hd + 8) * 2.0 ** -24 * size + 2.0 ** -16 + len(seen) * 2.0 ** -24
            tol[r] = (2 * one * vv.abs().amax(0).amax(-1)[:, None]).reshape(-1, 1)
        return want, tol


def check_rows(out, want, tol, before=None):
    got, u = out.double().cpu(), half_step(out.dtype)
    tiny = 2.0 ** -25 if out.dtype is torch.float16 else 0.0
    for r, w in enumerate(want):
        if w is None:
            if before is not None:
                assert torch.equal(out[r].cpu(), before[r].cpu()), f"row {r} was written"
            continue
        err = (got[r] - w).abs()
        lim = tol[r] + u * (w.abs() + tol[r]) + tiny
        assert not torch.isnan(got[r]).any(), f"row {r} has NaN"
        assert bool((err <= lim).all()), f"row {r}: off by {float((err - lim).max()):.3g} more than allowed"


ATTEND = {
    # name: (lens, counts, nkv, group, hd, page, dtype, out, window, softcap)
    "one_position": ([1], [1], 1, 1, 64, 16, "bf16", "bf16", -1, 0.0),
    "f32_mha": ([257, 3], [1, 1], 3, 1, 64, 16, "f32", "f32", -1, 0.0),
    "f32_hd32": ([100, 33, 1], [1, 1, 1], 2, 4, 32, 7, "f32", "f32", -1, 0.0),
    "f32_hd128_drafts": ([300, 31, 5], [3, 1, 5], 2, 2, 128, 32, "f32", "f32", 40, 0.0),
    "f32_hd256": ([130, 64], [2, 1], 1, 8, 256, 5, "f32", "f32", -1, 20.0),
    "bf16_gqa": ([640, 65, 64, 63], [1, 1, 1, 1], 4, 2, 256, 64, "bf16", "bf16", -1, 0.0),
    "bf16_f32out": ([640, 1, 17], [1, 1, 1], 4, 2, 256, 64, "bf16", "f32", -1, 0.0),
    "bf16_hd128": ([1025, 16, 15], [1, 1, 1], 2, 8, 128, 16, "bf16", "f32", -1, 0.0),
    "bf16_hd32": ([500, 2], [1, 1], 3, 3, 32, 16, "bf16", "f32", -1, 0.0),
    "bf16_hd64_window0": ([500, 1], [1, 1], 2, 2, 64, 16, "bf16", "f32", 0, 0.0),
    "bf16_window": ([900, 100, 40], [1, 1, 1], 2, 4, 128, 16, "bf16", "bf16", 100, 0.0),
    "bf16_softcap": ([900, 100, 40], [1, 1, 1], 2, 2, 256, 16, "bf16", "f32", -1, 50.0),
    "f16_drafts": ([333, 70, 5, 1], [5, 3, 5, 1], 2, 2, 256, 16, "f16", "f16", -1, 0.0),
    "f16_drafts_window": ([333, 70, 5, 129], [5, 3, 5, 4], 4, 4, 64, 16, "f16", "f32", 64, 0.0),
    "f16_page1": ([77, 20], [2, 1], 2, 3, 64, 1, "f16", "f16", -1, 0.0),
    "bf16_rows32": ([200, 90], [4, 3], 1, 8, 128, 128, "bf16", "f32", -1, 0.0),
    "bf16_rows64": ([200, 90], [8, 8], 2, 8, 256, 16, "bf16", "bf16", 33, 30.0),
    "bf16_rows_odd": ([150, 90, 33], [7, 2, 33], 1, 9, 64, 16, "bf16", "f32", -1, 0.0),
    "bf16_prompt": ([150, 97], [150, 40], 2, 2, 64, 16, "bf16", "f32", -1, 0.0),
    "f32_prompt": ([90], [80], 1, 3, 128, 16, "f32", "f32", 16, 0.0),
    "bf16_hd32_rows64": ([70, 10], [20, 10], 1, 3, 32, 16, "bf16", "f32", -1, 0.0),
    "f32_hd32_rows64": ([70, 10], [20, 10], 1, 3, 32, 16, "f32", "f32", -1, 0.0),
    "empty_sequences": ([0, 50, 0, 7], [0, 1, 0, 2], 2, 2, 64, 16, "bf16", "f32", -1, 0.0),
    "rows_before_position_0": ([2, 0, 30], [5, 3, 1], 2, 2, 128, 16, "bf16", "f32", -1, 0.0),
    "f32_1row_hd128": ([300, 65, 1, 64], [1, 1, 1, 1], 2, 1, 128, 16, "f32", "f32", 100, 0.0),
    "f32_1row_hd256": ([300, 33, 1, 32], [1, 1, 1, 1], 2, 1, 256, 7, "f32", "f32", -1, 30.0),
    "f32_2rows_hd64": ([900, 65, 2, 64], [2, 1, 2, 2], 2, 1, 64, 16, "f32", "f32", 70, 0.0),
    "f32_2rows_hd256": ([300, 65, 2, 64], [1, 1, 1, 1], 2, 2, 256, 16, "f32", "f32", -1, 0.0),
    "f32_3rows_hd32": ([300, 65, 3, 64], [3, 2, 3, 1], 3, 1, 32, 1, "f32", "f32", 20, 0.0),
    "f32_4rows_hd128": ([700, 65, 2, 64], [2, 1, 2, 2], 3, 2, 128, 16, "f32", "f32", 33, 25.0),
    "f32_4rows_before_0": ([2, 0, 30, 0], [4, 3, 1, 0], 2, 1, 64, 16, "f32", "f32", -1, 0.0),
    "long_f32": ([5000, 4097], [1, 2], 2, 2, 64, 16, "f32", "f32", -1, 0.0),
    "many_pieces": ([1 + (37 * i) % 200 for i in range(90)], [1 + i % 3 if 1 + (37 * i) % 200 > 3 else 1 for i in range(90)],
                    8, 2, 128, 16, "bf16", "f32", -1, 0.0),
    "many_pieces_f32": ([1 + (37 * i) % 200 for i in range(90)], [1 for i in range(90)], 8, 2, 64, 16, "f32", "f32", 64, 0.0),
    "long": ([5000, 4097], [1, 2], 2, 2, 128, 16, "bf16", "f32", -1, 0.0),
}


@pytest.mark.parametrize("name", list(ATTEND))
def test_attend_matches_plain_form(paged, name):
    lens, counts, nkv, group, hd, page, dtype, out, window, softcap = ATTEND[name]
    case = Case(lens, counts, nkv, group, hd, page, dtype, seed=3, behind=2, spread=2.0)
    cache = case.cache(paged)
    want, tol = case.attend(hd ** -0.5, softcap, window)
    buf = torch.full((case.q.shape[0], nkv * group, hd), 7.0, dtype=TYPES[out], device="cuda")
    before = buf.clone()
    got = cache.attend(case.q.cuda(), out=buf, starts=case.dstarts, max_tokens=max(counts), softcap=softcap, window=window)
    assert got is buf
    check_rows(got, want, tol, before)


def test_attend_without_starts_default_out_and_scale(paged):
    case = Case([90, 40, 3], [2, 2, 2], 2, 2, 64, 16, "bf16", seed=1)
    cache = case.cache(paged)
    want, tol = case.attend(0.3, 0.0, -1)
    got = cache.attend(case.q.cuda(), scale=0.3)
    assert got.dtype is torch.bfloat16
    check_rows(got, want, tol)


def test_attend_rows_past_max_tokens_are_left(paged):
    case = Case([90, 40], [4, 1], 2, 2, 64, 16, "bf16", seed=1)
    cache = case.cache(paged)
    want, tol = case.attend(0.125, 0.0, -1, most=2)
    buf = torch.full((5, 4, 64), 3.0, device="cuda")
    before = buf.clone()
    check_rows(cache.attend(case.q.cuda(), out=buf, starts=case.dstarts, max_tokens=2), want, tol, before)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_and_append_without_pages(paged, dtype):
    """A pool of no pages, and a table of no columns: rows see nothing, nothing is written."""
    case = Case([5, 40], [1, 2], 2, 2, 64, 16, dtype, seed=4)
    lens = torch.tensor(case.lens, dtype=torch.int32).cuda()
    starts = torch.tensor(case.starts, dtype=torch.int32).cuda()
    q, k, v = case.q.cuda(), case.kn.cuda(), case.vn.cuda()
    none = torch.zeros((0, 2, 16, 64), dtype=TYPES[dtype], device="cuda")
    pool = torch.full((3, 2, 16, 64), 5.0, dtype=TYPES[dtype], device="cuda")
    for pages, table in ((none, case.table.cuda()), (pool, torch.zeros((2, 0), dtype=torch.int32, device="cuda"))):
        cache = paged.PagedKV(pages, pages.clone(), table, lens)
        cache.append(k, v, starts=starts)
        out = torch.full_like(q, 3.0)
        cache.attend(q, out=out, starts=starts, max_tokens=2)
        assert bool((out == 0).all()) and bool((pool == 5.0).all())


@pytest.mark.parametrize("hd,dtype", [(128, "bf16"), (64, "f32"), (256, "f16")])
def test_attend_evicted_and_bad_pages_are_left_out(paged, hd, dtype):
    case = Case([200, 90, 40], [2, 1, 1], 2, 2, hd, 16, dtype, seed=5)
    case.table[0, :3] = -1
    case.table[0, 7] = case.pages + 5
    case.table[1, 2] = -2 ** 31
    case.table[2, :] = 2 ** 31 - 1  # nothing of this sequence is there
    cache = case.cache(paged)
    want, tol = case.attend(hd ** -0.5, 0.0, -1)
    check_rows(cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=2), want, tol)


def test_attend_length_past_the_table(paged):
    case = Case([100, 20], [1, 1], 2, 2, 64, 16, "bf16", seed=6)
    case.lens = [case.width * 16 + 9, 20]
    cache = case.cache(paged)
    want, tol = case.attend(0.125, 0.0, -1)
    check_rows(cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=1), want, tol)
    want, tol = case.attend(0.125, 0.0, 3)  # a window wholly behind the table sees nothing
    check_rows(cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=1, window=3), want, tol)


@pytest.mark.parametrize("hd,dtype,group,count", [(32, "bf16", 2, 5), (64, "f32", 2, 5), (128, "bf16", 2, 5),
                                                  (256, "f16", 2, 5), (256, "f32", 2, 5), (128, "bf16", 1, 2),
                                                  (256, "bf16", 8, 5), (64, "f32", 1, 2), (128, "f32", 2, 2),
                                                  (256, "f32", 1, 4), (32, "f32", 1, 3)])
@pytest.mark.parametrize("bad", [INF, -INF, math.nan])
def test_attend_unseen_positions_may_hold_anything(paged, hd, dtype, group, count, bad):
    """Page tails, evicted pages, positions before the window, and later drafts."""
    case = Case([77, 40], [count, min(3, count)], 2, group, hd, 16, dtype, seed=7)
    case.table[0, 0] = -1
    window = 30
    want, tol = case.attend(hd ** -0.5, 0.0, window)
    seen = {(case.page_at(b, j), j % 16) for r, b, pos in case.rows() for j in range(max(0, pos - window), pos + 1)}
    k, v = case.k.clone(), case.v.clone()
    for p in range(case.pages):
        for o in range(16):
            if (p, o) not in seen:
                k[p, :, o] = bad
                v[p, :, o] = bad
    cache = case.cache(paged, k.cuda(), v.cuda())
    check_rows(cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=count, window=window), want, tol)
    # the newest draft of sequence 0 (position 76) is unseen by its other rows, and the oldest
    # position that row 0 sees by the rows behind it
    p, o = case.page_at(0, 76), 76 % 16
    p2, o2 = case.page_at(0, 77 - count - 30), (77 - count - 30) % 16
    k[p, :, o] = bad
    v[p, :, o, 1::2] = bad
    v[p2, :, o2, 3] = bad
    cache = case.cache(paged, k.cuda(), v.cuda())
    got = cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=count, window=window)
    w2 = list(want)
    w2[0] = w2[count - 1] = None
    check_rows(got, w2, tol)
    g0 = got[0].double().cpu()
    assert not torch.isfinite(g0[:, 3]).any()  # row 0 does see that value
    keep = [d for d in range(hd) if d != 3]
    assert bool(((g0[:, keep] - want[0][:, keep]).abs() <= tol[0] + 2 * half_step(got.dtype) * want[0][:, keep].abs() + 1e-7).all())


def test_attend_extreme_scores(paged):
    """Scores far apart, all equal, and at the type's lowest value."""
    case = Case([300, 300, 300], [1, 1, 1], 1, 2, 64, 16, "bf16", seed=8)
    case.q[1] = 0.0
    case.q[0] *= 300.0
    case.q[2] = torch.finfo(torch.bfloat16).min / 64  # scores of +-1e36 times a few: one position takes all
    cache = case.cache(paged)
    want, tol = case.attend(0.125, 0.0, -1)
    tol[2] = torch.zeros_like(tol[2])
    tol[0] = tol[0].clamp(max=1e-2)
    check_rows(cache.attend(case.q.cuda(), out=torch.empty(3, 2, 64, device="cuda"), starts=case.dstarts, max_tokens=1), want, tol)


def test_attend_other_layouts(paged):
    """A [pages, page, heads, dim] pool, queries sliced from a fused projection, an output with gaps."""
    case = Case([210, 33], [3, 1], 4, 2, 128, 16, "bf16", seed=9)
    pool = torch.zeros((case.pages, 2, 16, 4, 128 + 8), dtype=torch.bfloat16, device="cuda")
    k, v = pool[:, 0].transpose(1, 2)[..., :128], pool[:, 1].transpose(1, 2)[..., :128]
    k.copy_(case.k)
    v.copy_(case.v)
    cache = case.cache(paged, k, v)
    table = torch.full((2, case.width + 5), 99, dtype=torch.int32, device="cuda")
    table[:, :case.width] = case.table.cuda()
    cache = paged.PagedKV(k, v, table[:, :case.width], case.dlens)
    fused = torch.zeros((4, 24, 128), dtype=torch.bfloat16, device="cuda")
    fused[:, 4:12] = case.q.cuda()
    out = torch.full((4, 9, 160), 5.0, device="cuda")
    want, tol = case.attend(128 ** -0.5, 0.0, -1)
    got = cache.attend(fused[:, 4:12], out=out[:, :8, 16:144], starts=case.dstarts, max_tokens=3)
    check_rows(got, want, tol)
    assert bool((out[:, 8] == 5).all() and (out[:, :, :16] == 5).all() and (out[:, :, 144:] == 5).all())


def test_attend_far_pages(paged):
    """Page offsets past 2^31 elements and past 2^32 bytes."""
    hd, page = 128, 64
    pages = (2 ** 31) // (hd * page) + 40
    pool = torch.zeros((pages, 1, page, hd), dtype=torch.bfloat16, device="cuda")
    case = Case([1000], [2], 1, 4, hd, page, "bf16", seed=10)
    far = [pages - 1 - int(p) for p in case.table[0]]
    for p, f in zip(case.table[0].tolist(), far):
        pool[f] = case.k[p].cuda()
    vpool = torch.zeros_like(pool)
    for p, f in zip(case.table[0].tolist(), far):
        vpool[f] = case.v[p].cuda()
    case.cache(paged)
    cache = paged.PagedKV(pool, vpool, torch.tensor([far], dtype=torch.int32).cuda(), case.dlens)
    want, tol = case.attend(hd ** -0.5, 0.0, -1)
    check_rows(cache.attend(case.q.cuda(), starts=case.dstarts, max_tokens=2), want, tol)
    freq = paged.rope_inv_freq(hd, device="cuda")
    cache.append(case.kn.cuda(), case.vn.cuda(), starts=case.dstarts, rope=paged.Rope(freq))
    for r, b, pos in case.rows():
        assert torch.equal(vpool[far[pos // page], 0, pos % page].cpu(), case.vn[r, 0])


def test_attend_same_result_every_time(paged):
    case = Case([4000, 700, 9], [1, 2, 1], 2, 4, 128, 16, "bf16", seed=11)
    cache = case.cache(paged)
    q = case.q.cuda()
    first = cache.attend(q, starts=case.dstarts, max_tokens=2).clone()
    for _ in range(5):
        assert torch.equal(cache.attend(q, starts=case.dstarts, max_tokens=2), first)


# ------------------------------------------------------------------- append
APPEND = {
    # name: (lens, counts, nkv, group or 0, hd, page, dtype, rotary, interleaved, scale)
    "one": ([1], [1], 4, 2, 256, 64, "bf16", 256, False, 1.0),
    "no_rope": ([9, 40], [3, 1], 2, 1, 64, 16, "f32", 0, False, 1.0),
    "half_bf16": ([300, 17, 64], [5, 1, 3], 2, 2, 128, 16, "bf16", 128, False, 1.0),
    "half_f16_part": ([300, 17, 64], [5, 1, 3], 2, 2, 256, 16, "f16", 128, False, 1.0),
    "half_f32": ([300, 17], [5, 2], 3, 2, 64, 7, "f32", 64, False, 0.7),
    "interleaved_bf16": ([300, 17, 64], [5, 1, 3], 2, 4, 64, 16, "bf16", 64, True, 1.0),
    "interleaved_f16_part": ([90, 17], [2, 3], 2, 2, 128, 1, "f16", 40, True, 1.3),
    "interleaved_f32": ([90, 17], [2, 3], 1, 5, 32, 16, "f32", 32, True, 1.0),
    "half_odd_part": ([50, 20], [3, 3], 2, 2, 64, 16, "bf16", 22, False, 1.0),
    "interleaved_odd_part": ([50, 20], [3, 3], 2, 2, 64, 16, "bf16", 22, True, 1.0),
    "f32_half_odd_part": ([50, 20], [3, 3], 2, 2, 64, 16, "f32", 6, False, 1.0),
    "keys_only": ([50, 20], [3, 3], 2, 0, 128, 16, "bf16", 128, False, 1.0),
    "prompt": ([700, 333], [700, 300], 2, 3, 64, 128, "bf16", 64, False, 1.0),
    "far_position": ([1000003], [2], 1, 1, 32, 4096, "f32", 32, False, 1.0),
    "before_position_0": ([2, 0], [4, 2], 2, 1, 64, 16, "bf16", 64, False, 1.0),
    "many_sequences": ([5 + i % 9 for i in range(1100)], [i % 3 for i in range(1100)], 1, 1, 32, 16, "bf16", 32, False, 1.0),
}


def rotate(x, pos, freq, interleaved, scale):
    """The rotated f64 rows and the sum |x1| + |x2| each element's error goes by (0: copied)."""
    x = x.double()
    y, size, n = x.clone(), torch.zeros_like(x), freq.shape[0]
    if n:
        a = pos * freq.double()
        c, s = torch.cos(a) * scale, torch.sin(a) * scale
        one = slice(0, 2 * n, 2) if interleaved else slice(0, n)
        two = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
        x1, x2 = x[..., one], x[..., two]
        y[..., one], y[..., two] = x1 * c - x2 * s, x2 * c + x1 * s
        size[..., one] = size[..., two] = (x1.abs() + x2.abs()) * abs(scale)
    return y, size


def check_rotated(got, want, size, dtype):
    err = (got.double() - want).abs()
    off = 2.0 ** -21 * size
    lim = torch.where(size > 0, off + half_step(dtype) * (want.abs() + off) + (2.0 ** -25 if dtype is torch.float16 else 0), 0.0)
    assert bool((err <= lim).all()), f"off by {float((err - lim).max()):.3g} more than allowed"


def check_append(case, cache, q_out, freq, interleaved, scale, q_before=None):
    dk, dv = cache.k_pages.cpu(), cache.v_pages.cpu()
    kept = torch.ones(case.pages, case.page, dtype=torch.bool)
    for r, b, pos in case.rows():
        if q_out is not None:
            check_rotated(q_out[r].cpu(), *rotate(case.q[r], pos, freq, interleaved, scale), case.dtype)
        p = case.page_at(b, pos)
        if p is None:
            continue
        kept[p, pos % case.page] = False
        check_rotated(dk[p, :, pos % case.page], *rotate(case.kn[r], pos, freq, interleaved, scale), case.dtype)
        assert torch.equal(dv[p, :, pos % case.page], case.vn[r])
    kept = kept[:, None, :, None].expand_as(dk)
    assert torch.equal(dk[kept], case.k[kept]) and torch.equal(dv[kept], case.v[kept]), "other rows of the pages changed"
    if q_out is not None and q_before is not None:
        assert torch.equal(q_out[case.starts[-1]:].cpu(), q_before[case.starts[-1]:].cpu()), "rows behind the last changed"


@pytest.mark.parametrize("name", list(APPEND))
def test_append_matches_plain_form(paged, name):
    lens, counts, nkv, group, hd, page, dtype, rotary, interleaved, scale = APPEND[name]
    case = Case(lens, counts, nkv, max(1, group), hd, page, dtype, seed=21, behind=3)
    cache = case.cache(paged)
    freq = paged.rope_inv_freq(rotary, 10000.0)
    rope = paged.Rope(freq.cuda(), interleaved, scale) if rotary else None
    q = case.q.cuda() if group else None
    out = torch.full_like(q, 9.0) if group else None
    got = cache.append(case.kn.cuda(), case.vn.cuda(), q=q, q_out=out, starts=case.dstarts, rope=rope)
    assert got is out
    check_append(case, cache, out, freq, interleaved, scale, torch.full_like(case.q, 9.0))


def test_append_in_place_strided_and_unaligned(paged):
    for shift in (0, 1):
        case = Case([60, 5], [3, 2], 2, 2, 64, 16, "bf16", seed=22)
        cache = case.cache(paged)
        fused = torch.zeros((5, 8 * 64 + 16), dtype=torch.bfloat16, device="cuda")
        cut = fused[:, shift:shift + 512].unflatten(1, (8, 64))
        cut[:, :4], cut[:, 4:6], cut[:, 6:] = case.q.cuda(), case.kn.cuda(), case.vn.cuda()
        freq = paged.rope_inv_freq(64)
        got = cache.append(cut[:, 4:6], cut[:, 6:], q=cut[:, :4], starts=case.dstarts, rope=paged.Rope(freq.cuda()))
        assert got.data_ptr() == cut.data_ptr()
        check_append(case, cache, got, freq, False, 1.0)
        assert torch.equal(cut[:, 4:6].cpu(), case.kn)


def test_append_bad_pages_are_left_out(paged):
    case = Case([60, 33, 40], [3, 2, 4], 2, 2, 64, 16, "bf16", seed=23)
    case.table[0, 3] = case.pages
    case.table[1, 2] = -1
    case.table[2, 2] = -2 ** 31
    cache = case.cache(paged)
    freq = paged.rope_inv_freq(64)
    q = torch.empty_like(case.q, device="cuda")
    cache.append(case.kn.cuda(), case.vn.cuda(), q=case.q.cuda(), q_out=q, starts=case.dstarts, rope=paged.Rope(freq.cuda()))
    check_append(case, cache, q, freq, False, 1.0)


def test_append_length_past_the_table(paged):
    case = Case([64, 20], [3, 1], 2, 1, 64, 16, "bf16", seed=24)
    case.lens = [65, 20]
    cache = case.cache(paged)
    cache.append(case.kn.cuda(), case.vn.cuda(), starts=case.dstarts)
    check_append(case, cache, None, torch.zeros(0), False, 1.0)


def test_rope_matches_the_models_rotation(paged):
    """The half layout is the rotation the decoder graphs print (attention.clj:63-133)."""
    import numpy as np
    from cljxla_b200.host import nn, stablehlo as shlo, tensor as t
    from oracle import interp
    hd, heads, pos = 64, 3, 37
    for rotary in (64, 32):
        def f(x, p):
            return nn.apply_rope(x, None, p, hd, 10000.0, rotary)
        g = t.trace_graph("rope", [("x", ("tensor", (1, heads, 1, hd), "f32")), ("p", ("tensor", (1, 1), "i32"))], f)
        x = np.random.default_rng(0).standard_normal((1, heads, 1, hd)).astype(np.float32)
        want = interp.run_mlir(shlo.graph_to_mlir_text(g), [x, np.array([[pos]], np.int32)])[0]
        case = Case([pos + 1], [1], heads, 1, hd, 16, "f32")
        case.kn = torch.from_numpy(x[0, :, 0])[None]
        cache = case.cache(paged)
        cache.append(case.kn.cuda(), case.vn.cuda(), rope=paged.Rope(paged.rope_inv_freq(rotary, device="cuda")))
        got = case.dk[case.page_at(0, pos), :, pos % 16].cpu().numpy()
        # the graph's angle is an f32 product of a rounded frequency: 37 * 2^-23 rad
        assert np.abs(got - want[0, :, 0]).max() <= 37 * 2.0 ** -22 * np.abs(x).max() * 2


# ------------------------------------------------------------------- verify
def verify_oracle(target, draft, tokens, starts, uniform, race, greedy, temp, dtemp, most):
    """Plain f64 form; asserts that no choice is nearer to its border than 1e-5."""
    seqs = len(starts) - 1
    out = torch.full((seqs, most), -1, dtype=torch.int32)
    logs = torch.zeros((seqs, most), dtype=torch.float64)
    taken = []
    for b in range(seqs):
        first, count = starts[b], min(starts[b + 1] - starts[b], most)
        n = 0
        while n < count:
            row = target[first + n].double()
            top = float(row.max())
            if top == -INF:
                break
            log = torch.log_softmax(row / temp, 0)
            p = log.exp()
            best = int(torch.nonzero(row == row.max())[0])
            if n < count - 1:
                x = int(tokens[first + n + 1])
                if greedy:
                    good = x == best
                elif not 0 <= x < row.shape[0]:
                    good = False
                else:
                    q = 1.0 if draft is None else float(torch.softmax(draft[first + n].double() / dtemp, 0)[x])
                    lhs, rhs = float(uniform[first + n]) * q, float(p[x])
                    assert abs(lhs - rhs) > 1e-5 * max(lhs, rhs) or lhs == rhs == 0
                    good = lhs < rhs
                if good:
                    out[b, n], logs[b, n] = x, log[x]
                    n += 1
                    continue
            if greedy:
                token = best
            else:
                w = p
                if n < count - 1:
                    if draft is None:
                        w = p.clone()
                        if 0 <= x < row.shape[0]:
                            w[x] = 0
                    else:
                        w = (p - torch.softmax(draft[first + n].double() / dtemp, 0)).clamp(min=0)
                    if not (w > 0).any():
                        w = p
                key = w / race[b].double()
                two = torch.topk(key, min(2, key.shape[0])).values
                assert len(two) < 2 or two[0] > two[1] * (1 + 1e-5)
                token = int(key.argmax())
            out[b, n], logs[b, n] = token, log[token]
            break
        taken.append(n)
    return out, torch.tensor(taken, dtype=torch.int32), logs


def verify_case(vocab, counts, dtype, drafts, greedy, seed, gain=2.0):
    g = torch.Generator().manual_seed(seed)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    rows = starts[-1] + 2
    target = (torch.randn((rows, vocab), generator=g) * gain).to(TYPES[dtype])
    draft = (target.float() + torch.randn((rows, vocab), generator=g) * 0.7).to(TYPES[dtype]) if drafts else None
    tokens = torch.randint(vocab, (rows,), generator=g, dtype=torch.int32)
    noise = -torch.log(-torch.log(torch.rand((rows, vocab), generator=g).clamp(1e-9, 1 - 1e-7)))
    tokens[1:] = ((draft if drafts else target).float() + (0 if greedy else noise)).argmax(1)[:-1].int()
    flip = torch.rand((rows,), generator=g) < 0.2
    tokens[flip] = torch.randint(vocab, (int(flip.sum()),), generator=g, dtype=torch.int32)
    uniform = torch.rand((rows,), generator=g)
    race = torch.empty((len(counts), vocab)).exponential_(generator=g).clamp_(min=1e-30)
    return dict(target=target, draft=draft, tokens=tokens, starts=starts, uniform=uniform, race=race, greedy=greedy)


def verify_run(paged, c, temp=1.0, dtemp=None, most=None, use_starts=True, new_in_place=False):
    seqs = len(c["starts"]) - 1
    most = most or max(1, max(b - a for a, b in zip(c["starts"], c["starts"][1:])))
    cuda = lambda x: None if x is None else x.cuda()
    lens = torch.arange(100, 100 + seqs, dtype=torch.int32, device="cuda")
    old = lens.cpu().clone()
    new = lens if new_in_place else torch.full_like(lens, -9)
    out = torch.full((seqs, most), -77, dtype=torch.int32, device="cuda")
    acc = torch.full((seqs,), -77, dtype=torch.int32, device="cuda")
    logs = torch.full((seqs, most), 77.0, device="cuda")
    starts = torch.tensor(c["starts"], dtype=torch.int32).cuda() if use_starts else None
    paged.verify_draft(cuda(c["target"]), cuda(c["tokens"]), starts, out_tokens=out, accepted=acc, logprobs=logs,
                       draft_logits=cuda(c["draft"]), uniform=None if c["greedy"] else cuda(c["uniform"]),
                       race=None if c["greedy"] else cuda(c["race"]), temperature=temp, draft_temperature=dtemp,
                       greedy=c["greedy"], seq_lens=lens, new_lens=new)
    want, taken, wlogs = verify_oracle(c["target"], c["draft"], c["tokens"], c["starts"], c["uniform"], c["race"],
                                       c["greedy"], temp, temp if dtemp is None else dtemp, most)
    assert torch.equal(acc.cpu(), taken), (acc.cpu(), taken)
    assert torch.equal(out.cpu(), want)
    assert bool(((logs.cpu().double() - wlogs).abs() <= 2.0 ** -18 + 2.0 ** -22 * wlogs.abs()).all())
    counts = torch.tensor([min(b - a, most) for a, b in zip(c["starts"], c["starts"][1:])])
    assert torch.equal(new.cpu().long(), old - (counts - 1 - taken).clamp(min=0))
    return out, acc


VERIFY = {
    # name: (vocab, counts, dtype, drafts, greedy, temperature, draft temperature)
    "one_f32": (50257, [5], "f32", True, False, 1.0, None),
    "batch_bf16": (4001, [5, 1, 3, 4, 2, 5, 5], "bf16", True, False, 0.8, 1.1),
    "batch_f16": (1000, [5, 1, 3, 9, 2], "f16", True, False, 1.5, None),
    "no_distribution": (997, [4, 4, 1, 6, 2, 5], "f32", False, False, 0.7, None),
    "greedy": (4099, [4, 4, 1, 6, 2, 5], "bf16", False, True, 1.0, None),
    "greedy_f32": (513, [3, 8, 1], "f32", False, True, 2.0, None),
    "no_rows": (300, [0, 3, 0, 0, 2, 0], "bf16", True, False, 1.0, None),
    "only_samples": (2048, [1, 1, 1, 1], "f16", False, False, 1.0, None),
    "tiny_vocab": (2, [3, 3, 3, 3, 3], "f32", True, False, 1.0, None),
    "vocab_1": (1, [3, 1], "f32", True, False, 1.0, None),
    "longest_draft": (64, [128, 100, 33], "f32", True, False, 1.0, None),
    "large_vocab": (262144, [3, 2], "bf16", True, False, 1.0, None),
    "hot": (5000, [6, 6, 6], "f32", True, False, 0.05, 0.05),
    "cold": (5000, [6, 6, 6], "bf16", True, False, 40.0, 20.0),
}


@pytest.mark.parametrize("name", list(VERIFY))
def test_verify_matches_plain_form(paged, name):
    vocab, counts, dtype, drafts, greedy, temp, dtemp = VERIFY[name]
    c = verify_case(vocab, counts, dtype, drafts, greedy, seed=31)
    verify_run(paged, c, temp, dtemp)
    verify_run(paged, c, temp, dtemp, new_in_place=True)


def test_verify_without_starts(paged):
    c = verify_case(700, [3, 3, 3], "bf16", True, False, seed=33)
    for n in ("target", "draft", "tokens", "uniform"):
        c[n] = c[n][:9].contiguous()
    verify_run(paged, c, use_starts=False, most=5)


def test_verify_rows_past_max_tokens_count_as_rejected(paged):
    c = verify_case(700, [5, 2, 4], "f32", False, True, seed=41)
    cuda = {n: c[n].cuda() for n in ("target", "tokens")}
    out, acc = torch.zeros((3, 3), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    lens = torch.tensor([50, 60, 70], dtype=torch.int32, device="cuda")
    paged.verify_draft(cuda["target"], cuda["tokens"], torch.tensor(c["starts"], dtype=torch.int32).cuda(), out_tokens=out,
                       accepted=acc, greedy=True, seq_lens=lens, new_lens=lens)
    want, taken, _ = verify_oracle(c["target"], None, c["tokens"], c["starts"], None, None, True, 1.0, 1.0, 3)
    assert torch.equal(out.cpu(), want) and torch.equal(acc.cpu(), taken)
    assert lens.tolist() == [50 - (4 - int(taken[0])), 60 - (1 - int(taken[1])), 70 - (3 - int(taken[2]))]


def test_calls_without_rows(paged):
    """No rows at all: attention and append leave everything, verification says so."""
    case = Case([5, 40], [0, 0], 2, 2, 64, 16, "bf16", seed=4)
    cache = case.cache(paged)
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    none = z(0, 4, 64, dtype=torch.bfloat16)
    cache.append(z(0, 2, 64, dtype=torch.bfloat16), z(0, 2, 64, dtype=torch.bfloat16), q=none)
    assert cache.attend(none).shape == (0, 4, 64)
    assert torch.equal(cache.k_pages.cpu(), case.k)
    for greedy in (False, True):
        out, acc, logs = z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32) + 7, z(2, 3) + 7
        lens = torch.tensor([9, 4], dtype=torch.int32, device="cuda")
        paged.verify_draft(z(0, 50), z(0, dtype=torch.int32), out_tokens=out, accepted=acc, logprobs=logs, uniform=z(0),
                           race=z(2, 50) + 1, greedy=greedy, seq_lens=lens, new_lens=lens)
        assert out.tolist() == [[-1] * 3] * 2 and acc.tolist() == [0, 0] and lens.tolist() == [9, 4] and not logs.any()


def test_python_refusals(paged):
    case = Case([20, 40], [2, 1], 2, 2, 64, 16, "bf16", seed=4)
    cache = case.cache(paged)
    q, k, v = case.q.cuda(), case.kn.cuda(), case.vn.cuda()
    z = lambda *s, **kw: torch.zeros(s, device="cuda", **kw)
    with pytest.raises(ValueError, match="q:"):
        cache.attend(q.float())
    with pytest.raises(ValueError, match="q:"):
        cache.attend(case.q)
    with pytest.raises(ValueError, match="contiguous"):
        cache.attend(q.transpose(1, 2).contiguous().transpose(1, 2), starts=case.dstarts)
    with pytest.raises(ValueError, match="out"):
        cache.attend(q, out=z(3, 4, 64, dtype=torch.float16), starts=case.dstarts)
    with pytest.raises(ValueError, match="starts"):
        cache.attend(q, starts=case.dstarts.long())
    with pytest.raises(ValueError, match="starts"):
        cache.attend(q, starts=case.dstarts[:2])
    with pytest.raises(ValueError, match="v:"):  # the rows are counted by k
        cache.append(k[:2], v, starts=case.dstarts)
    with pytest.raises(ValueError, match="q_out"):
        cache.append(k, v, q_out=q, starts=case.dstarts)
    with pytest.raises(ValueError, match="page_table"):
        paged.PagedKV(case.dk, case.dv, case.dtable.long(), case.dlens)
    with pytest.raises(ValueError, match="seq_lens"):
        paged.PagedKV(case.dk, case.dv, case.dtable, case.dlens[:1])
    from cljxla_b200.host.pjrt import PJRTError
    with pytest.raises(PJRTError, match="multiple of num_seqs"):
        cache.attend(q)
    with pytest.raises(PJRTError, match="multiple of kv_heads"):
        cache.attend(z(3, 3, 64, dtype=torch.bfloat16), starts=case.dstarts)
    with pytest.raises(PJRTError, match="head_dim"):
        paged.PagedKV(z(2, 1, 16, 96), z(2, 1, 16, 96), z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32)).attend(z(1, 1, 96))
    with pytest.raises(PJRTError, match="16-byte"):
        cache.attend(z(3, 4, 72, dtype=torch.bfloat16)[:, :, 4:68], starts=case.dstarts)
    with pytest.raises(ValueError, match="uniform and race"):
        paged.verify_draft(z(2, 9), z(2, dtype=torch.int32), out_tokens=z(1, 2, dtype=torch.int32), accepted=z(1, dtype=torch.int32))
    with pytest.raises(PJRTError, match="max_tokens"):
        paged.verify_draft(z(2, 9), z(2, dtype=torch.int32), out_tokens=z(1, 1, dtype=torch.int32),
                           accepted=z(1, dtype=torch.int32), greedy=True)


def test_verify_captured_follows_its_inputs(paged):
    c = verify_case(5000, [4, 1, 3], "bf16", True, False, seed=42)
    d = {n: c[n].cuda() for n in ("target", "draft", "tokens", "uniform", "race")}
    starts = torch.tensor(c["starts"], dtype=torch.int32).cuda()
    out, acc = torch.zeros((3, 4), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    run = lambda: paged.verify_draft(d["target"], d["tokens"], starts, out_tokens=out, accepted=acc, draft_logits=d["draft"],
                                     uniform=d["uniform"], race=d["race"])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (43, 44):
        c = verify_case(5000, [2, 3, 3] if seed == 43 else [4, 4, 0], "bf16", True, False, seed=seed)
        for n in d:
            k = min(d[n].shape[0], c[n].shape[0])
            d[n][:k].copy_(c[n][:k])
        starts.copy_(torch.tensor(c["starts"], dtype=torch.int32))
        graph.replay()
        want, taken, _ = verify_oracle(c["target"], c["draft"], c["tokens"], c["starts"], c["uniform"], c["race"], False, 1.0, 1.0, 4)
        assert torch.equal(out.cpu(), want) and torch.equal(acc.cpu(), taken)


def test_first_calls_may_be_captured():
    """A process whose first calls are made under capture (nothing is loaded or set up before)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys
sys.path.insert(0, %r)
import __graft_entry__ as g
g._pkg()
import torch
from cljxla_b200.host import paged
z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
i32 = torch.int32
pages = z(9, 2, 16, 64, dtype=torch.bfloat16)
cache = paged.PagedKV(pages, z(9, 2, 16, 64, dtype=torch.bfloat16) + 2, torch.arange(8, dtype=i32, device="cuda").view(1, 8), z(1, dtype=i32) + 100)
q, k = z(2, 4, 64, dtype=torch.bfloat16), z(2, 2, 64, dtype=torch.bfloat16) + 2
logits, toks, out, acc = z(2, 5000), z(2, dtype=i32), z(1, 2, dtype=i32), z(1, dtype=i32)
uniform, race = z(2) + 0.5, z(1, 5000) + 1
rope = paged.Rope(paged.rope_inv_freq(64, device="cuda"))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    cache.append(k, k, q=q, rope=rope)
    o = cache.attend(q)
    paged.verify_draft(logits, toks, out_tokens=out, accepted=acc, uniform=uniform, race=race)
graph.replay()
torch.cuda.synchronize()
assert bool((o == 2).all()), o
assert out.tolist()[0][0] in (0, 1), out
print("captured")
""" % root
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_verify_identical_draft_is_accepted_whole(paged):
    c = verify_case(999, [5, 4], "f32", True, False, seed=34)
    c["draft"] = c["target"].clone()
    c["uniform"] = c["uniform"] * 0.99
    _, acc = verify_run(paged, c)
    assert acc.tolist() == [4, 3]


def test_verify_masked_logits(paged):
    """-inf logits (filtered vocabularies), the type's lowest value, and a token that the target rules out."""
    c = verify_case(1003, [4, 4, 4, 2], "bf16", True, False, seed=35)
    c["target"][:, 100:900] = -INF
    c["draft"][:, 400:] = -INF
    c["target"][2, 50:] = torch.finfo(torch.bfloat16).min
    c["tokens"][9] = 500
    verify_run(paged, c)
    c["target"][0, :] = -INF
    c["target"][0, 77] = -3.0  # one token left
    verify_run(paged, c)
    g = dict(c, greedy=True, draft=None)
    verify_run(paged, g)


def test_verify_row_without_a_finite_logit(paged):
    for greedy in (False, True):
        c = verify_case(500, [3, 1, 2], "f32", not greedy, greedy, seed=36)
        c["target"][0] = -INF
        c["target"][3] = -INF
        out, acc = verify_run(paged, c)
        assert out[0].tolist() == [-1] * 3 and out[1].tolist() == [-1] * 3 and acc.tolist()[:2] == [0, 0]
        c["target"][0] = math.nan
        out = torch.zeros((3, 3), dtype=torch.int32, device="cuda")
        acc = torch.zeros(3, dtype=torch.int32, device="cuda")
        paged.verify_draft(c["target"].cuda(), c["tokens"].cuda(), torch.tensor(c["starts"], dtype=torch.int32).cuda(),
                           out_tokens=out, accepted=acc, uniform=c["uniform"].cuda(), race=c["race"].cuda(), greedy=greedy)
        assert out[0].tolist() == [-1] * 3 and int(acc[0]) == 0


def test_verify_tokens_outside_the_vocabulary(paged):
    for greedy in (False, True):
        c = verify_case(500, [3, 3, 3], "f32", False, greedy, seed=37)
        c["tokens"][1], c["tokens"][4], c["tokens"][7] = -1, 500, 2 ** 31 - 1
        _, acc = verify_run(paged, c)
        assert acc.tolist() == [0, 0, 0]


def test_verify_ties_go_to_the_lowest_index(paged):
    c = verify_case(9001, [2, 1, 1], "bf16", False, True, seed=38)
    c["target"][0, [7000, 40, 8999]] = 30.0
    c["target"][2, :] = 1.0
    c["target"][3, [9000, 8192]] = 25.0
    c["tokens"][1] = 40
    out, acc = verify_run(paged, c)
    assert out.tolist()[0][0] == 40 and out.tolist()[1] == [0, -1] and out.tolist()[2] == [8192, -1]
    # equal keys of the race
    c = verify_case(4000, [1, 1], "f32", False, False, seed=39)
    c["target"][:] = 0.0
    c["race"][:] = 1.0
    o = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    acc = torch.zeros(2, dtype=torch.int32, device="cuda")
    paged.verify_draft(c["target"].cuda(), c["tokens"].cuda(), torch.tensor(c["starts"], dtype=torch.int32).cuda(),
                       out_tokens=o, accepted=acc, uniform=c["uniform"].cuda(), race=c["race"].cuda())
    assert o.tolist() == [[0], [0]]


def test_verify_strided_logits(paged):
    c = verify_case(1001, [3, 2], "bf16", True, False, seed=40)
    wide = torch.full((7, 1013), 99.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 5:1006] = c["target"].cuda()
    out, out2 = (torch.zeros((2, 3), dtype=torch.int32, device="cuda") for _ in range(2))
    acc = torch.zeros(2, dtype=torch.int32, device="cuda")
    starts = torch.tensor(c["starts"], dtype=torch.int32).cuda()
    kw = dict(accepted=acc, draft_logits=c["draft"].cuda(), uniform=c["uniform"].cuda(), race=c["race"].cuda())
    paged.verify_draft(wide[:, 5:1006], c["tokens"].cuda(), starts, out_tokens=out, **kw)
    paged.verify_draft(c["target"].cuda(), c["tokens"].cuda(), starts, out_tokens=out2, **kw)
    assert torch.equal(out, out2)


def test_verify_draws_follow_the_target(paged):
    """Whatever the draft proposes, the first token's distribution is the target's."""
    vocab, seqs = 6, 20000
    g = torch.Generator(device="cuda").manual_seed(5)
    t = torch.tensor([0.1, 1.0, -1.0, 0.5, 0.0, -2.0], device="cuda")
    d = torch.tensor([1.5, -1.0, 0.3, 0.0, 0.2, 0.1], device="cuda")
    target, draft = t.repeat(2 * seqs, 1), d.repeat(2 * seqs, 1)
    tokens = torch.multinomial(torch.softmax(d, 0), 2 * seqs, replacement=True, generator=g).int()
    uniform = torch.rand(2 * seqs, device="cuda", generator=g)
    race = torch.empty((seqs, vocab), device="cuda").exponential_(generator=g)
    out = torch.zeros((seqs, 2), dtype=torch.int32, device="cuda")
    acc = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    paged.verify_draft(target, tokens, out_tokens=out, accepted=acc, draft_logits=draft, uniform=uniform, race=race)
    share = torch.bincount(out[:, 0].long(), minlength=vocab).double() / seqs
    p = torch.softmax(t.double(), 0)
    assert bool(((share - p).abs() < 5 * (p * (1 - p) / seqs).sqrt()).all())  # five standard deviations


# ------------------------------------------------- streams, graphs, together
def test_other_stream_and_two_at_once(paged):
    cases = [Case([3000, 500], [1, 2], 2, 4, 128, 16, "bf16", seed=50 + i) for i in range(2)]
    caches = [c.cache(paged) for c in cases]
    wants = [c.attend(128 ** -0.5, 0.0, -1) for c in cases]
    qs, starts = [c.q.cuda() for c in cases], [c.dstarts for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(caches[i].attend(qs[i], starts=starts[i], max_tokens=2))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            check_rows(o, *wants[i])


def test_captured_step_follows_lengths_and_two_graphs_overlap(paged):
    """One decode step captured, replayed with other lengths, starts and pages; two graphs at once."""
    pairs = []
    for seed in (60, 61):
        a = Case([700, 120, 33], [2, 1, 3], 2, 2, 128, 16, "bf16", seed=seed, width=80, behind=2)
        cache = a.cache(paged)
        q, kn, vn = a.q.cuda(), a.kn.cuda(), a.vn.cuda()
        rope = paged.Rope(paged.rope_inv_freq(128, device="cuda"))
        qr, out = torch.zeros_like(q), torch.zeros(q.shape, device="cuda")

        def step():
            cache.append(kn, vn, q=q, q_out=qr, starts=a.dstarts, rope=rope)
            cache.attend(qr, out=out, starts=a.dstarts, max_tokens=3)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        pairs.append((a, cache, graph, qr, out, (q, kn, vn, rope, step)))
    for lens, counts in (([700, 120, 33], [2, 1, 3]), ([701, 1, 34], [1, 1, 1]), ([64, 130, 35], [3, 3, 0])):
        for a, cache, graph, qr, out, _ in pairs:
            a.lens, a.counts = lens, counts
            a.starts = [0, counts[0], counts[0] + counts[1], sum(counts)]
            order = torch.randperm(a.pages)
            at = 0
            for b, n in enumerate(lens):  # pages of the longest case are enough for all
                m = min(-(-n // 16), a.pages - at)
                a.table[b] = -1
                a.table[b, :m] = order[at:at + m].int()
                at += m
            cache.page_table.copy_(a.table)
            cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            a.dstarts.copy_(torch.tensor(a.starts, dtype=torch.int32))
            a.dk.copy_(a.k)
            a.dv.copy_(a.v)
            out.fill_(7.0)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in pairs]
        for _ in range(3):
            for (_, _, graph, *_), s in zip(pairs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for a, cache, graph, qr, out, _ in pairs:
            keep = a.k, a.v, a.q
            a.k, a.v, a.q = a.dk.cpu(), a.dv.cpu(), qr.cpu()
            want, tol = a.attend(128 ** -0.5, 0.0, -1)
            a.k, a.v, a.q = keep
            check_rows(out, want, tol, torch.full_like(out, 7.0))


def test_serving_loop_against_a_plain_decoder(paged):
    """append, attend and verify as a serving loop runs them, on a client's stream, against the same loop in 64 bits:
    one attention layer over a tied embedding, drafts of mixed quality, greedy; every sequence must read what plain
    greedy decoding reads."""
    from cljxla_b200 import LIB_PATH
    from cljxla_b200.host import core
    ctx = core.init_backend(LIB_PATH)
    stream = torch.cuda.ExternalStream(core.client_stream(ctx))
    V, H, KV, D, page, steps, most = 211, 4, 2, 64, 8, 12, 4
    g = torch.Generator().manual_seed(70)
    emb = torch.randn((V, H * D), generator=g)
    wq, wk, wv = (torch.randn((H * D, n * D), generator=g) * (H * D) ** -0.5 for n in (H, KV, KV))
    freq = paged.rope_inv_freq(D)
    prompts = [[3, 5, 8], [100], [7, 7, 7, 7, 7, 9, 2]]

    def logits64(seq):
        x = emb[seq].double()
        q, k, v = ((x @ w.double()).unflatten(1, (-1, D)) for w in (wq, wk, wv))
        q = torch.stack([rotate(q[i], i, freq, False, 1.0)[0] for i in range(len(seq))])
        k = torch.stack([rotate(k[i], i, freq, False, 1.0)[0] for i in range(len(seq))])
        s = torch.einsum("hgd,nhd->hgn", q[-1].view(KV, H // KV, D), k) * D ** -0.5
        o = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(-1)
        return (x[-1] + o) @ emb.double().T

    plain = []
    for p in prompts:
        seq = list(p)
        for _ in range(steps * most):
            l = logits64(seq)
            two = torch.topk(l, 2).values
            assert two[0] - two[1] > 1e-3  # no near ties, f32 decides the same
            seq.append(int(l.argmax()))
        plain.append(seq)

    with torch.cuda.stream(stream):
        cuda = lambda x: x.cuda()
        demb, dq, dk, dv = map(cuda, (emb, wq, wk, wv))
        rope = paged.Rope(freq.cuda())
        seqs = len(prompts)
        table = torch.randperm(seqs * 16, generator=g).int().view(seqs, 16).cuda()
        lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        kp, vp = (torch.full((seqs * 16, KV, page, D), math.nan, device="cuda") for _ in range(2))
        cache = paged.PagedKV(kp, vp, table, lens)
        read = [list(p) for p in prompts]
        feed = [list(p) for p in prompts]  # the prompt, then the newest token with drafts behind it
        drafted = [0] * seqs
        rng = torch.Generator().manual_seed(71)
        for step in range(steps):
            counts = [len(f) for f in feed]
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c)
            ds = torch.tensor(starts, dtype=torch.int32).cuda()
            flat = torch.tensor(sum(feed, []), dtype=torch.int32).cuda()
            lens += ds[1:] - ds[:-1]
            x = demb[flat.long()]
            q, k, v = ((x @ w).unflatten(1, (-1, D)) for w in (dq, dk, dv))
            q = cache.append(k, v, q=q, starts=ds, rope=rope)
            o = cache.attend(q, starts=ds, max_tokens=max(counts))
            logits = (x + o.flatten(1)) @ demb.T
            # verify the newest token's row and the drafts behind it: a prompt's earlier rows are not drafts
            rows = [starts[b + 1] - 1 - drafted[b] for b in range(seqs)]
            sel = sum((list(range(r, starts[b + 1])) for b, r in enumerate(rows)), [])
            vs = [0]
            for b in range(seqs):
                vs.append(vs[-1] + drafted[b] + 1)
            sel = torch.tensor(sel).cuda()
            out = torch.zeros((seqs, most), dtype=torch.int32, device="cuda")
            acc = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            paged.verify_draft(logits[sel], flat[sel], torch.tensor(vs, dtype=torch.int32).cuda(), out_tokens=out,
                               accepted=acc, greedy=True, seq_lens=lens, new_lens=lens)
            got = out.cpu()
            for b in range(seqs):
                new = [t for t in got[b].tolist() if t >= 0]
                read[b] += new
                n = int(torch.randint(0, most, (), generator=rng))
                ahead = plain[b][len(read[b]):len(read[b]) + n]
                if n and step % 3 == 1:
                    ahead[-1] = (ahead[-1] + 1) % V  # a wrong guess
                feed[b], drafted[b] = [read[b][-1]] + ahead, len(ahead)
    torch.cuda.synchronize()
    for b in range(seqs):
        assert len(read[b]) >= len(prompts[b]) + steps
        assert read[b] == plain[b][:len(read[b])]
        assert int(lens[b]) == len(read[b]) - 1
