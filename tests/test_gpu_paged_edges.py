"""Paged-cache operators where values are extreme: logits far from zero, finite
masks, the ends of a type's range, dominant positions; and calls at the edge of
what the interface allows.

Forms and tolerances are those of test_gpu_paged.py; where a case adds to them,
the count stands beside it.  Probabilities are held in f32, so one below 2^-126 is
zero: the oracle here takes a residual weight max(p - q, 0) below that as nothing
(the operator then draws from p, as documented), which 64 bits would still tell
apart.
"""
import math

import pytest
import torch

from test_gpu_paged import INF, TYPES, Case, half_step, paged, verify_case  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -126


# -------------------------------------------------------------- verification
def decided(c, temp, most, got):
    """The plain form in 64 bits: tokens, accepted counts, log-probabilities.  No
    choice is nearer to its border than 1e-5, but for tokens without a probability
    in f32 (there the accepted counts `got` decide)."""
    seqs = len(c["starts"]) - 1
    out, taken = torch.full((seqs, most), -1, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32)
    logs = torch.zeros((seqs, most), dtype=torch.float64)
    for b in range(seqs):
        first, n = c["starts"][b], 0
        count = min(c["starts"][b + 1] - first, most)
        while n < count:
            row, last = c["target"][first + n].double(), n == count - 1
            log = torch.log_softmax(row / temp, 0)
            p, best = log.exp(), int(torch.nonzero(row == row.max())[0])
            x = None if last else int(c["tokens"][first + n + 1])
            logq = torch.full_like(p, -INF)
            if not last and c["draft"] is not None and not c["greedy"]:
                logq = torch.log_softmax(c["draft"][first + n].double() / temp, 0)
            elif not last:
                logq[x] = 0.0
            q = logq.exp()
            if c["greedy"]:
                good = x == best
            elif not last:  # in logarithms: a masked token's p and q are below what 64 bits hold
                left, right = math.log(float(c["uniform"][first + n])) + float(logq[x]), float(log[x])
                good = left < right
                # c, the product, log2 and the sums: at most 2^-21 of each side; a base-2
                # logarithm past f32's largest (2.35e38 of a natural one) is -inf
                beyond = max(left, right) < -2.35e38
                if (abs(left - right) <= 1e-5 + 2.0 ** -21 * (abs(left) + abs(right)) or beyond) and right > -INF:
                    assert right < math.log(LEAST)  # a token that neither side would give: f32 cannot tell, either answer is right
                    good = int(got[b]) > n
            if not last and good:
                out[b, n], logs[b, n] = x, log[x]
                n += 1
                continue
            token = best
            if not c["greedy"]:
                w = p if last else torch.where(q == 1.0, 0.0, p) if c["draft"] is None else p - q
                w = w if float(w.max()) >= LEAST else p
                key = w / c["race"][b].double()
                two = torch.topk(key, 2).values
                assert two[0] > two[1] * (1 + 1e-5)
                token = int(key.argmax())
            out[b, n], logs[b, n] = token, log[token]
            break
        taken[b] = n
    return out, taken, logs


def verify(paged, c, temp=1.0):
    """One call, compared with the plain form."""
    seqs = len(c["starts"]) - 1
    most = max(b - a for a, b in zip(c["starts"], c["starts"][1:]))
    d = {n: None if c[n] is None else c[n].cuda() for n in ("target", "draft", "tokens", "uniform", "race")}
    out, acc = (torch.full(s, -77, dtype=torch.int32, device="cuda") for s in ((seqs, most), (seqs,)))
    logs = torch.full((seqs, most), 77.0, device="cuda")
    paged.verify_draft(d["target"], d["tokens"], torch.tensor(c["starts"], dtype=torch.int32).cuda(), out_tokens=out, accepted=acc,
                       logprobs=logs, draft_logits=d["draft"], uniform=d["uniform"], race=d["race"], temperature=temp,
                       greedy=c["greedy"])
    want, taken, wlogs = decided(c, temp, most, acc.cpu())
    assert torch.equal(acc.cpu(), taken), (acc.cpu(), taken)
    assert torch.equal(out.cpu(), want), (out.cpu(), want)
    assert bool(((logs.cpu().double() - wlogs).abs() <= 2.0 ** -18 + 2.0 ** -22 * wlogs.abs()).all())
    return acc


def low_case(dtype, drafts, greedy, temp, change, seed, which=("target", "draft"), vocab=6007):
    """A case whose logits `change` has been over, with tokens that fit them: drafts drawn from the changed draft."""
    c = verify_case(vocab, [4, 1, 5, 3, 2], dtype, drafts, greedy, seed)
    for n in which:
        if c[n] is not None:
            c[n] = change(c[n].float()).to(TYPES[dtype])
    g = torch.Generator().manual_seed(seed + 1)
    noise = -torch.log(-torch.log(torch.rand(c["target"].shape, generator=g).clamp(1e-9, 1 - 1e-7)))
    base = (c["draft"] if drafts else c["target"]).double() / temp
    drawn = (base if greedy else base + noise).argmax(1)[:-1].int()
    c["tokens"][1:] = torch.where(torch.rand(drawn.shape, generator=g) < 0.15, c["tokens"][1:], drawn)
    if drafts or greedy:
        c["uniform"] *= 0.5
    else:
        c["uniform"] *= 2.0 ** -20  # a guess without a distribution is rarely taken
    return c


def masked(value, how):
    """Sets `value` in the first half (whole slices of a row), all but a few (whole vectors), or all but one."""
    def change(x):
        x = x.clone()
        if how == "half":
            x[:, :3400] = value
        elif how == "most":
            keep = torch.rand(x.shape, generator=torch.Generator().manual_seed(7)) < 0.01
            keep[:, 5000] = True
            x[~keep] = value
        else:
            x[:, :4100], x[:, 4101:] = value, value
        return x
    return change


LOW = {
    # name: (dtype, temperature, change)
    **{f"shift_{d}_{v}": (d, 0.8, lambda x, v=v: x + v) for d in TYPES for v in (-100, -1000)},
    "shift_f32_cold": ("f32", 0.01, lambda x: x * 0.01 - 3.0),
    "shift_f32_far": ("f32", 1.0, lambda x: x * 512 - 2.0 ** 20),
    "shift_f32_up": ("f32", 0.5, lambda x: x + 700.0),
    **{f"mask_{d}_{how}_{v:g}": (d, 0.8, masked(v, how)) for d, vs in (("f32", (-1e4, -1e9)), ("bf16", (-1e4, -1e9)), ("f16", (-1e4, -65504.0)))
       for v in vs for how in ("half", "most", "one")},
}


@pytest.mark.parametrize("mode", ["drafts", "guesses", "greedy"])
@pytest.mark.parametrize("name", list(LOW))
def test_verify_low_logits(paged, name, mode):
    """A softmax does not see an offset, and a finite mask is as good as -inf: rows and vectors of very low logits."""
    dtype, temp, change = LOW[name]
    c = low_case(dtype, mode == "drafts", mode == "greedy", temp, change, seed=60)
    acc = verify(paged, c, temp)
    assert int(acc.sum()) >= 2


@pytest.mark.parametrize("which", ["target", "draft"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_verify_one_side_low(paged, dtype, which):
    c = low_case(dtype, True, False, 1.0, lambda x: x - 1000, seed=61, which=(which,))
    verify(paged, c)
    c = low_case(dtype, True, False, 1.0, masked(-1e4, "half"), seed=62, which=(which,))
    verify(paged, c)


ENDS = {
    # name: (dtype, temperature, change): a maximum times log2(e) / temperature does not fit f32
    **{f"{d}_lowest_{how}_{t}": (d, t, masked(torch.finfo(TYPES[d]).min, how)) for d in ("f32", "bf16") for how in ("half", "most", "one")
       for t in (0.8, 1.0, 2.0)},
    "f32_all_lowest": ("f32", 0.8, lambda x: torch.full_like(x, torch.finfo(torch.float32).min)),
    "bf16_all_lowest": ("bf16", 0.7, lambda x: torch.full_like(x, torch.finfo(torch.bfloat16).min)),
    "f32_all_highest": ("f32", 0.8, lambda x: torch.full_like(x, torch.finfo(torch.float32).max)),
    "f32_low_two": ("f32", 0.5, lambda x: torch.where(x > 5.0, -2.5e38, -3e38)),
    "bf16_high_two": ("bf16", 0.5, lambda x: torch.where(x > 5.0, 3e38, 2.9e38)),
    "f32_high_some": ("f32", 0.8, lambda x: torch.where(x > 5.0, 3.3e38, x)),
    "f16_coldest": ("f16", 1e-35, lambda x: x * 5000),
    "f32_middle": ("f32", 40.0, lambda x: x * 1024 - 2.0 ** 30),  # products of 2^25, whole steps of 2
    "f32_border": ("f32", 1.0, lambda x: x * 3 - 11629080.0),  # products on both sides of 2^24
    "f32_border_high": ("f32", 1.0, lambda x: x * 3 + 11629080.0),
    "bf16_far_mask": ("bf16", 0.03, masked(-1e9, "most")),
    "f32_wide": ("f32", 0.9, lambda x: x * 3e37),
}


@pytest.mark.parametrize("mode", ["drafts", "guesses", "greedy"])
@pytest.mark.parametrize("name", list(ENDS))
def test_verify_logits_at_the_ends_of_the_range(paged, name, mode):
    """Every row with a finite maximum has an answer, the type's lowest and largest values included."""
    dtype, temp, change = ENDS[name]
    c = low_case(dtype, mode == "drafts", mode == "greedy", temp, change, seed=63)
    verify(paged, c, temp)


@pytest.mark.parametrize("mode", ["drafts", "guesses", "greedy"])
@pytest.mark.parametrize("name", ["shift_f32_-1000", "shift_bf16_-100", "shift_f16_-1000", "mask_bf16_half_-1e+09", "mask_f16_one_-65504",
                                  "f32_lowest_half_0.8", "bf16_lowest_most_1.0", "bf16_all_lowest", "f32_border"])
@pytest.mark.parametrize("vocab", [8192, 40000])
def test_verify_low_logits_in_aligned_rows(paged, vocab, name, mode):
    """Vocabularies of whole vectors, raced by one CTA's and by a whole cluster's vector loads."""
    dtype, temp, change = {**LOW, **ENDS}[name]
    c = low_case(dtype, mode == "drafts", mode == "greedy", temp, change, seed=66, vocab=vocab)
    verify(paged, c, temp)


@pytest.mark.parametrize("mode", ["drafts", "guesses", "greedy"])
def test_verify_a_row_with_plus_infinity_has_no_token(paged, mode):
    def change(x):
        x = x.clone()
        x[:, [17, 4000]] = INF
        return x
    c = low_case("f32", mode == "drafts", mode == "greedy", 1.0, change, seed=64, which=("target",))
    d = {n: None if c[n] is None else c[n].cuda() for n in ("target", "draft", "tokens", "uniform", "race")}
    out, acc = torch.zeros((5, 5), dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    paged.verify_draft(d["target"], d["tokens"], torch.tensor(c["starts"], dtype=torch.int32).cuda(), out_tokens=out, accepted=acc,
                       draft_logits=d["draft"], uniform=d["uniform"], race=d["race"], greedy=c["greedy"])
    assert bool((out == -1).all()) and not acc.any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("with_starts", [False, True])
def test_verify_draft_without_the_last_row(paged, dtype, with_starts):
    """A draft model gives one distribution fewer than there are rows: through the C entry, where the draft's
    last row may be missing.  Here it is memory of this test's own that holds NaN."""
    import ctypes
    vocab, rows = 6007, 4
    c = verify_case(vocab, [rows], dtype, True, False, seed=65)
    d = {n: c[n].cuda() for n in ("target", "tokens", "uniform", "race")}
    draft = torch.cat([c["draft"][:rows - 1], torch.full((1, vocab), math.nan, dtype=TYPES[dtype])]).cuda()
    out, acc = torch.zeros((1, rows), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    a = paged._VerifyArgs(ctypes.sizeof(paged._VerifyArgs), d["target"].data_ptr(), draft.data_ptr(), d["tokens"].data_ptr(),
                          starts.data_ptr() if with_starts else None, d["uniform"].data_ptr(), d["race"].data_ptr(), rows, 1, vocab,
                          rows, vocab, vocab, vocab, 1.0, 1.0, paged._TYPES[TYPES[dtype]], 0, out.data_ptr(), acc.data_ptr(), None,
                          None, None, work.data_ptr(), work.numel())
    err = ctypes.create_string_buffer(512)
    assert paged._library().verify(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream, err, 512) == 0, err.value
    want, taken, _ = decided(c, 1.0, rows, acc.cpu())
    assert torch.equal(out.cpu(), want) and torch.equal(acc.cpu(), taken)


# ----------------------------------------------------------------- attention
SINKS = {
    # name: (length, position of the dominant key, head_dim, query heads per KV head, rows)
    "one_tile": (50, 0, 64, 2, 1),
    "middle": (5000, 2400, 128, 2, 1),
    "long": (131071, 0, 64, 1, 1),
    "long_last": (40000, 39990, 256, 2, 1),
    "sixteen_rows": (3000, 1, 32, 4, 4),
    "many_rows": (3000, 1500, 64, 8, 5),
    "wide_many_rows": (2000, 700, 256, 16, 3),
}


@pytest.mark.parametrize("gap", [4.0, 11.0, 17.0, 17.4, 18.0, 22.0])
@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("name", list(SINKS))
def test_attend_one_position_outweighs_the_others(paged, name, dtype, out, gap):
    """An attention sink: one key whose score is far above all others, which are equal, and whose value is 0, so
    that the result is what the others' small weights leave.

    All scores are exact (one element of q and k each) but for their factor log2(e), 2^-23 of at most 32, so a
    weight is off by 2^-18 relatively (exp2 in it); sums over tiles and ranges add at most 64 terms in a row,
    2^-18.  bf16 weights for bf16 outputs have 16 bits, 2^-16; f16 ones have steps of 2^-39 of their tile's
    largest, so in the dominant one's tile each of the 63 others is off by up to 2^-40 e^gap of itself.
    Then the output's own half step; f16 outputs below 2^-14 have steps of 2^-24."""
    length, at, hd, group, rows = SINKS[name]
    c = Case([length], [rows], 2, group, hd, 64, dtype, seed=70)
    c.k.zero_()
    col = torch.arange(hd) % 16
    c.v[:] = (1 + col / 16.0).to(c.dtype)
    page, row = int(c.table[0, at // 64]), at % 64
    c.k[page, :, row, 3] = 2.0
    c.v[page, :, row] = 0.0
    c.q.zero_()
    c.q[:, :, 3] = gap / 2  # exact in bf16
    c.q[:, :, 3] += (torch.arange(rows)[:, None] + torch.arange(2 * group)) % 2 * 0.5
    real = 2.0 * c.q[:, :, 3].double()  # [rows, heads]
    others = torch.tensor([length - rows + i for i in range(rows)], dtype=torch.float64)[:, None]
    want = (others / (others + real.exp()))[..., None] * (1 + col / 16.0).double()
    got = torch.empty((rows, 2 * group, hd), dtype=TYPES[out], device="cuda")
    c.cache(paged).attend(c.q.cuda(), out=got, starts=c.dstarts, scale=1.0)
    rel = 2.0 ** -18 + 2.0 ** -18 + (2.0 ** -16 if dtype == "bf16" and out == "bf16" else 0)
    if dtype == "f16":
        rel = rel + (63 / others.clamp(min=63)) * (2.0 ** -40 * real.exp())
    tol = want * (rel[..., None] if torch.is_tensor(rel) else rel)
    own = half_step(TYPES[out])
    tol = tol + (want + tol) * own + (2.0 ** -25 if out == "f16" else 0)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / want).max())


@pytest.mark.parametrize("hd,group,rows", [(64, 1, 1), (128, 2, 5), (256, 4, 8)])
def test_attend_f16_weights_after_a_dominant_tile(paged, hd, group, rows):
    """Random scores, one key 20 above them whose value is 0, unseen positions that hold NaN (products made one by
    one there).  Per weight: its score's sum, (head_dim + 8) 2^-24 of sum |q k|, and 2^-17 as in the test before;
    the quotient has that twice; 64 weights of the dominant one's tile are off by 2^-40 of it."""
    c = Case([3000, 700], [rows, rows], 2, group, hd, 16, "f16", seed=71)
    scale = 0.125
    c.k *= 0.25
    c.q[:, :, 0], c.k[..., 0] = 1.0, 0.0
    sinks = (1234, 0)
    for b, at in enumerate(sinks):
        p = int(c.table[b, at // 16])
        c.k[p, :, at % 16] = 0.0
        c.k[p, :, at % 16, 0] = 20.0 / scale
        c.v[p, :, at % 16] = 0.0
    want, tol = [], []
    for b in (0, 1):
        r, n = c.starts[b], c.lens[b] - rows + 1
        j = torch.arange(n)
        k, v = (x[c.table[b, j // 16].long(), :, j % 16].double() for x in (c.k, c.v))  # [n, nkv, hd]
        q = c.q[r].double().view(2, group, hd)
        w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) * scale, -1)
        size = torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()) * scale
        size[..., sinks[b]] = 0.0
        want.append(torch.einsum("hgn,nhd->hgd", w, v).reshape(-1, hd))
        one = (hd + 8) * 2.0 ** -24 * float(size.max()) + 2.0 ** -17
        tol.append((2 * one * torch.einsum("hgn,nhd->hgd", w, v.abs()) + 64 * 2.0 ** -40 * float(v.abs().max())).reshape(-1, hd))
        for at in range(n, c.lens[b]):  # the later rows' own positions
            c.v[int(c.table[b, at // 16]), :, at % 16] = math.nan
    got = torch.zeros(c.q.shape, device="cuda")
    c.cache(paged).attend(c.q.cuda(), out=got, starts=c.dstarts, scale=scale)
    for b in (0, 1):
        r = c.starts[b]
        off = (got[r].cpu().double() - want[b]).abs()
        assert bool((off <= tol[b]).all()), float((off / tol[b]).max())
        assert bool(got[r + 1:r + rows].isnan().all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd,group,rows", [(64, 1, 1), (128, 4, 2), (32, 8, 3)])
def test_attend_huge_scores(paged, hd, group, rows, dtype):
    """Scores whose steps are wider than any weight's exponent: the positions of the largest share the result."""
    c = Case([300], [rows], 2, group, hd, 16, dtype, seed=72)
    c.q.zero_()
    c.k.zero_()
    c.q[..., 0] = 60000.0
    at = [3, 70, 250]
    for sign in (1.0, -1.0):
        for j in range(300):
            c.k[int(c.table[0, j // 16]), :, j % 16, 0] = sign * (60000.0 if (j in at) == (sign > 0) else 30000.0)
        want = torch.stack([c.v[int(c.table[0, j // 16]), :, j % 16].double() for j in at]).mean(0)  # [nkv, hd]
        got = torch.empty((rows, 2 * group, hd), device="cuda")
        c.cache(paged).attend(c.q.cuda(), out=got, starts=c.dstarts, scale=1.0)
        off = (got.cpu().double().view(rows, 2, group, hd) - want[None, :, None]).abs()
        assert bool((off <= 2.0 ** -15 * 4).all()), float(off.max())  # bf16 weights of 1, a third in f32: 2^-22 and less


# ------------------------------------------------------------------ refusals
def test_tensors_that_need_gradients_are_refused(paged):
    """The operators have no backward pass: a gradient would be lost in silence."""
    c = Case([20, 40], [2, 1], 2, 2, 64, 16, "bf16", seed=4)
    cache = c.cache(paged)
    q, k, v = c.q.cuda(), c.kn.cuda(), c.vn.cuda()
    want = lambda t: t.detach().clone().requires_grad_()
    for kw in (dict(q=want(q)), dict(q=q, out=want(q))):
        with pytest.raises(ValueError, match="gradient"):
            cache.attend(starts=c.dstarts, **kw)
    for a in ((want(k), v, q), (k, want(v), q), (k, v, want(q)), (k, v, q, want(q))):
        with pytest.raises(ValueError, match="gradient"):
            cache.append(*a, starts=c.dstarts)
    with pytest.raises(ValueError, match="gradient"):
        paged.PagedKV(want(c.dk), c.dv, c.dtable, c.dlens)
    with pytest.raises(ValueError, match="gradient"):
        paged.PagedKV(c.dk, want(c.dv), c.dtable, c.dlens)
    with pytest.raises(ValueError, match="gradient"):
        paged.Rope(torch.ones(4, device="cuda", requires_grad=True))
    z = lambda *s, **kw: torch.zeros(s, device="cuda", **kw)
    out, acc = z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32)
    f = dict(target_logits=z(2, 9), draft_logits=z(2, 9), uniform=z(2), race=z(1, 9) + 1)
    for n in f:
        with pytest.raises(ValueError, match="gradient"):
            paged.verify_draft(**{**f, n: want(f[n])}, tokens=z(2, dtype=torch.int32), out_tokens=out, accepted=acc)
    # without gradients being recorded, the same tensors serve
    with torch.no_grad():
        assert torch.equal(cache.attend(want(q), starts=c.dstarts), cache.attend(q, starts=c.dstarts))
        paged.verify_draft(**{n: want(f[n]) for n in f}, tokens=z(2, dtype=torch.int32), out_tokens=out, accepted=acc)
    assert int(out[0, 0]) == 0
