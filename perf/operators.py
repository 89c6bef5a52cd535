"""Cases and plain forms of the paged-cache serving operators.

Three operators of one decode step over a paged key-value cache:

* ``append``: new keys and values into the pages of their sequences, with the
  position rotation of keys and queries applied on the way;
* ``attend``: attention of the newest token, or of the last few (a token and
  the drafted ones behind it), over the pages of each sequence;
* ``verify``: drafted tokens accepted or replaced under the target's logits,
  from given random numbers (or greedily).

A step's tokens are packed: sequence ``b`` has rows ``starts[b]`` to
``starts[b + 1]``, and ``seq_lens[b]`` counts its positions, those rows among
them.  A page is ``[kv_heads, page_size, head_dim]``; position ``j`` of a
sequence is row ``j % page_size`` of page ``page_table[b, j // page_size]``.

``run`` computes the plain form in torch, or with ``own`` set calls the
library.  Lengths and page orders belong to a case (``lengths`` seeds them);
the values come from ``prepare``'s seed.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the KV write of one decode step at batch 1: latency is all there is
        dict(name="append 1 token", op="append", dtype="bf16", seqs=1, tokens=1, ragged=False, longest=2049, lengths=1,
             q_heads=8, kv_heads=4, head_dim=256, page=64, rotary=256, interleaved=False, factor=1.0),
        # a serving batch that verifies up to four drafted tokens a sequence, far positions, rotation scaled by 8
        dict(name="append drafts", op="append", dtype="bf16", seqs=64, tokens=5, ragged=True, longest=300, lengths=2,
             q_heads=32, kv_heads=16, head_dim=128, page=16, rotary=128, interleaved=False, factor=8.0),
        # prompts of a few thousand tokens, interleaved pairs over half of the head
        dict(name="append prompts", op="append", dtype="f16", seqs=4, tokens=2048, ragged=True, longest=2600, lengths=3,
             q_heads=16, kv_heads=8, head_dim=256, page=128, rotary=128, interleaved=True, factor=1.0),
        # one sequence of the smallest configuration in f32, no shared heads
        dict(name="attend short f32", op="attend", dtype="f32", out="f32", seqs=1, tokens=1, ragged=False, longest=257,
             lengths=4, q_heads=12, kv_heads=12, head_dim=64, page=16, window=-1, softcap=0.0),
        # batch 1 behind a 2048-token prompt, two query heads per KV head
        dict(name="attend prompt 2048", op="attend", dtype="bf16", out="f32", seqs=1, tokens=1, ragged=False,
             longest=2305, lengths=5, q_heads=8, kv_heads=4, head_dim=256, page=64, window=-1, softcap=0.0),
        # one long context
        dict(name="attend long", op="attend", dtype="bf16", out="bf16", seqs=1, tokens=1, ragged=False, longest=131071,
             lengths=6, q_heads=32, kv_heads=16, head_dim=128, page=128, window=-1, softcap=0.0),
        # a batch whose lengths differ by orders of magnitude, scores capped at 50
        dict(name="attend ragged batch", op="attend", dtype="bf16", out="bf16", seqs=32, tokens=1, ragged=True,
             longest=8447, lengths=7, q_heads=8, kv_heads=4, head_dim=256, page=16, window=-1, softcap=50.0),
        # drafted tokens in a sliding-window layer
        dict(name="attend drafts window", op="attend", dtype="f16", out="f16", seqs=16, tokens=5, ragged=True,
             longest=8192, lengths=8, q_heads=16, kv_heads=8, head_dim=256, page=32, window=1024, softcap=0.0),
        # many short chats
        dict(name="attend many short", op="attend", dtype="bf16", out="bf16", seqs=256, tokens=1, ragged=True,
             longest=601, lengths=9, q_heads=32, kv_heads=16, head_dim=128, page=16, window=-1, softcap=0.0),
        # one sequence, small vocabulary in f32
        dict(name="verify one", op="verify", dtype="f32", seqs=1, tokens=5, ragged=False, lengths=10, vocab=50257,
             drafts=True, greedy=False),
        # a batch against a large vocabulary, the draft's distribution given
        dict(name="verify batch", op="verify", dtype="bf16", seqs=32, tokens=5, ragged=True, lengths=11, vocab=262144,
             drafts=True, greedy=False),
        # greedy verification of guesses that have no distribution
        dict(name="verify greedy", op="verify", dtype="bf16", seqs=64, tokens=4, ragged=True, lengths=12, vocab=256000,
             drafts=False, greedy=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = dict(op=op, dtype=dtype, ragged=rng.random() < 0.7, lengths=rng.randrange(1 << 20))
    if op == "verify":
        case.update(vocab=_log(rng, 1001, 262144), tokens=rng.randint(1, 9), drafts=rng.random() < 0.6,
                    greedy=rng.random() < 0.3)
        room = 350_000_000 // (case["vocab"] * (case["tokens"] * SIZE[dtype] * (2 if case["drafts"] else 1) + 4))
        case.update(seqs=_log(rng, 1, max(1, min(128, room))))
        return case
    head_dim, kv_heads = rng.choice([32, 64, 128, 256]), rng.choice([1, 2, 4, 8, 12, 16])
    case.update(head_dim=head_dim, kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 3, 4, 8]),
                page=rng.choice([1, 7, 16, 16, 32, 64, 128, 256]))
    row = 2 * kv_heads * head_dim * SIZE[dtype]  # one position's keys and values
    if op == "append":
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, 0])
        case.update(rotary=rotary, interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 1.0, 4.0]))
        case.update(seqs=_log(rng, 1, 128))
        case.update(tokens=_log(rng, 1, max(1, min(2048, 30_000_000 // (row * case["seqs"])))))
        case.update(longest=case["tokens"] + _log(rng, 1, max(2, min(4096, 60_000_000 // (row * case["seqs"])))))
        return case
    case.update(out=rng.choice([dtype, "f32"]), tokens=rng.choice([1, 1, 1, 2, 4, 5, 8]), softcap=rng.choice([0.0, 0.0, 30.0]))
    case.update(seqs=_log(rng, 1, 256))
    case.update(longest=max(case["tokens"], _log(rng, 1, max(8, min(131071, 600_000_000 // (row * case["seqs"]))))))
    case.update(window=rng.choice([-1, -1, 1024, _log(rng, 1, 4096)]))
    return case


def _counts(case):
    """Tokens of this step and positions of each sequence (those tokens among them): the case's own."""
    rng = random.Random(case["lengths"])
    seqs, most = case["seqs"], case["tokens"]
    counts = [rng.randint(1, most) if case["ragged"] else most for _ in range(seqs)]
    longest = case.get("longest", most)
    if case["ragged"]:
        lens = [max(counts[b], _log(rng, 1, longest)) for b in range(seqs)]
        lens[rng.randrange(seqs)] = longest
    else:
        lens = [longest] * seqs
    return counts, lens


def _width(case):
    return -(-case["longest"] // case["page"])


def _values(gen, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    counts, lens = _counts(case)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    rows, seqs, dtype = starts[-1], case["seqs"], TYPES[case["dtype"]]
    s = dict(op=case["op"], starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), most=case["tokens"])
    if case["op"] == "verify":
        vocab = case["vocab"]
        target = _values(gen, (rows, vocab), torch.float32, 2.0)
        tokens = torch.randint(vocab, (rows,), generator=gen, device="cuda")
        if case["drafts"]:
            # a draft that knows the target roughly; its tokens are drawn from its own distribution
            draft = (target + _values(gen, (rows, vocab), torch.float32, 0.7)).to(dtype)
            race = torch.rand((rows, vocab), generator=gen, device="cuda").log_().neg_().log_()
            tokens[1:] = (draft.float() * 1.25 - race).argmax(1)[:-1]
            s["draft"] = None if case["greedy"] else draft
        else:
            # guesses: the likeliest token two times in three
            likely = target.to(dtype).float().argmax(1)
            hit = torch.rand((rows,), generator=gen, device="cuda") < 0.67
            tokens[1:] = torch.where(hit, likely, tokens)[:-1]
            s["draft"] = None
        s.update(target=target.to(dtype), tokens=tokens.int(), greedy=case["greedy"], temperature=0.8,
                 uniform=None if case["greedy"] else torch.rand((rows,), generator=gen, device="cuda"),
                 race=None if case["greedy"] else
                 torch.empty((seqs, vocab), device="cuda").exponential_(generator=gen).clamp_(min=1e-30),
                 seq_lens=torch.tensor([700 + n for n in counts], dtype=torch.int32, device="cuda"),
                 new_lens=torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                 out_tokens=torch.zeros((seqs, case["tokens"]), dtype=torch.int32, device="cuda"),
                 accepted=torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                 logprobs=torch.zeros((seqs, case["tokens"]), device="cuda"))
        return s
    heads, shared, dim, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 1
    order = list(range(pages))
    random.Random(case["lengths"] + 1).shuffle(order)
    table = torch.full((seqs, _width(case)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s.update(k_pages=_values(gen, (pages, shared, page, dim), dtype), v_pages=_values(gen, (pages, shared, page, dim), dtype),
             table=table.cuda(), seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    # queries, keys and values are slices of one projection's rows
    fused = _values(gen, (rows, heads + 2 * shared, dim), dtype, 1.5)
    s["q"] = fused[:, :heads]
    if case["op"] == "append":
        s.update(k=fused[:, heads:heads + shared], v=fused[:, heads + shared:], q_out=torch.zeros((rows, heads, dim), dtype=dtype, device="cuda"),
                 rotary=case["rotary"], interleaved=case["interleaved"])
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half)) / case["factor"]
        s["inv_freq"] = freq.float().cuda()
        return s
    s.update(out=torch.zeros((rows, heads, dim), dtype=TYPES[case["out"]], device="cuda"), scale=dim ** -0.5,
             window=case["window"], softcap=case["softcap"])
    return s


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "verify": _verify}[state["op"]](state)


# ---------------------------------------------------------------- plain forms
def _rows(s, rows):
    """The sequence of each packed row, its place among the sequence's rows, and its position."""
    r = torch.arange(rows, device="cuda")
    b = (r[:, None] >= s["starts"][None, 1:]).sum(1)
    i = r - s["starts"][b]
    return b, i, (s["seq_lens"][b] - (s["starts"][b + 1] - s["starts"][b]) + i).long()


def _turned(x, cos, sin, rotary, interleaved):
    x = x.float()
    if not rotary:
        return x
    part, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([part, rest], -1)


def _append(s):
    b, _, pos = _rows(s, s["q"].shape[0])
    # the angle of a far position needs 64 bits
    angle = pos[:, None].double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    dtype, size = s["q"].dtype, s["k_pages"].shape[2]
    page = s["table"][b, pos // size].long()
    s["k_pages"][page, :, pos % size] = _turned(s["k"], cos, sin, s["rotary"], s["interleaved"]).to(dtype)
    s["v_pages"][page, :, pos % size] = s["v"]
    s["q_out"].copy_(_turned(s["q"], cos, sin, s["rotary"], s["interleaved"]))
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    table, size = s["table"].long().clamp(min=0), s["k_pages"].shape[2]
    seqs, (rows, heads, dim) = table.shape[0], s["q"].shape
    shared, most, span = s["k_pages"].shape[1], s["most"], table.shape[1] * size
    # [seqs, shared, span, dim] of the pages in order
    k = s["k_pages"][table].float().permute(0, 2, 1, 3, 4).reshape(seqs, shared, span, dim)
    v = s["v_pages"][table].float().permute(0, 2, 1, 3, 4).reshape(seqs, shared, span, dim)
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(most, device="cuda")
    at = (s["starts"][:-1, None] + i).clamp(max=rows - 1)
    q = s["q"].float()[at].reshape(seqs, most, shared, heads // shared, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, shared, -1, dim), k.transpose(2, 3)).view(seqs, shared, -1, most, span) * s["scale"]
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    pos = (s["seq_lens"].long() - count)[:, None] + i
    j = torch.arange(span, device="cuda")
    seen = j <= pos[..., None]
    if s["window"] >= 0:
        seen &= j >= pos[..., None] - s["window"]
    seen = seen[:, None, None]
    score = torch.where(seen, score, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    live = (j < s["seq_lens"][:, None])[:, None, :, None]
    total = weight.sum(-1, keepdim=True)
    got = torch.matmul(weight.reshape(seqs, shared, -1, span), torch.where(live, v, 0.0)).view(seqs, shared, -1, most, dim)
    got = torch.where(total > 0, got / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    b, i, _ = _rows(s, rows)
    s["out"].copy_(got[b, i])
    return s["out"]


def _verify(s):
    rows, vocab = s["target"].shape
    seqs, most = s["accepted"].shape[0], s["most"]
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    seq, place, _ = _rows(s, rows)
    last = place == count[seq] - 1
    scaled = s["target"].float() / s["temperature"]
    scaled -= scaled.amax(1, keepdim=True)
    weight = scaled.exp()
    norm = weight.sum(1, keepdim=True)
    guess = torch.where(last, s["tokens"], s["tokens"].roll(-1)).long()  # the token that row r + 1 holds
    best = s["target"].argmax(1)
    if s["greedy"]:
        good = guess == best
    else:
        p = (weight.gather(1, guess[:, None]) / norm)[:, 0]
        if s["draft"] is None:
            good = s["uniform"] < p
        else:
            other = s["draft"].float() / s["temperature"]
            other -= other.amax(1, keepdim=True)
            other = other.exp()
            below = other.sum(1, keepdim=True)
            good = s["uniform"] * (other.gather(1, guess[:, None]) / below)[:, 0] < p
    i = torch.arange(most, device="cuda")
    at = (s["starts"][:-1, None] + i).clamp(max=rows - 1)
    drafted = i < count[:, None] - 1
    taken = (good[at] & drafted).long().cumprod(1).sum(1)
    stop = s["starts"][:-1] + taken  # the row that the sequence's own token comes from
    if s["greedy"]:
        token = best[stop]
    else:
        left = weight[stop] / norm[stop]
        if s["draft"] is None:
            out = (torch.arange(vocab, device="cuda") == guess[stop][:, None]) & ~last[stop][:, None]
            rest = torch.where(out, 0.0, left)
        else:
            rest = torch.where(last[stop][:, None], left, (left - other[stop] / below[stop]).clamp(min=0))
        rest = torch.where(rest.amax(1, keepdim=True) > 0, rest, left)
        token = (rest / s["race"]).argmax(1)
    said = torch.where(i < taken[:, None], guess[at], torch.where(i == taken[:, None], token[:, None], -1))
    prob = scaled[at, said.clamp(min=0)] - norm[at, 0].log()
    s["out_tokens"].copy_(said)
    s["accepted"].copy_(taken)
    s["logprobs"].copy_(torch.where(said >= 0, prob, 0.0))
    s["new_lens"].copy_(s["seq_lens"] - (count - 1 - taken))
    return {"tokens": s["out_tokens"], "accepted": s["accepted"], "logprobs": s["logprobs"], "lens": s["new_lens"]}


# ------------------------------------------------------------ the library's calls
_library = None


def _paged():
    global _library
    if _library is None:
        import __graft_entry__
        __graft_entry__._pkg()
        from cljxla_b200.host import paged
        _library = paged
    return _library


def _own(s):
    if s["op"] == "verify":
        _paged().verify_draft(s["target"], s["tokens"], s["starts"], out_tokens=s["out_tokens"], accepted=s["accepted"],
                              logprobs=s["logprobs"], draft_logits=s["draft"], uniform=s["uniform"], race=s["race"],
                              temperature=s["temperature"], greedy=s["greedy"], seq_lens=s["seq_lens"], new_lens=s["new_lens"])
        return {"tokens": s["out_tokens"], "accepted": s["accepted"], "logprobs": s["logprobs"], "lens": s["new_lens"]}
    cache = s.get("cache")
    if cache is None:  # the handle that a program keeps beside its pages
        cache = s["cache"] = _paged().PagedKV(s["k_pages"], s["v_pages"], s["table"], s["seq_lens"])
    if s["op"] == "append":
        if "rope" not in s:
            s["rope"] = _paged().Rope(s["inv_freq"], interleaved=s["interleaved"]) if s["rotary"] else None
        cache.append(s["k"], s["v"], q=s["q"], q_out=s["q_out"], starts=s["starts"], rope=s["rope"])
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    cache.attend(s["q"], out=s["out"], starts=s["starts"], max_tokens=s["most"], scale=s["scale"], softcap=s["softcap"],
                 window=s["window"])
    return s["out"]


# ------------------------------------------------------------ work and 64 bits
def work(case):
    counts, lens = _counts(case)
    rows, seqs, size = sum(counts), case["seqs"], SIZE[case["dtype"]]
    if case["op"] == "verify":
        # the target's rows, the draft's rows but each sequence's last, one race row a sequence
        read = rows * case["vocab"] * size + (0 if case["greedy"] else seqs * case["vocab"] * 4)
        read += (rows - seqs) * case["vocab"] * size if case["drafts"] and not case["greedy"] else 0
        passes = (2 * rows - seqs if case["drafts"] else rows) + seqs
        return {"bytes": read + 8 * rows + seqs * (8 * case["tokens"] + 16), "flops": 4 * passes * case["vocab"]}
    heads, shared, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
    small = 4 * (2 * seqs + 1)
    if case["op"] == "append":
        table = 4 * sum(-(-n // case["page"]) for n in counts)
        return {"bytes": 2 * rows * (heads + 2 * shared) * dim * size + small + table + 2 * case["rotary"],
                "flops": 3 * rows * (heads + shared) * case["rotary"]}
    wide = case["window"] if case["window"] >= 0 else 1 << 40
    live = sum(n - max(0, n - c - wide) for c, n in zip(counts, lens))
    pairs = sum(min(n - c + i, wide) + 1 for c, n in zip(counts, lens) for i in range(c))
    return {"bytes": 2 * live * shared * dim * size + rows * heads * dim * (size + SIZE[case["out"]]) + small + 4 * live // case["page"],
            "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    s = prepare(case, seed)
    counts, lens = _counts(case)
    at = 0
    if case["op"] == "append":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        half, kp, vp = case["rotary"] // 2, s["k_pages"].double(), s["v_pages"].double()
        pos = torch.cat([torch.arange(n - c, n) for c, n in zip(counts, lens)]).cuda()
        # a pair turned by its angle is a complex product
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None, None] * s["inv_freq"].double())

        def spin(x):
            y = x.clone()
            if half:
                one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
                z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * turn
                y[..., one], y[..., two] = z.real, z.imag
            return y

        q, k = spin(q), spin(k)
        where = torch.cat([s["table"][b, torch.arange(n - c, n).cuda() // case["page"]] for b, (c, n) in enumerate(zip(counts, lens))]).long()
        kp[where, :, pos % case["page"]] = k
        vp[where, :, pos % case["page"]] = v
        return {"q": q, "k_pages": kp, "v_pages": vp}
    if case["op"] == "attend":
        got = []
        for b, (c, n) in enumerate(zip(counts, lens)):
            low = 0 if case["window"] < 0 else max(0, n - c - case["window"])
            j = torch.arange(low, n, device="cuda")
            where = s["table"][b, j // case["page"]].long()
            k, v = (s[x][where, :, j % case["page"]].double() for x in ("k_pages", "v_pages"))
            for i in range(c):
                me = n - c + i
                first = 0 if case["window"] < 0 else max(0, me - case["window"])
                kk, vv = k[first - low:me + 1 - low], v[first - low:me + 1 - low]
                q = s["q"][at + i].double().view(case["kv_heads"], -1, case["head_dim"])
                x = torch.einsum("hgd,jhd->hgj", q, kk) * s["scale"]
                if s["softcap"]:
                    x = torch.tanh(x / s["softcap"]) * s["softcap"]
                got.append(torch.einsum("hgj,jhd->hgd", torch.softmax(x, -1), vv).reshape(case["q_heads"], case["head_dim"]))
            at += c
        return torch.stack(got)
    tokens = torch.full((case["seqs"], case["tokens"]), -1, dtype=torch.int64)
    logs, taken, left = torch.zeros((case["seqs"], case["tokens"]), dtype=torch.float64), [], []
    fed = s["tokens"].tolist()
    for b, c in enumerate(counts):
        n = 0
        while True:
            row = s["target"][at + n].double() / s["temperature"]
            log = torch.log_softmax(row, 0)
            p = log.exp()
            if n < c - 1:
                x = fed[at + n + 1]
                if s["draft"] is None:
                    q = torch.zeros_like(p)
                    q[x] = 1
                else:
                    q = torch.softmax(s["draft"][at + n].double() / s["temperature"], 0)
                if s["greedy"]:
                    good = x == int(s["target"][at + n].argmax())
                else:
                    good = float(s["uniform"][at + n]) * float(q[x]) < float(p[x])
                if good:
                    tokens[b, n], logs[b, n] = x, float(log[x])
                    n += 1
                    continue
                p2 = (p - q).clamp(min=0)
                p = p2 if float(p2.max()) > 0 else p
            x = int(s["target"][at + n].argmax()) if s["greedy"] else int((p / s["race"][b].double()).argmax())
            tokens[b, n], logs[b, n] = x, float(log[x])
            break
        taken.append(n)
        left.append(700 + c - (c - 1 - n))
        at += c
    return {"tokens": tokens, "accepted": torch.tensor(taken), "logprobs": logs, "lens": torch.tensor(left)}
