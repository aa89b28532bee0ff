"""What a decoder does around the paged 4-bit K/V cache, as cases to time and compare.

A case is a dict of plain values; its "op" names the operator:

  weights  the attention weight that every cached position got from new rows, added up: one row a sequence (decode) or many
  evict    keeps the latest, the first and the heaviest positions of each kv head, moves them together in the cache, and reads
           the kept rows back as the values they stand for
  beam     the best continuations of every sequence's beams: log-softmax over the vocabulary, top k over beams and tokens
  reorder  page tables that follow the beams' parents, with a page of its own for what a beam goes on writing; the rows
           of that page are read back
  rope     rotates rows by positions along several axes (time, height, width), or takes gradients back through that

run() computes the operators in plain torch, or, where `own` is true, through klearu_amd.  exact() gives the outputs in 64
bits from the definitions.

The cache's format: 32 neighbouring values of a head share a scale s and a minimum m, both BF16: m is the smallest
value rounded down, s is (largest - m) / 15 rounded up, a value x is held as c = rint((x - m) / s) in 0..15, and stands
for s * c + m.  The quotients are f32 ones.
"""
from __future__ import annotations

import math

import torch

own = False

HALF, INTERLEAVED = "half", "interleaved"
GROUP = 32


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of one sequence of a 7B-class model, half of the heads selected: latency.
        dict(name="weights_b1_f32", op="weights", batch=1, rows=1, ragged=False, cached=1999, heads=32, kv_heads=32,
             dim=128, page=64, selected=16, window=0, dtype="f32"),
        # A serving batch of a 1.1B-class model (32 heads over 4), contexts of every length.
        dict(name="weights_b64_ragged", op="weights", batch=64, rows=1, ragged=True, cached=4095, heads=32, kv_heads=4,
             dim=64, page=16, selected=0, window=0, dtype="bf16"),
        # A prompt: which of its own positions it looks at.
        dict(name="weights_prompt", op="weights", batch=1, rows=4096, ragged=False, cached=0, heads=32, kv_heads=8,
             dim=128, page=64, selected=0, window=0, dtype="bf16"),
        # The cache of one sequence is a page over its budget.
        dict(name="evict_b1", op="evict", batch=1, length=2111, ragged=False, keep=2048, recent=512, first=4,
             kv_heads=32, dim=128, page=64),
        # A serving batch, every length, some below the budget.
        dict(name="evict_b64_ragged", op="evict", batch=64, length=4099, ragged=True, keep=1024, recent=256, first=0,
             kv_heads=4, dim=64, page=16),
        # One long document cut to a quarter before the questions.
        dict(name="evict_b1_long", op="evict", batch=1, length=131072, ragged=False, keep=32768, recent=1000, first=16,
             kv_heads=8, dim=128, page=64),
        # A step of four beams of one sequence: latency.
        dict(name="beam_b1_f32", op="beam", batch=1, beams=4, vocab=32000, k=8, done=False, first=False, dtype="f32"),
        # A batch with a large vocabulary, some beams at their end.
        dict(name="beam_b64", op="beam", batch=64, beams=8, vocab=131071, k=16, done=True, first=False, dtype="bf16"),
        # The four beams' tables of that step, 7B-class layer.
        dict(name="reorder_b1", op="reorder", batch=1, beams=4, length=1999, ragged=False, kv_heads=32, dim=128, page=64),
        # A batch of beams, grouped heads.
        dict(name="reorder_b64", op="reorder", batch=64, beams=8, length=8190, ragged=True, kv_heads=8, dim=128, page=64),
        # A video's tokens: 64 pairs of a head's elements go by time, height and width.
        dict(name="rope_axes_8191", op="rope", tokens=8191, heads=32, dim=128, sections="16,24,24", restart=False,
             layout=HALF, max_pos=32768, dtype="bf16", back=False),
        # Gradients of an image's patches: height and width with frequencies of their own, sections that end inside a vector.
        dict(name="rope_axes_back_2049", op="rope", tokens=2049, heads=16, dim=72, sections="18,18", restart=True,
             layout=INTERLEAVED, max_pos=1024, dtype="f32", back=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["weights", "weights", "evict", "beam", "reorder", "rope"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    if op == "rope":
        axes = rng.choice([2, 3, 3, 4])
        pairs = rng.choice([axes * 4 + 1, 16, 32, 36, 64, 64])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if rng.random() < 0.5 else \
            [pairs // axes // 4 * 4 * (i + 1) for i in range(axes - 1)]
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        dim = 2 * pairs + rng.choice([0, 0, 16, 2 * pairs])
        heads = _logint(rng, 1, 64)
        tokens = _logint(rng, 1, max(2, 8191 * 32 * 128 // (heads * dim * (2 if dtype == "f32" else 1))))
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, sections=",".join(str(n) for n in sections),
                    restart=rng.random() < 0.4, layout=rng.choice([HALF, INTERLEAVED]), max_pos=_logint(rng, 64, 32768),
                    dtype=dtype, back=rng.random() < 0.4)
    if op == "beam":
        batch, vocab = _logint(rng, 1, 64), _logint(rng, 100, 131071)
        beams = rng.choice([1, 2, 3, 4, 5, 8])
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, k=min(vocab, rng.choice([beams, 2 * beams, 2 * beams + 1])),
                    done=rng.random() < 0.4, first=rng.random() < 0.2, dtype=dtype)
    if op == "reorder":
        return dict(op=op, batch=_logint(rng, 1, 64), beams=rng.choice([2, 3, 4, 5, 8]), length=_logint(rng, 1, 8190),
                    ragged=rng.random() < 0.7, kv_heads=min(kv, 8), dim=min(dim, 128), page=page)
    if op == "evict":
        batch = _logint(rng, 1, 64)
        length = _logint(rng, 20, min(131072, 131072 * 8 * 128 // (batch * kv * dim)))
        keep = max(1, int(length * rng.uniform(0.1, 0.98)))
        recent = int(keep * rng.uniform(0, 0.9))
        return dict(op=op, batch=batch, length=length, ragged=rng.random() < 0.7, keep=keep, recent=recent,
                    first=min(keep - recent, rng.choice([0, 4, 16])), kv_heads=kv, dim=dim, page=page)
    group = rng.choice([1, 1, 2, 4, 8])
    heads = kv * group if kv * group <= 64 else kv
    window = rng.choice([0, 0, _logint(rng, 16, 2048)])
    if rng.random() < 0.6:  # decode
        batch = _logint(rng, 1, 64)
        cached = _logint(rng, 1, max(2, min(131071, 64 * 4096 * 4 * 64 // (batch * kv * dim))))
        return dict(op=op, batch=batch, rows=1, ragged=rng.random() < 0.6, cached=cached, heads=heads, kv_heads=kv,
                    dim=dim, page=page, selected=rng.choice([0, 0, max(1, heads // 2)]), window=window, dtype=dtype)
    batch = rng.choice([1, 1, 2, 3, 5])
    rows = _logint(rng, 2, 2000 // batch if dtype == "bf16" else 700 // batch)
    cached = rng.choice([0, _logint(rng, 1, 4000)])
    cached = min(cached, max(0, 4096 * 4096 * 16 * 128 // (batch * rows * heads * dim) - rows))
    return dict(op=op, batch=batch, rows=rows, ragged=rng.random() < 0.7, cached=cached, heads=heads, kv_heads=kv,
                dim=dim, page=page, selected=0, window=window, dtype=dtype)


# ------------------------------------------------------------------ inputs
class State:
    pass


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _spread(n, count, salt, least=0.05):
    """`count` numbers up to n, the first of them n."""
    part = torch.rand(count, generator=torch.Generator().manual_seed(n * 7919 + count + salt)).tolist()
    return [n] + [max(1, int(n * (least + (1 - least) * p))) for p in part[1:]]


def _sizes(case):
    """Rows and lengths of each sequence, on the host."""
    b = case["batch"]
    if case["op"] in ("evict", "reorder"):
        return None, _spread(case["length"], b, 1) if case["ragged"] else [case["length"]] * b
    rows, before = [case["rows"]] * b, [case["cached"]] * b
    if case["ragged"]:
        rows = _spread(case["rows"], b, 2)
        before = [min(c, case["cached"]) for c in _spread(max(1, case["cached"]), b, 3, 0.02)][::-1]
    return rows, [r + c for r, c in zip(rows, before)]


def _keys(gen, n, heads, dim):
    """Keys or values as a layer makes them: normal, a few channels of each head far larger and off zero."""
    gain = 0.6 + 0.8 * torch.rand(heads, dim, generator=gen, device="cuda")
    big = (torch.rand(heads, dim, generator=gen, device="cuda") < 0.03).float()
    shift = torch.randn(heads, dim, generator=gen, device="cuda") * (0.1 + 3.0 * big)
    x = torch.randn(n, heads, dim, generator=gen, device="cuda")
    return (x * gain * (1 + big) + shift).to(torch.bfloat16)


def _tables(lens, page, seed, spare=0):
    """Page tables over shuffled pages, `spare` columns more than the lengths need, and the pool's pages."""
    need = [-(-n // page) + spare for n in lens]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(int(seed) + 1)).to(torch.int32)
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), sum(need) + 3


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


def _off(n):
    return _i64([0] + list(n)).cumsum(0)


def _inputs(case, seed):
    """What the seed alone gives: tensors on the GPU and sizes on the host."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = State()
    s.case = case
    if case["op"] == "rope":
        n, m, axes = case["tokens"], case["max_pos"], len(_sections(case))
        s.x = torch.randn(n, case["heads"], case["dim"], generator=gen, device="cuda").to(_dtype(case))
        # a grid walked in order: the last axis fastest, each axis from a place of its own
        side = [max(1, min(m, round(n ** (1 / axes)) + a)) for a in range(axes)]
        at, pos = torch.arange(n, device="cuda"), []
        for a in reversed(range(axes)):
            pos.append((at % side[a] if a else at) % m)
            at = at // side[a]
        first = torch.randint(0, max(1, m - max(side)), (axes, 1), generator=torch.Generator().manual_seed(int(seed)))
        s.pos = (torch.stack(pos[::-1]) + first.cuda()) % m
        return s
    if case["op"] == "beam":
        b, w, n = case["batch"], case["beams"], case["vocab"]
        x = torch.randn(b, w, n, generator=gen, device="cuda") * 2.5
        x += 6.0 * (torch.rand(b, w, n, generator=gen, device="cuda") < 20.0 / n)  # the likely ones
        s.logits = x.to(_dtype(case))
        s.scores = -20.0 * torch.rand(b, w, generator=gen, device="cuda")
        if case["first"]:
            s.scores[:, 1:] = -math.inf  # all beams are alike yet
        s.done = torch.rand(b, w, generator=gen, device="cuda") < 0.3 if case["done"] else None
        s.end = 2
        return s
    rows, lens = _sizes(case)
    s.lens_host = lens
    kv, dim, ps = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "reorder":
        w = case["beams"]
        s.len = _i64(lens)
        # a parent's pages are its own here, as after a prompt that every beam has read
        s.row_lens = [n for n in lens for _ in range(w)]
        s.parent = torch.randint(0, w, (case["batch"], w), generator=gen, device="cuda").to(torch.int32)
        s.table, s.pages = _tables(s.row_lens, ps, seed, spare=1)
        # what is read back, and what lies there: the rows in the page that is not full
        s.tail = [n % ps for n in s.row_lens]
        s.tail_start, s.tail_off = _i64([n - t for n, t in zip(s.row_lens, s.tail)]), _off(s.tail)
        n = sum(s.tail)
        s.all_k, s.all_v = _keys(gen, n, kv, dim), _keys(gen, n, kv, dim)
        return s
    s.table, s.pages = _tables(lens, ps, seed)
    s.cap = s.table.shape[1] * ps
    s.all_k = _keys(gen, sum(lens), kv, dim)
    s.len = _i64(lens)
    live = torch.arange(s.cap, device="cuda") < s.len[:, None, None]
    # weights so far: a few positions have most of them
    s.acc = torch.exp(1.5 * torch.randn(len(lens), kv, s.cap, generator=gen, device="cuda")) * live
    if case["op"] == "evict":
        s.all_v = _keys(gen, sum(lens), kv, dim)
        left = [min(n, case["keep"]) for n in lens]
        s.left_off, s.left, s.zero = _off(left), sum(left), torch.zeros_like(s.len)
        return s
    s.rows, s.total, s.off = rows, sum(rows), _off(rows)
    s.start = s.len - _i64(rows)
    heads = case["heads"]
    s.qkv = torch.empty(s.total, heads + 2 * kv, dim, dtype=_dtype(case), device="cuda")
    s.q = s.qkv[:, :heads]  # queries lie in the projection's rows
    s.q.copy_(torch.randn(s.total, heads, dim, generator=gen, device="cuda") * 1.2)
    s.scale = dim ** -0.5
    s.lse = _log_sums(s)
    if case["selected"]:  # heads that a row does not list have seen nothing
        rank = torch.rand(s.total, heads, generator=gen, device="cuda").argsort(1)
        s.lse = s.lse.masked_fill(rank >= case["selected"], -math.inf)
    s.most_rows, s.most_len = max(rows), max(lens)
    return s


def _hidden(s, b):
    """[rows, length] which positions the rows of sequence b do not see."""
    n, r, w = s.lens_host[b], s.rows[b], s.case["window"]
    ahead = torch.arange(n - r, n, device="cuda")[:, None] - torch.arange(n, device="cuda")
    return (ahead < 0) | (ahead >= w) if w else ahead < 0


def _log_sums(s):
    """log sum exp of every row's scores, as attention gives it with its result (64 bits, rounded once)."""
    out, at, row = [], 0, 0
    heads, kv = s.case["heads"], s.case["kv_heads"]
    for b, (n, r) in enumerate(zip(s.lens_host, s.rows)):
        k, hide = _exact_held(s.all_k[at:at + n].double()), _hidden(s, b)
        one = [torch.logsumexp((s.q[row:row + r, h].double() @ k[:, h * kv // heads].T * s.scale).masked_fill(hide, -math.inf), -1)
               for h in range(heads)]
        out.append(torch.stack(one, 1))
        at, row = at + n, row + r
    return torch.cat(out).float()


# ------------------------------------------------------------------ plain forms
def _bf16_down(x):
    """Largest BF16 value at or below x (f32 in and out)."""
    r = x.to(torch.bfloat16)
    down = torch.nextafter(r, torch.full_like(r, -math.inf))
    return torch.where(r.float() > x, down, r).float()


def _quantize(x):
    """x [..., dim] f32 -> (codes packed two to a byte, s, m)."""
    g = x.unflatten(-1, (-1, GROUP))
    m = _bf16_down(g.amin(-1))
    # a tensor of fifteens: torch multiplies by the reciprocal of a plain number
    s = -_bf16_down(-((g.amax(-1) - m) / torch.full_like(m, 15.0)))
    c = torch.where(s[..., None] > 0, ((g - m[..., None]) / s[..., None]).round(), torch.zeros_like(g))
    c = c.clamp(0, 15).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4, s.to(torch.bfloat16), m.to(torch.bfloat16)


def _values(c, s, m):
    x = torch.stack([c & 15, c >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (x * s[..., None].float() + m[..., None].float()).flatten(-2)


def _pool(s, case):
    """The cache, with one page more: moves that do nothing go there."""
    n = (s.pages + 1, case["page"], 2, case["kv_heads"])
    s.code = torch.zeros(*n, case["dim"] // 2, dtype=torch.uint8, device="cuda")
    s.s = torch.zeros(*n, case["dim"] // GROUP, dtype=torch.bfloat16, device="cuda")
    s.m = torch.zeros_like(s.s)


def _places(off, start, table, total, page):
    """(page, place in it) of each row."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(off, row, right=True) - 1
    pos = start[seq] + row - off[seq]
    return table[seq, pos // page].long(), pos % page


def _plain_put(s, k, v, off, start, table, page):
    pg, at = _places(off, start, table, k.shape[0], page)
    s.code[pg, at], s.s[pg, at], s.m[pg, at] = _quantize(torch.stack([k.float(), v.float()], 1))


def _plain_read(s, off, start, table, total, page):
    pg, at = _places(off, start, table, total, page)
    x = _values(s.code[pg, at], s.s[pg, at], s.m[pg, at]).to(torch.bfloat16)
    return x[:, 0], x[:, 1]


def _plain_weights(s, case):
    kv, dim, heads = case["kv_heads"], case["dim"], case["heads"]
    b, gs, n, most = len(s.rows), heads // kv, s.most_len, s.most_rows
    t = s.table.long()
    k = _values(s.code[t][:, :, :, 0], s.s[t][:, :, :, 0], s.m[t][:, :, :, 0]).flatten(1, 2)[:, :n].permute(0, 2, 3, 1)
    i = torch.arange(most, device="cuda")
    row = (s.off[:-1, None] + i).clamp(max=s.total - 1)
    q = s.q[row].float().view(b, most, kv, gs, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, gs * most, dim)
    lse = s.lse[row].view(b, most, kv, gs).permute(0, 2, 3, 1).reshape(b, kv, gs * most, 1)
    pos = (s.start[:, None] + i)[:, :, None]
    j = torch.arange(n, device="cuda")
    seen = (j <= pos) & (i < (s.off[1:] - s.off[:-1])[:, None])[:, :, None]
    if case["window"]:
        seen = seen & (j > pos - case["window"])
    seen = seen[:, None, None] & (lse.view(b, kv, gs, most, 1) > -math.inf)
    w = torch.exp(torch.matmul(q, k) * s.scale - lse).view(b, kv, gs, most, n).masked_fill(~seen, 0.0)
    s.acc[:, :, :n] += w.sum((2, 3))
    return s.acc


def _plain_evict(s, case):
    keep, ps, n = case["keep"], case["page"], s.cap
    b, kv = s.acc.shape[:2]
    j, length = torch.arange(n, device="cuda"), s.len[:, None, None]
    stays = (j < case["first"]) | (j >= length - case["recent"])
    rank = s.acc.masked_fill(stays, math.inf).masked_fill(j >= length, -math.inf)
    keep = min(keep, n)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    left = s.len.clamp(max=keep)
    to = torch.arange(keep, device="cuda").expand(b, kv, keep)
    moved = to < left[:, None, None]
    kept = torch.where(moved, best, torch.full_like(best, -1))
    acc = torch.zeros_like(s.acc)
    acc[..., :keep] = torch.where(moved, s.acc.gather(2, best), torch.zeros((), device="cuda"))
    t = s.table.long()
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(kv, device="cuda")[:, None]
    none = torch.full_like(best, s.pages)
    src, dst = (torch.where(moved, t[seq, p // ps], none) for p in (best, to))
    a, d = best % ps, to % ps
    for x in (s.code, s.s, s.m):
        x[dst, d, :, head] = x[src, a, :, head]
    k, v = _plain_read(s, s.left_off, s.zero, s.table, s.left, ps)
    short = case["keep"] - keep
    kept = torch.cat([kept, torch.full((b, kv, short), -1, device="cuda")], -1) if short else kept
    return kept.to(torch.int32), left, acc, k, v


def _plain_beam(s, case):
    w, n, k = case["beams"], case["vocab"], case["k"]
    x = s.logits.double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + (x - top).exp().sum(-1, keepdim=True).log()) + s.scores.double()[..., None]
    if s.done is not None:
        ends = torch.where(torch.arange(n, device="cuda") == s.end, s.scores.double()[..., None], -math.inf)
        x = torch.where(s.done[..., None], ends, x)
    x = x.flatten(1)
    # the k largest, of equal ones the first
    least = x.topk(k, 1).values[:, -1:]
    above = x > least
    same = x == least
    take = above | (same & (same.cumsum(1) <= k - above.sum(1, keepdim=True)))
    at = torch.arange(w * n, device="cuda").expand_as(x).masked_fill(~take, w * n).topk(k, 1, largest=False).values.sort(1).values
    y, order = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    return y.float(), (at // n).to(torch.int32), (at % n).to(torch.int32)


def _plain_reorder(s, case):
    b, w, ps = case["batch"], case["beams"], case["page"]
    p = s.parent.long()
    alike = p[:, :, None] == p[:, None, :]
    again = torch.tril(alike, -1).any(-1)  # a beam before it goes on from the same one
    gone = ~(p[:, None, :] == torch.arange(w, device="cuda")[:, None]).any(-1)
    free = (~gone).to(torch.int8).sort(dim=1, stable=True).indices
    giver = torch.where(again, free.gather(1, (again.cumsum(1) - 1).clamp(min=0)), p)
    base = torch.arange(b, device="cuda")[:, None] * w
    parent, giver = (base + p).flatten(), (base + giver).flatten()
    whole = (s.len // ps).repeat_interleave(w)[:, None]
    col = torch.arange(s.table.shape[1], device="cuda")
    table = torch.where(col < whole, s.table[parent], s.table[giver])
    src, dst = (s.table[x].long().gather(1, whole)[:, 0] for x in (parent, giver))
    here = torch.arange(ps, device="cuda")[:, None, None] < (s.len % ps).repeat_interleave(w)[:, None, None, None]
    for x in (s.code, s.s, s.m):
        x[dst] = torch.where(here[..., None], x[src], x[dst])
    return table, *_plain_read(s, s.tail_off, s.tail_start, table, sum(s.tail), ps)


def _frequencies(case):
    """Angles per position of the rotated pairs, f64, and each pair's axis."""
    sec = _sections(case)
    axis = torch.repeat_interleave(torch.arange(len(sec)), torch.tensor(sec)).cuda()
    half = sum(sec)
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    if not case["restart"]:
        return 10000.0 ** (-i / half), axis
    n = torch.tensor(sec, dtype=torch.float64, device="cuda")
    return 10000.0 ** (-(i - (n.cumsum(0) - n)[axis]) / n[axis]), axis


def _rotate(x, cos, sin, layout, back):
    """x [tokens, heads, dim] f32; cos, sin [tokens, rot / 2]."""
    h = cos.shape[1]
    c, s = cos[:, None], -sin[:, None] if back else sin[:, None]
    if layout == HALF:
        a, b = x[..., :h], x[..., h:2 * h]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * h:]], -1)


# ------------------------------------------------------------------ what is measured
def prepare(case, seed):
    s = _inputs(case, seed)
    ps = case.get("page")
    if case["op"] == "rope":
        freq, s.axis = _frequencies(case)
        if own:
            from klearu_amd import paged

            s.rope = paged.Rope(2 * sum(_sections(case)), case["max_pos"], sections=_sections(case), restart=case["restart"],
                                layout=paged.HALF if case["layout"] == HALF else paged.INTERLEAVED)
        else:
            a = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * freq
            s.cos, s.sin = a.cos().float(), a.sin().float()
    elif case["op"] != "beam":
        if case["op"] == "reorder":
            off, start, v = s.tail_off, s.tail_start, s.all_v
        else:
            off, start, v = _off(s.lens_host), torch.zeros_like(s.len), getattr(s, "all_v", s.all_k)
        if own:
            from klearu_amd import paged

            s.cache = paged.PagedKv(case["kv_heads"], case["dim"], s.pages, page_size=ps)
            s.cache.append(s.all_k, v, off, start, s.table)
        else:
            _pool(s, case)
            _plain_put(s, s.all_k, v, off, start, s.table, ps)
        s.all_k = s.all_v = v = None
    elif own:
        from klearu_amd import beam

        s.select = beam.select
    return s


def run(s):
    case = s.case
    if case["op"] == "weights":
        if own:
            return s.cache.attention_weights(s.q, s.lse, s.off, s.len, s.table, s.acc, scale=s.scale, window=case["window"],
                                             max_rows=s.most_rows, max_len=s.most_len)
        return _plain_weights(s, case)
    if case["op"] == "evict":
        if own:
            kept, left, acc = s.cache.evict(s.acc, s.len, s.table, case["keep"], recent=case["recent"], first=case["first"])
            return kept, left, acc, *s.cache.gather(s.left_off, s.zero, s.table, s.left, dtype=torch.bfloat16)
        return _plain_evict(s, case)
    if case["op"] == "beam":
        return s.select(s.logits, s.scores, case["k"], done=s.done, end=s.end) if own else _plain_beam(s, case)
    if case["op"] == "reorder":
        if own:
            table = s.cache.reorder(s.table, s.len, s.parent)
            return table, *s.cache.gather(s.tail_off, s.tail_start, table, sum(s.tail), dtype=torch.bfloat16)
        return _plain_reorder(s, case)
    if own:
        return s.rope.apply(s.x, s.pos, transpose=case["back"])
    pair = torch.arange(s.axis.numel(), device="cuda")
    at = s.pos[s.axis].T  # [tokens, pairs]
    return _rotate(s.x.float(), s.cos[at, pair], s.sin[at, pair], case["layout"], case["back"]).to(s.x.dtype)


def work(case):
    e = 4 if case.get("dtype") == "f32" else 2
    op = case["op"]
    if op == "rope":
        n, sec = case["tokens"] * case["heads"] * case["dim"], _sections(case)
        return {"bytes": 2 * n * e + case["tokens"] * (8 * sum(sec) + 8 * len(sec)), "flops": 3 * n}
    if op == "beam":
        n = case["batch"] * case["beams"]
        return {"bytes": n * (case["vocab"] * e + 4) + 12 * case["batch"] * case["k"], "flops": 4 * n * case["vocab"]}
    rows, lens = _sizes(case)
    kv, dim, ps = case["kv_heads"], case["dim"], case["page"]
    kept = dim / 2 + 4 * dim / GROUP  # bytes of one head's key or value
    if op == "reorder":
        w, tail = case["beams"], sum(n % ps for n in lens)
        cols = sum(-(-n // ps) + 1 for n in lens)
        # of w random parents (1 - 1 / w)^w are gone on average: as many pages are copied
        copied = tail * w * (1 - 1 / w) ** w
        return {"bytes": 8 * w * cols + copied * kv * 2 * 2 * kept + tail * w * kv * 2 * (kept + 2 * dim), "flops": 2 * tail * w * kv * 2 * dim}
    if op == "evict":
        left = sum(min(n, case["keep"]) for n in lens)
        moved = sum(case["keep"] for n in lens if n > case["keep"])
        return {"bytes": kv * (sum(lens) * 4 + left * 8 + moved * 2 * 2 * kept + left * 2 * (kept + 2 * dim)),
                "flops": 2 * left * kv * 2 * dim}
    heads, w = case["heads"], case["window"]
    share = case["selected"] / heads if case["selected"] else 1.0
    read = pairs = 0
    for r, n in zip(rows, lens):
        c = n - r
        lo = max(0, c + 1 - w) if w else 0
        read += n - lo
        full = r * c + r * (r + 1) // 2
        if w:  # rows that see more than the window
            short = max(0, min(r, w - c))
            full = short * c + short * (short + 1) // 2 + (r - short) * w
        pairs += full
    read_heads = min(kv, case["selected"]) if case["selected"] else kv
    return {"bytes": read * read_heads * (kept + 8) + sum(rows) * heads * (dim * e * share + 4),
            "flops": 2 * dim * heads * share * pairs}


# ------------------------------------------------------------------ 64 bits
def _exact_step_down(x):
    """x (f64) rounded to 8 significant bits, towards minus infinity."""
    frac, exp = torch.frexp(x)
    return torch.ldexp((frac * 256).floor(), exp - 8)


def _exact_held(x):
    """The values that a cache holding x (f64) stands for."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    m = _exact_step_down(g.min(-1, keepdim=True).values)
    # the quotients are f32 ones: f64's, rounded once more, are the same
    span = (g.max(-1, keepdim=True).values - m).float().double()
    s = -_exact_step_down(-(span / torch.full_like(span, 15)).float().double())
    c = ((g - m).float().double() / s).float().double().round().clamp(0, 15)
    return torch.where(s > 0, s * c + m, m + 0 * c).reshape(x.shape)


def exact(case, seed):
    s = _inputs(case, seed)
    op, kv, ps = case["op"], case.get("kv_heads"), case.get("page")
    if op == "weights":
        out, at, row = s.acc.double(), 0, 0
        heads = case["heads"]
        for b, (n, r) in enumerate(zip(s.lens_host, s.rows)):
            k, hide = _exact_held(s.all_k[at:at + n].double()), _hidden(s, b)
            for h in range(heads):
                norm = s.lse[row:row + r, h].double()
                a = s.q[row:row + r, h].double() @ k[:, h * kv // heads].T * s.scale
                a[hide] = -math.inf
                on = norm > -math.inf
                out[b, h * kv // heads, :n] += (a[on] - norm[on, None]).exp().sum(0)
            at, row = at + n, row + r
        return out
    if op == "evict":
        keep, n = case["keep"], s.cap
        kept = torch.full((case["batch"], kv, keep), -1, dtype=torch.int64, device="cuda")
        acc, ks, vs, at = torch.zeros_like(s.acc, dtype=torch.float64), [], [], 0
        for b, n in enumerate(s.lens_host):
            left = min(n, keep)
            for h in range(kv):
                held = set(range(min(case["first"], n))) | set(range(max(0, n - case["recent"]), n))
                if n > keep:
                    order = torch.argsort(-s.acc[b, h, :n].double(), stable=True).tolist()
                    rest = (j for j in order if j not in held)
                    mine = sorted(held | {next(rest) for _ in range(keep - len(held))})
                else:
                    mine = list(range(n))
                kept[b, h, :left] = _i64(mine)
                acc[b, h, :left] = s.acc[b, h, :n].double()[kept[b, h, :left]]
            rows = at + kept[b, :, :left].T  # [left, kv]
            head = torch.arange(kv, device="cuda")
            ks.append(_exact_held(s.all_k[rows, head].double()))
            vs.append(_exact_held(s.all_v[rows, head].double()))
            at += n
        return kept, s.len.clamp(max=keep), acc, torch.cat(ks), torch.cat(vs)
    if op == "beam":
        y = s.scores.double()[..., None] + torch.log_softmax(s.logits.double(), -1)
        if s.done is not None:
            y[s.done] = -math.inf
            y[..., s.end] = torch.where(s.done, s.scores.double(), y[..., s.end])
        y, at = y.flatten(1).sort(dim=1, descending=True, stable=True)
        k, n = case["k"], case["vocab"]
        return y[:, :k], at[:, :k].div(n, rounding_mode="floor"), at[:, :k].remainder(n)
    if op == "reorder":
        w, parent, table = case["beams"], s.parent.tolist(), s.table.tolist()
        k, v = _exact_held(s.all_k.double()), _exact_held(s.all_v.double())
        ends = s.tail_off.tolist()
        out, rows = [], []
        for b, n in enumerate(s.lens_host):
            free, used = [i for i in range(w) if i not in parent[b]], set()
            for i, p in enumerate(parent[b]):
                giver = free.pop(0) if p in used else p
                used.add(p)
                out.append(table[b * w + p][:n // ps] + table[b * w + giver][n // ps:])
                rows.append(torch.arange(ends[b * w + p], ends[b * w + p + 1], device="cuda"))
        rows = torch.cat(rows)
        return torch.tensor(out, device="cuda"), k[rows], v[rows]
    # the rotation as a product of complex numbers, pair by pair
    sec, freq, axis = _sections(case), [], []
    for a, n in enumerate(sec):
        for i in range(n):
            freq.append(10000.0 ** (-i / n if case["restart"] else -len(freq) / sum(sec)))
            axis.append(a)
    ang = s.pos.double()[axis].T * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones_like(ang), -ang if case["back"] else ang)[:, None]
    r, x = 2 * len(freq), s.x.double()
    if case["layout"] == HALF:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn
        y = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    return torch.cat([y, x[..., r:]], -1)
