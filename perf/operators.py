"""Rotary positions, the paged 4-bit K/V cache and the attention that reads it, as cases to time and compare.

A case is a dict of plain values; its "op" names the operator:

  rope    rotates rows x [tokens, heads, dim] by their positions (or, with "back", takes gradients back through that)
  append  rotates the keys of new tokens, puts keys and values into the pages of their sequences in 4 bits, and reads
          those rows back as the values they now stand for
  attn    attention of new rows over their sequences' pages: one row a sequence (decode) or many (prefill, chunks)

run() computes the operators in plain torch, or, where `own` is true, through klearu_amd.paged.  exact() gives the
outputs in 64 bits from the definitions.

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
        # One decode step's queries of a 7B-class model: launch latency.
        dict(name="rope_b1_f32", op="rope", tokens=1, heads=32, dim=128, rot=128, layout=HALF, scaling="none",
             factor=1.0, max_pos=4096, dtype="f32", back=False),
        # A prompt's queries at the far positions of a context sixteen times the trained one.
        dict(name="rope_8191_far", op="rope", tokens=8191, heads=32, dim=128, rot=128, layout=HALF, scaling="by_parts",
             factor=16.0, max_pos=131072, dtype="bf16", back=False),
        # Gradients of queries whose heads rotate in their first half only, interleaved pairs.
        dict(name="rope_back_2049", op="rope", tokens=2049, heads=32, dim=64, rot=32, layout=INTERLEAVED,
             scaling="linear", factor=4.0, max_pos=16384, dtype="f32", back=True),
        # One new token of one sequence, 7B-class layer.
        dict(name="append_b1_f32", op="append", batch=1, rows=1, ragged=False, start=1999, kv_heads=32, dim=128,
             page=64, layout=HALF, dtype="f32"),
        # A serving batch's decode step, 1.1B-class layer (four heads of 64), pages of 16.
        dict(name="append_b64", op="append", batch=64, rows=1, ragged=False, start=4000, kv_heads=4, dim=64, page=16,
             layout=HALF, dtype="bf16"),
        # Prompts of different lengths put into the cache together.
        dict(name="append_prompts", op="append", batch=5, rows=4001, ragged=True, start=0, kv_heads=8, dim=128,
             page=64, layout=INTERLEAVED, dtype="bf16"),
        # Decode of one sequence over about 2000 positions, half of the heads selected, as the head predictor gives them.
        dict(name="attn_b1_f32", op="attn", batch=1, rows=1, ragged=False, cached=1999, heads=32, kv_heads=32, dim=128,
             page=64, selected=16, window=0, lse=False, dtype="f32"),
        # Eight sequences of that model, every head.
        dict(name="attn_b8", op="attn", batch=8, rows=1, ragged=False, cached=2047, heads=32, kv_heads=32, dim=128,
             page=64, selected=0, window=0, lse=False, dtype="bf16"),
        # A serving batch of a 1.1B-class model (32 heads over 4), contexts of every length.
        dict(name="attn_b64_ragged", op="attn", batch=64, rows=1, ragged=True, cached=4095, heads=32, kv_heads=4,
             dim=64, page=16, selected=0, window=0, lse=False, dtype="bf16"),
        # One long document, one question: all the parallelism is along the cache.
        dict(name="attn_b1_long", op="attn", batch=1, rows=1, ragged=False, cached=131071, heads=32, kv_heads=8,
             dim=128, page=64, selected=0, window=0, lse=True, dtype="bf16"),
        # A prompt attends to itself.
        dict(name="attn_prompt", op="attn", batch=1, rows=4096, ragged=False, cached=0, heads=32, kv_heads=8, dim=128,
             page=64, selected=0, window=0, lse=False, dtype="bf16"),
        # Chunks of several prompts over what is cached of them, a sliding window, wide heads.
        dict(name="attn_chunks", op="attn", batch=4, rows=331, ragged=True, cached=5000, heads=16, kv_heads=2, dim=256,
             page=32, selected=0, window=1024, lse=True, dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    layout = rng.choice([HALF, INTERLEAVED])
    if op == "rope":
        heads = _logint(rng, 1, 64)
        tokens = _logint(rng, 1, max(2, 8191 * 32 * 128 // (heads * dim * (2 if dtype == "f32" else 1))))
        scaling = rng.choice(["none", "linear", "base", "by_parts"])
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, rot=dim // rng.choice([1, 1, 2, 4]), layout=layout,
                    scaling=scaling, factor=1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 16])),
                    max_pos=_logint(rng, 2048, 131072), dtype=dtype, back=rng.random() < 0.4)
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    if op == "append":
        batch = _logint(rng, 1, 128)
        rows = rng.choice([1, _logint(rng, 2, 4001)])
        rows = max(1, min(rows, 20000 * 8 * 128 // (2 * batch * kv * dim)))
        return dict(op=op, batch=batch, rows=rows, ragged=rows > 1 and rng.random() < 0.7,
                    start=rng.choice([0, _logint(rng, 1, 4000)]), kv_heads=kv, dim=dim, page=page, layout=layout,
                    dtype=dtype)
    group = rng.choice([1, 1, 2, 4, 8])
    heads = kv * group if kv * group <= 64 else kv
    window = rng.choice([0, 0, _logint(rng, 16, 2048)])
    if rng.random() < 0.6:  # decode
        batch = _logint(rng, 1, 64)
        cached = _logint(rng, 1, max(2, min(131071, 64 * 4096 * 4 * 64 // (batch * kv * dim))))
        return dict(op=op, batch=batch, rows=1, ragged=rng.random() < 0.6, cached=cached, heads=heads, kv_heads=kv,
                    dim=dim, page=page, selected=rng.choice([0, 0, max(1, heads // 2)]), window=window,
                    lse=rng.random() < 0.3, dtype=dtype)
    batch = rng.choice([1, 1, 2, 3, 5])
    rows = _logint(rng, 2, 2000 // batch if dtype == "bf16" else 700 // batch)
    cached = rng.choice([0, _logint(rng, 1, 4000)])
    cached = min(cached, max(0, 4096 * 4096 * 16 * 128 // (batch * rows * heads * dim) - rows))
    return dict(op=op, batch=batch, rows=rows, ragged=rng.random() < 0.7, cached=cached, heads=heads, kv_heads=kv,
                dim=dim, page=page, selected=0, window=window, lse=rng.random() < 0.3, dtype=dtype)


# ------------------------------------------------------------------ inputs
class State:
    pass


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _sizes(case):
    """Rows and earlier positions of each sequence, on the host: as given, or spread below that when ragged."""
    b = case["batch"]
    g = torch.Generator().manual_seed(case["rows"] * 7919 + b)
    rows, before = [case["rows"]] * b, [case.get("cached", case.get("start", 0))] * b
    if case["ragged"]:
        part = torch.rand(2, b, generator=g)
        rows = [max(1, int(r * (0.05 + 0.95 * float(p)))) for r, p in zip(rows, part[0])]
        before = [int(c * (0.02 + 0.98 * float(p))) for c, p in zip(before, part[1])]
        rows[0], before[-1] = case["rows"], before[-1] if case["op"] == "append" else case.get("cached", 0)
    return rows, before


def _keys(gen, n, heads, dim):
    """Keys or values as a layer makes them: normal, a few channels of each head far larger and off zero."""
    gain = 0.6 + 0.8 * torch.rand(heads, dim, generator=gen, device="cuda")
    big = (torch.rand(heads, dim, generator=gen, device="cuda") < 0.03).float()
    shift = torch.randn(heads, dim, generator=gen, device="cuda") * (0.1 + 3.0 * big)
    x = torch.randn(n, heads, dim, generator=gen, device="cuda")
    return x * gain * (1 + big) + shift


def _inputs(case, seed):
    """What the seed alone gives: tensors on the GPU and sizes on the host."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dt, s = _dtype(case), State()
    if case["op"] == "rope":
        s.x = torch.randn(case["tokens"], case["heads"], case["dim"], generator=gen, device="cuda").to(dt)
        n, m = case["tokens"], case["max_pos"]
        first = int(torch.randint(0, max(1, m - n), (1,), generator=torch.Generator().manual_seed(int(seed))))
        s.pos = (first + torch.arange(n, device="cuda")) % m
        return s
    rows, before = _sizes(case)
    s.rows, s.before, s.total = rows, before, sum(rows)
    kv, dim, ps = case["kv_heads"], case["dim"], case["page"]
    s.lens = [r + c for r, c in zip(rows, before)]
    s.off = torch.tensor([0] + rows, device="cuda").cumsum(0)
    s.start = torch.tensor(before, dtype=torch.int64, device="cuda")
    s.len = torch.tensor(s.lens, dtype=torch.int64, device="cuda")
    need = [-(-n // ps) for n in s.lens]
    s.cols, s.pages = max(need), sum(need) + 3
    order = torch.randperm(s.pages, generator=torch.Generator().manual_seed(int(seed) + 1))
    table, at = torch.zeros(len(rows), s.cols, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    s.table = table.cuda()
    if case["op"] == "append":
        # one projection gives keys and values side by side
        s.kv = torch.cat([_keys(gen, s.total, kv, dim), _keys(gen, s.total, kv, dim)], 1).to(dt)
        s.k, s.v = s.kv[:, :kv], s.kv[:, kv:]
        s.max_pos = max(4096, max(s.lens))
        return s
    heads = case["heads"]
    s.all_k = _keys(gen, sum(s.lens), kv, dim).to(dt)
    s.all_v = _keys(gen, sum(s.lens), kv, dim).to(dt)
    s.qkv = torch.empty(s.total, heads + 2 * kv, dim, dtype=dt, device="cuda")
    s.q = s.qkv[:, :heads]  # queries lie in the projection's rows
    s.q.copy_(torch.randn(s.total, heads, dim, generator=gen, device="cuda") * 1.2)
    s.scale = dim ** -0.5
    s.sel = None
    if case["selected"]:
        rank = torch.rand(s.total, heads, generator=gen, device="cuda").argsort(1)[:, :case["selected"]]
        s.sel = rank.sort(1).values.to(torch.int32)
    return s


# ------------------------------------------------------------------ plain forms
def _frequencies(case, dev):
    """Angles per position of the rotated pairs, f64."""
    r = case.get("rot", case["dim"])
    i = torch.arange(0, r, 2, dtype=torch.float64, device=dev) / r
    scaling, factor, theta = case.get("scaling", "none"), case.get("factor", 1.0), 10000.0
    if scaling == "base":
        theta *= factor ** (r / (r - 2))
    f = theta ** -i
    if scaling == "linear":
        f = f / factor
    if scaling == "by_parts":  # whole turns over the trained length decide: few are stretched, many are kept
        turns = f * _trained(case) / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f


def _trained(case):
    return max(1, int(case["max_pos"] / case["factor"]))


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case.get("scaling") == "by_parts" else 1.0


def _table(case, max_pos):
    a = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * _frequencies(case, "cuda")
    return (a.cos() * _magnitude(case)).float(), (a.sin() * _magnitude(case)).float()


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


def _bf16_down(x):
    """Largest BF16 value at or below x (f32 in and out)."""
    r = x.to(torch.bfloat16)
    over = r.float() > x
    down = torch.nextafter(r, torch.full_like(r, -math.inf))
    return torch.where(over, down, r).float()


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
    n = (s.pages, case["page"], 2, case["kv_heads"])
    s.code = torch.zeros(*n, case["dim"] // 2, dtype=torch.uint8, device="cuda")
    s.s = torch.zeros(*n, case["dim"] // GROUP, dtype=torch.bfloat16, device="cuda")
    s.m = torch.zeros_like(s.s)


def _places(off, start, table, total, page):
    """(page, place in it, position, sequence) of each row."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(off, row, right=True) - 1
    pos = start[seq] + row - off[seq]
    return table[seq, pos // page].long(), pos % page, pos, seq


def _plain_append(s, k, v, off, start, total, page, rope=None, layout=HALF):
    pg, at, pos, _ = _places(off, start, s.table, total, page)
    k = k.float()
    if rope is not None:
        k = _rotate(k, rope[0][pos], rope[1][pos], layout, False)
    s.code[pg, at], s.s[pg, at], s.m[pg, at] = _quantize(torch.stack([k, v.float()], 1))
    return pg, at


def _plain_attention(s, case):
    kv, dim, ps, heads = case["kv_heads"], case["dim"], case["page"], case["heads"]
    b, gs, n, most = len(s.rows), heads // kv, max(s.lens), max(s.rows)
    t = s.table.long()
    x = _values(s.code[t], s.s[t], s.m[t]).flatten(1, 2)[:, :n]  # [b, n, 2, kv, dim]
    k, v = x[:, :, 0].permute(0, 2, 3, 1), x[:, :, 1].transpose(1, 2)
    i = torch.arange(most, device="cuda")
    q = s.q[(s.off[:-1, None] + i).clamp(max=s.total - 1)].float()  # [b, most, heads, dim]
    q = q.view(b, most, kv, gs, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, gs * most, dim)
    w = torch.matmul(q, k).view(b, kv, gs, most, n) * s.scale
    pos = (s.start[:, None] + i)[:, :, None]
    j = torch.arange(n, device="cuda")
    seen = j <= pos
    if case["window"]:
        seen = seen & (j > pos - case["window"])
    w = w.masked_fill(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - top)
    tot = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(b, kv, gs * most, n), v).view(b, kv, gs, most, dim) / tot
    lse = (top + tot.log())[..., 0]
    row = torch.arange(s.total, device="cuda")
    seq = torch.searchsorted(s.off, row, right=True) - 1
    at = row - s.off[seq]
    o, lse = (y.flatten(1, 2)[seq, :, at] for y in (o, lse))  # [total, heads, ...]
    if s.sel is not None:
        on = torch.zeros(s.total, heads, dtype=torch.bool, device="cuda").scatter(1, s.sel.long(), True)
        o, lse = o.masked_fill(~on[..., None], 0.0), lse.masked_fill(~on, -math.inf)
    return (o.to(s.q.dtype), lse) if case["lse"] else o.to(s.q.dtype)


# ------------------------------------------------------------------ what is measured
def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = case
    if own:
        from klearu_amd import paged

        if case["op"] != "attn":
            r, most = (case["rot"], case["max_pos"]) if case["op"] == "rope" else (case["dim"], s.max_pos)
            kind = {"none": paged.SCALE_NONE, "linear": paged.SCALE_LINEAR, "base": paged.SCALE_BASE,
                    "by_parts": paged.SCALE_BY_PARTS}[case.get("scaling", "none")]
            parts = dict(original_len=_trained(case)) if kind == paged.SCALE_BY_PARTS else {}
            s.rope = paged.Rope(r, most, layout=paged.HALF if case["layout"] == HALF else paged.INTERLEAVED,
                                scaling=kind, factor=case.get("factor", 1.0), magnitude=_magnitude(case), **parts)
        if case["op"] != "rope":
            s.cache = paged.PagedKv(case["kv_heads"], case["dim"], s.pages, page_size=case["page"])
    else:
        if case["op"] != "attn":
            s.rope = _table(case, case["max_pos"] if case["op"] == "rope" else s.max_pos)
        if case["op"] != "rope":
            _pool(s, case)
    if case["op"] == "attn":  # the cache holds every position, this step's rows too
        off = torch.tensor([0] + s.lens, device="cuda").cumsum(0)
        zero = torch.zeros_like(s.start)
        if own:
            s.cache.append(s.all_k, s.all_v, off, zero, s.table)
        else:
            _plain_append(s, s.all_k, s.all_v, off, zero, sum(s.lens), case["page"])
        del s.all_k, s.all_v
        s.most_rows, s.most_len = max(s.rows), max(s.lens)
    return s


def run(s):
    case = s.case
    if case["op"] == "rope":
        if own:
            return s.rope.apply(s.x, s.pos, transpose=case["back"])
        cos, sin = s.rope
        return _rotate(s.x.float(), cos[s.pos], sin[s.pos], case["layout"], case["back"]).to(s.x.dtype)
    if case["op"] == "append":
        if own:
            s.cache.append(s.k, s.v, s.off, s.start, s.table, rope=s.rope)
            return s.cache.gather(s.off, s.start, s.table, s.total, dtype=torch.bfloat16)
        pg, at = _plain_append(s, s.k, s.v, s.off, s.start, s.total, case["page"], s.rope, case["layout"])
        x = _values(s.code[pg, at], s.s[pg, at], s.m[pg, at]).to(torch.bfloat16)
        return x[:, 0], x[:, 1]
    if own:
        return s.cache.attention(s.q, s.off, s.len, s.table, scale=s.scale, window=case["window"], heads=s.sel,
                                 max_rows=s.most_rows, max_len=s.most_len, return_lse=case["lse"])
    return _plain_attention(s, case)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * e + case["tokens"] * (case["rot"] * 4 + 8), "flops": 3 * n}
    rows, before = _sizes(case)
    kept = case["dim"] / 2 + 4 * case["dim"] / GROUP  # bytes of one head's key or value
    if case["op"] == "append":
        n = 2 * sum(rows) * case["kv_heads"]
        return {"bytes": n * (case["dim"] * (e + 2) + 2 * kept), "flops": 12 * n * case["dim"]}
    heads, kv, w = case["heads"], case["kv_heads"], case["window"]
    share = case["selected"] / heads if case["selected"] else 1.0
    read = pairs = 0
    for r, c in zip(rows, before):
        lo = max(0, c + 1 - w) if w else 0
        read += c + r - lo
        full = r * c + r * (r + 1) // 2
        if w:  # rows that see more than the window
            short = max(0, min(r, w - c))
            full = short * c + short * (short + 1) // 2 + (r - short) * w
        pairs += full
    # of the kv heads, those with a selected head are read: at most as many as are selected
    read_heads = min(kv, case["selected"]) if case["selected"] else kv
    return {"bytes": 2 * read * read_heads * kept + sum(rows) * heads * case["dim"] * e * (1 + share),
            "flops": 4 * case["dim"] * heads * share * pairs}


# ------------------------------------------------------------------ 64 bits
def _exact_angles(case, pos):
    r = case.get("rot", case["dim"])
    scaling, factor = case.get("scaling", "none"), case.get("factor", 1.0)
    freq = []
    for i in range(r // 2):
        base = 10000.0 * factor ** (r / (r - 2)) if scaling == "base" else 10000.0
        f = base ** (-2.0 * i / r)
        if scaling == "linear":
            f /= factor
        elif scaling == "by_parts":
            turns = _trained(case) * f / (2 * math.pi)
            stay = min(1.0, max(0.0, (turns - 1.0) / 31.0))
            f = f * stay + f / factor * (1.0 - stay)
        freq.append(f)
    return pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")


def _exact_rope(case, x, pos, back):
    """The rotation as a product of complex numbers."""
    ang, mag = _exact_angles(case, pos), _magnitude(case)
    turn = torch.polar(torch.full_like(ang, mag), -ang if back else ang)[:, None]
    r, x = 2 * ang.shape[1], x.double()
    if case["layout"] == HALF:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn
        y = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    return torch.cat([y, x[..., r:]], -1)


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
    if case["op"] == "rope":
        return _exact_rope(case, s.x, s.pos, case["back"])
    if case["op"] == "append":
        pos = torch.cat([torch.arange(c, c + r, device="cuda") for r, c in zip(s.rows, s.before)])
        return _exact_held(_exact_rope(case, s.k, pos, False)), _exact_held(s.v.double())
    heads, kv = case["heads"], case["kv_heads"]
    out = torch.zeros(s.total, heads, case["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((s.total, heads), -math.inf, dtype=torch.float64, device="cuda")
    row = at = 0
    for r, c in zip(s.rows, s.before):
        n = r + c
        k, v = (_exact_held(y[at:at + n].double()) for y in (s.all_k, s.all_v))
        where = torch.arange(c, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None]
        hide = where < 0
        if case["window"]:
            hide |= where >= case["window"]
        for h in range(heads):
            a = s.q[row:row + r, h].double() @ k[:, h * kv // heads].T * s.scale
            a[hide] = -math.inf
            lse[row:row + r, h] = torch.logsumexp(a, -1)
            out[row:row + r, h] = torch.softmax(a, -1) @ v[:, h * kv // heads]
        row, at = row + r, at + n
    if s.sel is not None:
        keep = torch.zeros_like(lse).scatter_(1, s.sel.long(), 1.0) > 0
        out[~keep], lse[~keep] = 0.0, -math.inf
    return (out, lse) if case["lse"] else out
