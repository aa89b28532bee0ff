"""Plain forms of the paged 4-bit cache and its attention, on the host: the format by its
definition in f32, everything computed from it in f64."""
import numpy as np
import torch

G = 32


def bf16_down(x):
    """f32 -> the largest BF16 value at or below it (as f32)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    neg = u >> 31 == 1
    v = np.where(neg, (u + 0xFFFF) >> 16, u >> 16).astype(np.uint32)
    return (v << 16).astype(np.uint32).view(np.float32)


def quantize(x):
    """x [..., dim] f32 -> (c, s, m) of every element, f64; s NaN and c = m = 0 where a group stands for NaN."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // G, G)
    with np.errstate(all="ignore"):
        m = bf16_down(g.min(-1, keepdims=True))
        s = -bf16_down(-((g.max(-1, keepdims=True) - m) / np.float32(15)))
        bad = ~(np.abs(g) < np.float32(2.0 ** 100)).all(-1, keepdims=True)
        c = np.clip(np.rint((g - m) / s), 0, 15)
    c = np.where(s > 0, c, 0)
    c, s, m = np.where(bad, 0, c), np.where(bad, np.nan, s), np.where(bad, 0, m)
    shape = x.shape
    return tuple(np.broadcast_to(a, g.shape).reshape(shape).astype(np.float64) for a in (c, s, m))


def values(x):
    c, s, m = quantize(x)
    return s * c + m


def seen(n, length, causal, window):
    """[n, length] which positions each of the last n rows sees."""
    pos = np.arange(length - n, length)[:, None]
    j = np.arange(length)[None]
    ok = np.ones((n, length), bool)
    if causal:
        ok &= j <= pos
    if window:
        ok &= j > pos - window
    return ok


def attention(q, kraw, vraw, scale, causal=True, window=0, bf16=True, many=False, fine=False):
    """One sequence: q [n, heads, dim] f64, kraw, vraw [length, kv, dim] f32 as appended ->
    (out, lse, tolerance of out, tolerance of lse), f64.

    The tolerances count the roundings of the method: scores are f32 sums of q (128 + c) s and
    q (m - 128 s), so their magnitudes are B = scale sum |q| (271 s + |m|), summed by at most dim + 16
    additions; an exponential is off by 2^-21 and by 2^-22 of its argument; a weight that the second product
    takes is rounded to 8 bits (2^-8; f32 rows: three times 8, 2^-24) of p s c + p |m|; its sums over the positions have
    magnitudes sum p (271 s + |m|) and at most length / 4 + 64 additions in a row; out is rounded last.  Tiles of
    many BF16 rows (`many`) take keys and values rounded to 8 bits: 2^-8 of |q| |k| and of p |v| more, and divide by
    the sum of the rounded weights: 2^-8 of |o| <= sum p |v| once more.  Few positions (`fine`): weights in two
    terms, 2^-16."""
    n, heads, dim = q.shape
    length, kv = kraw.shape[:2]
    kc, ks, km = quantize(kraw)
    vc, vs, vm = quantize(vraw)
    k, v = ks * kc + km, vs * vc + vm
    ok = seen(n, length, causal, window)
    out, lse = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf)
    tol, tol_l = np.zeros((n, heads, dim)), np.zeros((n, heads))
    u = 2.0 ** -24
    up, uo = (2.0 ** -16 if fine else 2.0 ** -8, 2.0 ** -8) if bf16 else (u, u)
    for h in range(heads):
        g = h * kv // heads
        with np.errstate(all="ignore"):
            t = np.where(ok, q[:, h] @ k[:, g].T * scale, -np.inf)
            big = scale * (np.abs(q[:, h]) @ (271 * ks[:, g] + np.abs(km[:, g])).T)
        some = ok.any(-1)
        top = np.where(some, np.max(t, -1, where=ok, initial=-np.inf), 0.0)
        with np.errstate(all="ignore"):
            p = np.exp(t - top[:, None])
            p = np.where(ok, p, 0.0)
            tot = p.sum(-1)
            w = p / np.where(some, tot, 1.0)[:, None]
            o = w @ np.nan_to_num(v[:, g])
            o[(ok.astype(np.float64) @ np.isnan(v[:, g])) > 0] = np.nan
            err = (dim + 16) * u * big + 2.0 ** -21 + 2.0 ** -22 * np.abs(np.where(ok, t - top[:, None], 0.0))
            if many:
                err = err + 2.0 ** -8 * scale * (np.abs(q[:, h]) @ np.abs(np.nan_to_num(k[:, g])).T)
            err = np.where(ok, err, 0.0)
            depth = (length / 4 + 64) * u
            sg = np.nan_to_num(vs[:, g])  # groups that stand for NaN have no tolerance
            mag = sg * vc[:, g] + np.abs(vm[:, g])
            if many:
                mag = mag + 2 * np.abs(np.nan_to_num(v[:, g]))
            tol[:, h] = ((w * err) @ np.abs(np.nan_to_num(v[:, g])) + (w * err).sum(-1)[:, None] * np.abs(o)
                         + up * (w @ mag) + depth * (w @ (271 * sg + np.abs(vm[:, g]))) + uo * np.abs(o))
        out[:, h] = np.where(some[:, None], o, 0.0)
        lse[:, h] = np.where(some, top + np.log(np.where(some, tot, 1.0)), -np.inf)
        tol_l[:, h] = err.max(-1) + depth + 2.0 ** -22 * np.abs(np.where(some, lse[:, h], 0.0))
    return out, lse, tol, tol_l


class Pages:
    """Page tables of sequences over a pool: shuffled pages, unused entries out of range."""

    def __init__(self, lens, page, extra=2, seed=0, spare=1):
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + extra
        order = np.random.default_rng(seed).permutation(self.pages)
        cols = max(need + [1]) + spare
        t, at = np.full((len(lens), cols), -1, np.int32), 0
        for b, n in enumerate(need):
            t[b, :n] = order[at:at + n]
            at += n
        self.table = torch.from_numpy(t)


def offsets(rows):
    return torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int64)


def bf16_values(x):
    return torch.from_numpy(np.asarray(x, np.float32)).to(torch.bfloat16)


def keys(rng, n, heads, dim):
    """Rows as a layer makes them: a few channels off zero and large."""
    shift = rng.normal(0, 1, (heads, dim)) * np.where(rng.random((heads, dim)) < 0.05, 4.0, 0.2)
    return (rng.normal(0, 1, (n, heads, dim)) + shift).astype(np.float32)
