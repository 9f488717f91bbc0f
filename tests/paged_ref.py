"""The caller-owned paged KV cache in numpy, from the formulas of
include/intfer_amd.h, in float64: what the paged tests hold the kernels to."""
import functools
import math

import numpy as np

FP16, INT8, INT4 = 0, 1, 2
PAGE, GROUP = 32, 64
EPS32 = 2.0 ** -24  # half a step of fp32, relative
EPS16 = 2.0 ** -11  # half a step of fp16, relative


def part_bytes(fmt, hd):
    return {FP16: 64 * hd, INT8: 32 * hd + 64, INT4: 18 * hd}[fmt]


def _td(hd):
    return np.arange(PAGE)[:, None], np.arange(hd)[None, :]


@functools.lru_cache(None)
def element(fmt, hd, v):
    """Element number of (token, dim) in a K or V part."""
    t, d = _td(hd)
    if not v:
        if fmt == FP16:
            return (d // 8 * 32 + t) * 8 + d % 8
        return ((t * 4 + d // 8 % 4) * (hd // 32) + d // 32) * 8 + d % 8
    g, j = t % 16 // 4, 4 * (t // 16) + t % 4
    if fmt == FP16:
        return (g * hd + d) * 8 + j
    return ((g * 16 + d % 16) * (hd // 16) + d // 16) * 8 + j


@functools.lru_cache(None)
def scale_index(fmt, hd, v):
    """fp16 index of the scale of (token, dim) behind the codes; the minimum's offset."""
    t, d = _td(hd)
    u, g, j = d // GROUP, t % 16 // 4, 4 * (t // 16) + t % 4
    if fmt == INT8:
        return (g * 8 + j if v else t % 16 * 2 + t // 16) + 0 * d, 0
    if not v:
        return ((t % 16 * (hd // GROUP) + u) * 2 + t // 16) * 2, 1
    return (g * (hd // GROUP) + u) * 16 + j, 8


def read_part(part, fmt, hd, v):
    """One K or V part (uint8 [bytes]) -> (codes [32, hd], scale, minimum) or fp16 values."""
    e = element(fmt, hd, v)
    if fmt == FP16:
        return part.view(np.float16)[e], None, None
    sc = part[(32 if fmt == INT8 else 16) * hd:].view(np.float16)
    i, off = scale_index(fmt, hd, v)
    if fmt == INT8:
        return part[:32 * hd].view(np.int8)[e], sc[i], None
    nib = e // 8 * 8 + 4 * (e % 2) + e % 8 // 2
    b = part[nib // 2]
    return np.where(nib % 2 == 1, b >> 4, b & 15), sc[i], sc[i + off]


def values(codes, s, z, fmt):
    """fp16 values that codes stand for (float64 sums of a 4- or 8-bit code and fp16 are exact)."""
    if fmt == FP16:
        return codes
    with np.errstate(over="ignore", invalid="ignore"):
        x = codes.astype(np.float64) * s.astype(np.float64)
        return (x if z is None else x + z.astype(np.float64)).astype(np.float16)


def quantize(x, fmt):
    """fp32 [n, hd] -> codes, scales [n, hd], minima [n, hd] by the format's rule in fp32."""
    x = np.asarray(x, np.float32)
    one = np.float32(1)
    with np.errstate(all="ignore"):
        if fmt == FP16:
            return x.astype(np.float16), None, None
        if fmt == INT8:
            bad = ~np.isfinite(x).all(-1, keepdims=True)
            s = np.where(bad, np.float32(0), np.abs(x)).max(-1, keepdims=True) * (one / np.float32(127))
            s = np.minimum(s, np.float32(515.5)).astype(np.float16)  # 127 * 516 would round to infinity
            f = s.astype(np.float32)
            y = np.where(bad, np.float32(0), x) * np.where(f > 0, one / f, np.float32(0))
            y = np.clip(y, np.float32(-127), np.float32(127))
            c = np.trunc(y + np.copysign(np.float32(0.5), y))
            s = np.where(bad, np.float16(np.nan), s)
            return c.astype(np.int8), np.broadcast_to(s, x.shape), None
        g = x.reshape(len(x), -1, GROUP)
        bad = ~np.isfinite(g).all(-1, keepdims=True)
        g = np.where(bad, np.float32(0), g)
        lo, hi = (np.clip(f(-1, keepdims=True), -65504, 65504).astype(np.float32) for f in (g.min, g.max))
        z, s = lo.astype(np.float16), ((hi - lo) * (one / np.float32(15))).astype(np.float16)
        over = 15 * s.astype(np.float64) + z.astype(np.float64) >= 65520  # code 15 would round to infinity
        s = np.where(over, (s.view(np.uint16) - 1).astype(np.uint16).view(np.float16), s)
        f = s.astype(np.float32)
        y = (g - z.astype(np.float32)) * np.where(f > 0, one / f, np.float32(0))
        c = np.clip(np.rint(y), 0, 15).astype(np.uint8)
        s, z = np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(0), z)
        rep = lambda a: np.broadcast_to(a, g.shape).reshape(x.shape)  # noqa: E731
        return c.reshape(x.shape), rep(s), rep(z)


def write_token(parts, fmt, hd, v, t, x):
    """Store one token's rows x (fp32 [n_kv, hd]) in its heads' parts (uint8 [n_kv, bytes]), in place."""
    c, s, z = quantize(x, fmt)
    e = element(fmt, hd, v)[t]
    if fmt == FP16:
        parts.view(np.float16)[:, e] = c
        return
    i, off = scale_index(fmt, hd, v)
    k = (32 if fmt == INT8 else 16) * hd
    sc = parts[:, k:].view(np.float16)
    sc[:, i[t]] = s
    if fmt == INT8:
        parts[:, :k].view(np.int8)[:, e] = c
        return
    sc[:, i[t] + off] = z
    nib = e // 8 * 8 + 4 * (e % 2) + e % 8 // 2
    lo, hi = nib % 2 == 0, nib % 2 == 1
    parts[:, nib[lo] // 2] = (parts[:, nib[lo] // 2] & 0xF0) | c[:, lo]
    parts[:, nib[hi] // 2] = (parts[:, nib[hi] // 2] & 0x0F) | (c[:, hi] << 4)


def tables(max_pos, rotary, theta=1e6):
    ang = np.arange(max_pos)[:, None] / theta ** (np.arange(rotary // 2)[None] * 2 / max(1, rotary))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rotate(x, pos, cos, sin):
    """fp16 [M, heads, hd] -> fp32, each product and the sum rounded."""
    h = cos.shape[1]
    x = x.astype(np.float32)
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    with np.errstate(all="ignore"):
        return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


class Cache:
    """Pages [n_pages, n_kv, 2, part] as bytes, and a batch over them."""

    def __init__(self, fmt, n_kv, hd, n_pages, rng=None, fill=None):
        self.fmt, self.n_kv, self.hd = fmt, n_kv, hd
        n = part_bytes(fmt, hd)
        shape = (n_pages, n_kv, 2, n)
        if fill is not None:
            self.pool = np.full(shape, fill, np.uint8)
            return
        if fmt == FP16:
            self.pool = rng.standard_normal((n_pages, n_kv, 2, n // 2)).astype(np.float16).view(np.uint8).reshape(shape)
            return
        self.pool = rng.integers(0, 256, shape, dtype=np.uint8)
        k = (32 if fmt == INT8 else 16) * hd
        sc = np.abs(rng.standard_normal((n_pages, n_kv, 2, (n - k) // 2))) * 0.1 + 0.02
        if fmt == INT8:
            self.pool[..., :k] = np.where(self.pool[..., :k] == 128, 0, self.pool[..., :k])
            sc *= 0.2
        else:  # minima where they belong
            sc[:, :, 0, 1::2] *= -8
            v = sc[:, :, 1].reshape(n_pages, n_kv, -1, 2, 8)
            v[..., 1, :] *= -8
        self.pool[..., k:] = sc.astype(np.float16).view(np.uint8)

    def gather(self, pages, n):
        """K and V of a sequence's first n tokens, float64 [n, n_kv, hd]."""
        out = []
        for v in (0, 1):
            x = np.empty((len(pages) * PAGE, self.n_kv, self.hd))
            for i, p in enumerate(pages):
                for h in range(self.n_kv):
                    x[i * PAGE:(i + 1) * PAGE, h] = values(*read_part(self.pool[p, h, v], self.fmt, self.hd, v), self.fmt)
            out.append(x[:n])
        return out

    def append(self, pages, pos, k, v):
        """Row (fp32 [n_kv, hd]) at position pos."""
        for w, x in ((0, k), (1, v)):
            write_token(self.pool[pages[pos // PAGE], :, w], self.fmt, self.hd, w, pos % PAGE, x)


def attention(q, k, v, pos, lo, hi, scale, cap, slopes, out_f32):
    """One sequence's rows q [r, nq, hd] over k, v [n, nkv, hd] (float64).  Returns the output and how far a
    kernel may be from it.

    The bound: a score is a sum of hd products in fp32 and some 12 roundings after it (scale, cap, bias, the factor
    log2 e, the difference to the maximum), so it is off by (hd + 12) eps of the sum of its terms' magnitudes; exp2
    adds two steps and the fp16 pair of a weight 2^-22 of it or, below 2^-14 of the largest, 2^-25.  A weight that is
    off by the factor 1 + e moves the output by at most 2 e sum p |v|.  Then the output's own rounding.  For an fp16
    output the weights of the numerator are rounded to fp16, each by at most 2^-11 of itself (the sum of the
    denominator is not): at most 2^-11 sum p |v| more."""
    r, nq, hd = q.shape
    n, nkv = k.shape[:2]
    out, bound = np.zeros((r, nq, hd)), np.zeros((r, nq, hd))
    t = np.arange(n)
    seen = (t >= lo[:, None]) & (t < hi[:, None])
    # rows at once where a zero weight takes a value out, else each over the tokens that it sees
    every = np.isfinite(k).all() and np.isfinite(v).all()
    parts = [(np.flatnonzero(seen.any(1)), t)] if every else \
        [(np.array([i]), np.flatnonzero(seen[i])) for i in range(r) if seen[i].any()]
    for h in range(nq):
        for i, ts in parts:
            kk, vv, see = k[ts, h // (nq // nkv)], v[ts, h // (nq // nkv)], seen[i][:, ts]
            av = np.abs(vv)
            with np.errstate(all="ignore"):
                a = scale * (q[i, h] @ kk.T)
                size = scale * (np.abs(q[i, h]) @ np.abs(kk).T)
                if cap:
                    a = cap * np.tanh(a / cap)
                if slopes is not None:
                    far = float(slopes[h]) * np.abs(pos[i, None] - ts)
                    a, size = a - far, size + far
                # only the terms whose weight counts carry their error into the output
                top = np.where(see, a, -np.inf).max(1, keepdims=True)
                w = np.where(see, np.exp(a - top), 0.0)
                total = w.sum(1, keepdims=True)
                p = w / total
                out[i, h] = p @ vv
                e = (hd + 12) * EPS32 * (size + np.abs(a) + np.abs(top)) + 2.0 ** -21
                e = p * np.where(see, e, 0.0)
                bound[i, h] = 2 * (e @ av + e.sum(1, keepdims=True) * (p @ av)) + 2.0 ** -25 * (see @ av) / total
                if not out_f32:
                    bound[i, h] += EPS16 * (p @ av)
    step = EPS32 if out_f32 else EPS16
    with np.errstate(all="ignore"):
        return out, bound + 2 * step * np.abs(out) + (0 if out_f32 else 2.0 ** -24)


def batch(rng, rows, lens, extra=2):
    """Fragmented page tables and rows' positions for sequences of the given lengths."""
    used = [-(-n // PAGE) for n in lens]
    n_pages = sum(used) + extra
    order = rng.permutation(n_pages)
    table = np.zeros((len(lens), max(used + [1])), np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)]).astype(np.int64) if rows else np.zeros(0, np.int64)
    return n_pages, table, pos


def expect(cache, rows, lens, table, q, first=None, prefix=None, scale=None, cap=0.0, slopes=None, out_f32=False):
    """The batch's attention and its bound, [M, nq, hd]."""
    outs, bounds, m = [], [], 0
    scale = scale or 1 / math.sqrt(cache.hd)
    for s, (r, n) in enumerate(zip(rows, lens)):
        if not r:
            continue
        k, v = cache.gather(table[s, :-(-n // PAGE)], n)
        pos = np.arange(n - r, n)
        lo = np.zeros(r, np.int64) if first is None else np.maximum(first[m:m + r], 0)
        hi = np.minimum(np.maximum(pos + 1, 0 if prefix is None else prefix[s]), n)
        o, b = attention(q[m:m + r].astype(np.float64), k, v, pos, lo, hi, scale, cap, slopes, out_f32)
        outs.append(o)
        bounds.append(b)
        m += r
    return np.concatenate(outs), np.concatenate(bounds)
