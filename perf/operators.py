"""The measured operators of the caller-owned paged KV cache.

  append  rows of K and V into the pages of their sequences (fp16, int8 or int4), K and Q rotated to their positions on
          the way; the rows are then read back as the fp16 values that the cache holds
  attn    causal GQA attention of new rows over such pages, optionally with scores capped by a tanh, a bias that falls
          with the distance, rows that start seeing at their document, or a prefix that every row of a sequence sees

With `own` false the operators run in plain torch on the same pools of pages; with it true they are the framework's
ifr_paged_* calls.  Head layouts are those of the repository's two model classes (16/8 and 40/8 heads of 128), of its
reference's hybrid class (8/2 heads of 256), and generic ones.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

PAGE = 32
GROUP = 64   # dims that share an int4 scale and minimum
THETA = 1e6
FP16, INT8, INT4 = 0, 1, 2


def _append(name, fmt, nq, nkv, hd, seqs, rows, ctx, rotary):
    return {"name": name, "op": "append", "fmt": fmt, "nq": nq, "nkv": nkv, "hd": hd, "seqs": seqs, "rows": rows,
            "ctx": ctx, "rotary": rotary}


def _attn(name, fmt, nq, nkv, hd, seqs, rows, ctx, chunk=0, cap=0.0, bias=False, docs=0, prefix=False, f32=False):
    return {"name": name, "op": "attn", "fmt": fmt, "nq": nq, "nkv": nkv, "hd": hd, "seqs": seqs, "rows": rows,
            "ctx": ctx, "chunk": chunk, "cap": cap, "bias": bias, "docs": docs, "prefix": prefix, "f32": f32}


def listed():
    return [
        # one user's decode token into a 4-bit cache: latency only
        _append("append_int4_1", INT4, 16, 8, 128, 1, 1, 1000, 128),
        # a full decode batch into an fp16 cache
        _append("append_fp16_64", FP16, 16, 8, 128, 64, 1, 1024, 128),
        # a long prompt's chunk of the wide model into an int8 cache, at a position inside a page
        _append("append_int8_2000", INT8, 40, 8, 128, 1, 2000, 2517, 128),
        # sixteen whole prompts into a 4-bit cache, a quarter of each head rotated
        _append("append_int4_prompts", INT4, 8, 2, 256, 16, 1100, 1100, 64),
        # one user's decode row over a 4-bit cache: the smallest attention
        _attn("int4_decode_1", INT4, 16, 8, 128, 1, 1, 1000),
        # the decode rows of a full batch, ragged contexts: the stream of 4-bit pages
        _attn("int4_decode_64", INT4, 16, 8, 128, 64, 1, 2048),
        # a few users with long documents in context, for which a cache is held in 4 bits at all
        _attn("int4_long_16", INT4, 16, 8, 128, 16, 1, 32000),
        # speculative verify rows of the wide model, in fp32 for the quantizer of the O projection
        _attn("int4_verify_28", INT4, 40, 8, 128, 28, 5, 1536, f32=True),
        # the ordinary mixed iteration over a 4-bit cache: decode rows and a prefill chunk
        _attn("int4_mixed", INT4, 16, 8, 128, 24, 1, 1024, chunk=512),
        # decode of a model with capped scores, heads of 256
        _attn("cap_decode_32", FP16, 8, 2, 256, 32, 1, 4096, cap=50.0),
        # one row of packed documents, prefilled in one call, with capped scores
        _attn("cap_docs_prefill", FP16, 16, 8, 128, 1, 8000, 8000, cap=30.0, docs=4),
        # a chunk of a prefix model with a distance bias and a head for each query head, int8 cache
        _attn("bias_prefix_chunk", INT8, 16, 16, 64, 2, 1000, 2777, bias=True, prefix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    nq, nkv, hd = rng.choice([(16, 8, 128), (16, 8, 128), (40, 8, 128), (8, 2, 256), (16, 16, 64), (32, 4, 128),
                              (12, 1, 128), (9, 3, 64)])
    fmt = rng.choice([FP16, INT8, INT4, INT4])
    if rng.random() < 0.3:
        seqs = _log(rng, 1, 64)
        rows = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, max(16, 16000 // seqs))])
        if seqs * rows * (nq + 2 * nkv) * hd <= 5.4e7:  # sixteen prompts of the largest listed case
            return {k: v for k, v in _append("", fmt, nq, nkv, hd, seqs, rows, rows + _log(rng, 1, 4096) - 1,
                                             rng.choice([hd, hd, hd // 2, 0])).items() if k != "name"}
    while True:
        form = rng.choice(["decode", "decode", "chunk", "mixed"])
        seqs, rows, chunk = _log(rng, 1, 64), rng.choice([1, 1, 1, _log(rng, 2, 8)]), 0
        ctx = _log(rng, 1, 16000) + rows - 1
        if form == "chunk":
            seqs, rows = rng.choice([1, 1, 2, 3]), _log(rng, 17, 2048)
            ctx = rows + _log(rng, 1, 4096) - 1
        elif form == "mixed":
            chunk, ctx = _log(rng, 17, 700), _log(rng, 16, 2048) + rows
        cap = rng.choice([0.0, 0.0, 30.0, 50.0])
        bias, prefix = rng.random() < 0.3, rng.random() < 0.25
        docs = rng.choice([0, 0, rng.randint(2, 9)])
        c = _attn("", fmt, nq, nkv, hd, seqs, rows, ctx, chunk, cap, bias, docs, prefix, rng.random() < 0.4)
        del c["name"]
        # within the largest listed cases, and within what the plain form pads its keys and scores to
        longest, w = min(2 * ctx + 64, 40000), work(c)
        if w["bytes"] <= 6e8 and w["flops"] <= 9e10 and seqs * longest * nkv * hd <= 5e8 and \
                (seqs + 1) * max(rows, chunk) * nq * (longest + chunk) <= 6e8:
            return c


# ---- the pages -----------------------------------------------------------------------------------------------------
# A page holds 32 tokens, per kv head one block [K codes | K scales | V codes | V scales], in the order of the
# framework's matrix instructions (IFR_PAGED_* in intfer_amd.h):
#   K  fp16  [hd/8][32 t][8]                 t = token of the page, d = 32 i + 8 g + e
#      int8, int4  [32 t][4 g][hd/32 i][8 e]   int4: element e in nibble 4 (e % 2) + e / 2 of its dword
#   V  token t = 16 jh + 4 g + jl
#      fp16  [4 g][hd][2 jh][4 jl]
#      int8, int4  [4 g][16 c][hd/16 n][2 jh][4 jl], d = 16 n + c; int4: element j = 4 jh + jl in nibble 4 (j % 2) + j / 2
#   scales, fp16: int8 K [16 t % 16][2 t / 16], V [4 g][2 jh][4 jl]
#                 int4 K [16 t % 16][hd/64 u][2 t / 16][scale, minimum], V [4 g][hd/64 u][scale, minimum][2 jh][4 jl]

def _part_bytes(fmt, hd):
    return {FP16: 64 * hd, INT8: 32 * hd + 64, INT4: 18 * hd}[fmt]


def _nibbles(device):
    e = torch.arange(8, device=device)
    return ((e % 2) * 4 + e // 2) * 4


def _to_k(x, fmt, hd):
    """[..., 32, hd] of elements -> the K order, [..., n]."""
    b = x.shape[:-2]
    if fmt == FP16:
        return x.reshape(*b, 32, hd // 8, 8).transpose(-3, -2).reshape(*b, -1)
    return x.reshape(*b, 32, hd // 32, 4, 8).transpose(-3, -2).reshape(*b, -1)


def _from_k(x, fmt, hd):
    b = x.shape[:-1]
    if fmt == FP16:
        return x.reshape(*b, hd // 8, 32, 8).transpose(-3, -2).reshape(*b, 32, hd)
    return x.reshape(*b, 32, 4, hd // 32, 8).transpose(-3, -2).reshape(*b, 32, hd)


def _to_v(x, fmt, hd):
    b = x.shape[:-2]
    n = len(b)
    if fmt == FP16:  # jh g jl d -> g d jh jl
        return x.reshape(*b, 2, 4, 4, hd).permute(*range(n), n + 1, n + 3, n, n + 2).reshape(*b, -1)
    # jh g jl n c -> g c n jh jl
    return x.reshape(*b, 2, 4, 4, hd // 16, 16).permute(*range(n), n + 1, n + 4, n + 3, n, n + 2).reshape(*b, -1)


def _from_v(x, fmt, hd):
    b = x.shape[:-1]
    n = len(b)
    if fmt == FP16:  # g d jh jl -> jh g jl d
        return x.reshape(*b, 4, hd, 2, 4).permute(*range(n), n + 2, n, n + 3, n + 1).reshape(*b, 32, hd)
    return x.reshape(*b, 4, 16, hd // 16, 2, 4).permute(*range(n), n + 3, n, n + 4, n + 2, n + 1).reshape(*b, 32, hd)


def _codes_bytes(c, fmt):
    """Codes in their order -> bytes."""
    if fmt == FP16:
        return c.contiguous().view(torch.uint8)
    if fmt == INT8:
        return c.to(torch.int8).view(torch.uint8)
    w = (c.reshape(*c.shape[:-1], -1, 8).to(torch.int64) << _nibbles(c.device)).sum(-1)
    w = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    return w.contiguous().view(torch.uint8)


def _bytes_codes(b, fmt):
    if fmt == FP16:
        return b.contiguous().view(torch.float16)
    if fmt == INT8:
        return b.contiguous().view(torch.int8)
    w = b.contiguous().view(torch.int32)
    return ((w[..., None] >> _nibbles(b.device).to(torch.int32)) & 15).to(torch.uint8).reshape(*w.shape[:-1], -1)


def _to_scales(s, fmt, hd, v):
    """Scales [..., 32, G, 1 or 2] fp16 -> bytes of their order."""
    b, n = s.shape[:-3], s.dim() - 3
    G, two = s.shape[-2:]
    if not v:  # t = (th, c): th c u w -> c u th w
        s = s.reshape(*b, 2, 16, G, two).permute(*range(n), n + 1, n + 2, n, n + 3)
    else:      # jh g jl u w -> g u w jh jl
        s = s.reshape(*b, 2, 4, 4, G, two).permute(*range(n), n + 1, n + 3, n + 4, n, n + 2)
    return s.reshape(*b, -1).contiguous().view(torch.uint8)


def _from_scales(x, fmt, hd, v):
    G, two = (1, 1) if fmt == INT8 else (hd // GROUP, 2)
    x = x.contiguous().view(torch.float16)
    b, n = x.shape[:-1], x.dim() - 1
    if not v:
        x = x.reshape(*b, 16, G, 2, two).permute(*range(n), n + 2, n, n + 1, n + 3)
    else:
        x = x.reshape(*b, 4, G, two, 2, 4).permute(*range(n), n + 3, n, n + 4, n + 1, n + 2)
    return x.reshape(*b, 32, G, two)


def _pack(codes, scales, fmt, hd, v):
    c = _codes_bytes((_to_v if v else _to_k)(codes, fmt, hd), fmt)
    return c if fmt == FP16 else torch.cat([c, _to_scales(scales, fmt, hd, v)], -1)


def _unpack(part, fmt, hd, v):
    """Bytes of a K or V part [..., n] -> codes [..., 32, hd], scales [..., 32, G, 1 or 2] or None."""
    n = part.shape[-1] if fmt == FP16 else 32 * hd // (1 if fmt == INT8 else 2)
    codes = (_from_v if v else _from_k)(_bytes_codes(part[..., :n], fmt), fmt, hd)
    return codes, None if fmt == FP16 else _from_scales(part[..., n:], fmt, hd, v)


def _quantize(x, fmt):
    """fp32 [..., hd] -> codes, scales as the cache stores them."""
    if fmt == FP16:
        return x.half(), None
    if fmt == INT8:
        s = (x.abs().amax(-1, keepdim=True) / 127).half()
        f = s.float()
        y = x * torch.where(f > 0, 1 / f, torch.zeros_like(f))
        return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127).to(torch.int8), s[..., None]
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    z, s = lo.half(), ((hi - lo) / 15).half()
    f = s.float()
    y = (g - z.float()) * torch.where(f > 0, 1 / f, torch.zeros_like(f))
    return torch.round(y).clamp(0, 15).to(torch.uint8).reshape(x.shape), torch.cat([s, z], -1)


def _values(codes, scales, fmt):
    """fp16 values that codes stand for."""
    if fmt == FP16:
        return codes
    if fmt == INT8:
        return (codes.float() * scales[..., 0].float()).half()
    g = codes.reshape(*codes.shape[:-1], -1, GROUP).float()
    return (g * scales[..., :1].float() + scales[..., 1:].float()).half().reshape(codes.shape)


# ---- one state -----------------------------------------------------------------------------------------------------

def _layout(case, seed):
    """Per sequence: new rows and cached tokens (the new ones among them)."""
    rng = np.random.default_rng([21, seed])
    S, R, ctx = case["seqs"], case["rows"], case["ctx"]
    if S == 1 or R > 16:
        lens = [ctx] * S
        lens = [int(max(R, n - rng.integers(0, max(1, n // 8)))) if i else n for i, n in enumerate(lens)]
    else:  # ragged contexts around the median (log-normal), as a serving batch has them
        lens = [int(x) for x in np.clip(np.round(ctx * np.exp(0.6 * rng.standard_normal(S))), R, min(2 * ctx + 64, 40000))]
    rows = [R] * S
    if case.get("chunk"):
        rows.append(case["chunk"])
        lens.append(case["chunk"] + int(rng.integers(0, case["ctx"] + 1)))
    return rows, lens


def _masks(case, seed, rows, lens):
    """First visible position of each row (packed documents) and the prefix of each sequence, or None."""
    rng = np.random.default_rng([22, seed])
    first = prefix = None
    if case.get("docs"):
        out = []
        for r, n in zip(rows, lens):
            starts = np.concatenate([[0], np.sort(rng.integers(1, max(n, 2), case["docs"] - 1))])
            pos = np.arange(n - r, n)
            out.append(starts[np.searchsorted(starts, pos, side="right") - 1])
        first = np.concatenate(out).astype(np.int32)
    if case.get("prefix"):
        prefix = np.array([rng.integers(0, n + 1) for n in lens], np.int32)
    return first, prefix


def _content(g, shape, nkv, hd):
    """Cached rows: unit values, with the few large channels that keys have."""
    x = torch.randn(*shape, nkv, hd, generator=g, device="cuda")
    ch = torch.randperm(hd, generator=g, device="cuda")[: hd // 32]
    x[..., ch] *= 4
    return x


def prepare(case, seed):
    c = dict(case)
    fmt, nq, nkv, hd = c["fmt"], c["nq"], c["nkv"], c["hd"]
    rows, lens = _layout(c, seed)
    first, prefix = _masks(c, seed, rows, lens)
    rng = np.random.default_rng([23, seed])
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, M, used = len(rows), sum(rows), [-(-n // PAGE) for n in lens]
    n_pages = sum(used) + 3
    table = np.zeros((S, max(used)), np.int32)
    order = rng.permutation(n_pages)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    part = _part_bytes(fmt, hd)
    pool = torch.empty(n_pages, nkv, 2, part, dtype=torch.uint8, device="cuda")
    for lo in range(0, n_pages, 4096):
        n = min(4096, n_pages - lo)
        for v in (0, 1):
            codes, scales = _quantize(_content(g, (n, PAGE), nkv, hd).transpose(1, 2).contiguous(), fmt)
            pool[lo:lo + n, :, v] = _pack(codes, scales, fmt, hd, v)
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    seq = np.repeat(np.arange(S), rows)
    s = {"case": c, "pool": pool, "rows": rows, "lens": lens, "np_table": table, "np_first": first, "np_prefix": prefix,
         "table": torch.from_numpy(table).cuda().long(), "pos": torch.from_numpy(pos).cuda(),
         "seq": torch.from_numpy(seq).cuda(), "len": torch.tensor(lens, device="cuda"), "M": M,
         "slot": torch.from_numpy(np.concatenate([np.arange(r) for r in rows])).cuda(),
         "first": torch.zeros(M, dtype=torch.int64, device="cuda") if first is None else torch.from_numpy(first).cuda().long(),
         "prefix": torch.zeros(S, dtype=torch.int64, device="cuda") if prefix is None else torch.from_numpy(prefix).cuda().long(),
         "q": torch.randn(M, nq, hd, generator=g, device="cuda").half()}
    if c["op"] == "append":
        s["k"], s["v"] = (_content(g, (M,), nkv, hd).half() for _ in range(2))
        half = c["rotary"] // 2
        ang = torch.arange(max(lens), device="cuda").double()[:, None] / THETA ** (
            torch.arange(half, device="cuda").double()[None] * 2 / max(1, c["rotary"]))
        s["cos"], s["sin"] = torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()
        s["out"] = {"q": torch.empty_like(s["q"]), "k": torch.empty_like(s["k"]), "v": torch.empty_like(s["v"])}
    else:
        s["slopes"] = None
        if c["bias"]:
            s["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, nq + 1, device="cuda").float() / nq).contiguous()
        s["out"] = torch.empty(M, nq, hd, device="cuda", dtype=torch.float32 if c["f32"] else torch.float16)
    if own:
        _plan(s)
    return s


# ---- the framework's calls -----------------------------------------------------------------------------------------

_device = []


def _plan(s):
    """The plan of this batch, as a serving program makes it once per iteration for all of its layers."""
    import intfer_amd as ia
    from intfer_amd import _abi
    c = s["case"]
    if not _device:
        _device.append(ia.Device(0))
    s["paged"] = ia.Paged(_device[0], c["fmt"], c["nq"], c["nkv"], c["hd"], s["pool"].shape[0])
    s["paged"].set(s["rows"], s["lens"], s["np_table"], first=s["np_first"], prefix=s["np_prefix"])
    p = lambda t: None if t is None else C.c_void_p(t.data_ptr())  # noqa: E731
    qw, kw = c["nq"] * c["hd"], c["nkv"] * c["hd"]
    if c["op"] == "append":
        o = s["out"]
        s["args"] = _abi.PagedRows(k=p(s["k"]), v=p(s["v"]), k_stride=kw, v_stride=kw, q=p(s["q"]), q_out=p(o["q"]),
                                   q_stride=qw, q_out_stride=qw, cos=p(s["cos"]), sin=p(s["sin"]), rotary=c["rotary"],
                                   max_pos=s["cos"].shape[0])
        s["read"] = (p(o["k"]), p(o["v"]))
    else:
        s["args"] = _abi.PagedQuery(q=p(s["q"]), q_stride=qw, out=p(s["out"]), out_stride=qw, out_f32=int(c["f32"]),
                                    scale=0.0, softcap=c["cap"], slopes=p(s["slopes"]))


def _run_own(s):
    from intfer_amd import _abi
    lib, h, pool = _abi.lib(), s["paged"].h, s["pool"].data_ptr()
    if s["case"]["op"] == "append":
        _abi.check(lib.ifr_paged_append(h, pool, C.byref(s["args"])), "ifr_paged_append")
        _abi.check(lib.ifr_paged_read(h, pool, *s["read"]), "ifr_paged_read")
    else:
        _abi.check(lib.ifr_paged_attention(h, pool, C.byref(s["args"])), "ifr_paged_attention")
    return s["out"]


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _rotate(x, s):
    half = s["cos"].shape[1]
    if not half:
        return x
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _run_append(s):
    c = s["case"]
    fmt, hd = c["fmt"], c["hd"]
    page, slot = s["table"][s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    touched, index = torch.unique(page, return_inverse=True)
    out = {"q": _rotate(s["q"].float(), s).half()}
    for v, (name, x) in enumerate((("k", _rotate(s["k"].float(), s)), ("v", s["v"].float()))):
        codes, scales = _unpack(s["pool"][touched, :, v], fmt, hd, v)
        new, ns = _quantize(x, fmt)
        codes[index, :, slot] = new
        if scales is not None:
            scales[index, :, slot] = ns
        s["pool"][touched, :, v] = _pack(codes, scales, fmt, hd, v)
        codes, scales = _unpack(s["pool"][touched, :, v], fmt, hd, v)
        out[name] = _values(codes[index, :, slot], None if scales is None else scales[index, :, slot], fmt)
    return out


def _run_attn(s):
    c = s["case"]
    fmt, nq, nkv, hd, M = c["fmt"], c["nq"], c["nkv"], c["hd"], s["M"]
    S, R, G = len(s["rows"]), max(s["rows"]), nq // nkv
    block = s["pool"][s["table"]]                            # [S, pages, nkv, 2, bytes]
    T = block.shape[1] * PAGE
    k, v = (_values(*_unpack(block[:, :, :, i], fmt, hd, i), fmt).float().permute(0, 2, 1, 3, 4).reshape(S, nkv, T, hd)
            for i in (0, 1))
    t = torch.arange(T, device="cuda")
    v = torch.where((t[None] < s["len"][:, None])[:, None, :, None], v, 0.0)
    q = torch.zeros(S, R, nq, hd, device="cuda")
    q[s["seq"], s["slot"]] = s["q"].float()
    pad = lambda x: torch.zeros(S, R, dtype=torch.int64, device="cuda").index_put_((s["seq"], s["slot"]), x)  # noqa: E731
    pos, first = pad(s["pos"]), pad(s["first"])
    q = q.reshape(S, R, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, G * R, hd)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(S, nkv, G, R, T) / math.sqrt(hd)
    if c["cap"]:
        a = c["cap"] * torch.tanh(a / c["cap"])
    if s["slopes"] is not None:
        far = (pos[:, :, None] - t).abs().float()            # [S, R, T]
        a = a - s["slopes"].reshape(1, nkv, G, 1, 1) * far[:, None, None]
    end = torch.minimum(torch.maximum(pos + 1, s["prefix"][:, None]), s["len"][:, None])
    seen = (t >= first[:, :, None]) & (t < end[:, :, None])
    a = torch.where(seen[:, None, None], a, -math.inf)
    m = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul((e / torch.where(total > 0, total, 1.0)).reshape(S, nkv, G * R, T), v)
    o = o.reshape(S, nkv, G, R, hd).permute(0, 3, 1, 2, 4).reshape(S, R, nq, hd)[s["seq"], s["slot"]]
    return o if c["f32"] else o.half()


def run(s):
    if own:
        return _run_own(s)
    return _run_append(s) if s["case"]["op"] == "append" else _run_attn(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    nq, nkv, hd, fmt = case["nq"], case["nkv"], case["hd"], case["fmt"]
    rows, lens = _layout(case, 0)
    M = sum(rows)
    token = nkv * 2 * _part_bytes(fmt, hd) / PAGE
    if case["op"] == "append":  # q, k, v read, q written, the rows' codes written, read again, and returned
        return {"bytes": M * (2 * (2 * nq * hd + 4 * nkv * hd) + 2 * token + 4 * case["rotary"]),
                "flops": 3.0 * M * (nq + nkv) * case["rotary"]}
    first, prefix = _masks(case, 0, rows, lens)
    bytes_, seen, m = M * nq * hd * (2.0 + (4 if case["f32"] else 2)), 0.0, 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        lo = np.zeros(r) if first is None else first[m:m + r]
        hi = np.maximum(np.arange(n - r, n) + 1, 0 if prefix is None else prefix[i])
        seen += float(np.maximum(hi - lo, 0).sum())
        bytes_ += (float(hi.max()) - float(lo.min())) * token
        m += r
    return {"bytes": bytes_, "flops": 4.0 * nq * hd * seen}


# ---- the same in 64 bits, sequence by sequence ---------------------------------------------------------------------

def _offsets(fmt, hd, v):
    """Element number of (token, dim) inside a part, by the formulas of the layout."""
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(hd, device="cuda")[None]
    if not v:
        if fmt == FP16:
            return ((d // 8) * 32 + t) * 8 + d % 8
        return ((t * 4 + (d // 8) % 4) * (hd // 32) + d // 32) * 8 + d % 8
    g, j = (t % 16) // 4, 4 * (t // 16) + t % 4
    if fmt == FP16:
        return (g * hd + d) * 8 + j
    return ((g * 16 + d % 16) * (hd // 16) + d // 16) * 8 + j


def _read64(part, fmt, hd, v):
    """uint8 [n, nkv, bytes] -> float64 [n * 32, nkv, hd] of the fp16 values."""
    at = _offsets(fmt, hd, v)
    n, nkv = part.shape[:2]
    t, u = torch.arange(PAGE, device="cuda")[:, None], torch.arange(hd, device="cuda")[None] // GROUP
    g, j = (t % 16) // 4, 4 * (t // 16) + t % 4
    if fmt == FP16:
        x = part.contiguous().view(torch.float16)[:, :, at.reshape(-1)].double()
    elif fmt == INT8:
        codes = part[:, :, at.reshape(-1)].view(torch.int8).double().reshape(n, nkv, PAGE, hd)
        sc = part[:, :, 32 * hd:].contiguous().view(torch.float16)
        x = codes * sc[:, :, (g * 8 + j if v else (t % 16) * 2 + t // 16).reshape(-1)].double()[..., None]
    else:
        e = at % 8
        nib = (e % 2) * 4 + e // 2
        b = part[:, :, (at // 8 * 4 + nib // 2).reshape(-1)].reshape(n, nkv, PAGE, hd)
        codes = torch.where(nib % 2 == 1, b >> 4, b & 15).double()
        sc = part[:, :, 16 * hd:].contiguous().view(torch.float16)
        U = hd // GROUP
        i_s = (g * U + u) * 16 + j if v else (((t % 16) * U + u) * 2 + t // 16) * 2
        i_z = i_s + (8 if v else 1)
        x = codes * sc[:, :, i_s.reshape(-1)].double().reshape(n, nkv, PAGE, hd)
        x = x + sc[:, :, i_z.reshape(-1)].double().reshape(n, nkv, PAGE, hd)
    return x.reshape(n, nkv, PAGE, hd).half().double().transpose(1, 2).reshape(n * PAGE, nkv, hd)


def _exact_append(s):
    c = s["case"]
    r = c["rotary"] // 2
    cos, sin = s["cos"].double()[s["pos"]][:, None, :], s["sin"].double()[s["pos"]][:, None, :]

    def turned(x):
        x = x.double().clone()
        a, b = x[..., :r].clone(), x[..., r:2 * r].clone()
        x[..., :r] = a * cos - b * sin
        x[..., r:2 * r] = b * cos + a * sin
        return x

    def held(x):
        if c["fmt"] == FP16:
            return x
        if c["fmt"] == INT8:
            sc = (x.abs().amax(-1, keepdim=True) / 127).half().double()
            y = x / sc
            return (torch.floor(y.abs() + 0.5).clamp(max=127) * torch.sign(y)) * sc
        y = x.reshape(x.shape[0], x.shape[1], -1, GROUP)
        z = y.amin(-1, keepdim=True)
        sc = ((y.amax(-1, keepdim=True) - z) / 15).half().double()
        z = z.half().double()
        return (torch.round((y - z) / sc).clamp(0, 15) * sc + z).reshape(x.shape)

    return {"q": turned(s["q"]), "k": held(turned(s["k"])), "v": held(s["v"].double())}


def _exact_attn(s):
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    out, m = [], 0
    for i, (r, n) in enumerate(zip(s["rows"], s["lens"])):
        part = s["pool"][s["table"][i, : -(-n // PAGE)]]
        k, v = (_read64(part[:, :, w], c["fmt"], hd, w)[:n] for w in (0, 1))
        t = torch.arange(n, device="cuda")[None]
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        hidden = (t < s["first"][m:m + r, None]) | ((t > pos) & (t >= s["prefix"][i]))
        for h in range(nq):
            a = s["q"][m:m + r, h].double() @ k[:, h // (nq // nkv)].T.contiguous() * hd ** -0.5
            if c["cap"]:
                a = torch.tanh(a / c["cap"]) * c["cap"]
            if s["slopes"] is not None:
                a = a - s["slopes"][h].double() * (pos - t).abs()
            a = a.masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)
            out.append(p @ v[:, h // (nq // nkv)].contiguous())
        out[-nq:] = [torch.stack(out[-nq:], 1)]
        m += r
    return torch.cat(out)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _exact_append(s) if case["op"] == "append" else _exact_attn(s)
