"""One batch through the caller-owned paged cache (append, read back, attention) against tests/paged_ref.py, and the
calls that it refuses; run on the GPU by test_gpu_paged.py and on the CPU emulation by tests/hipemu/runner.py."""
import ctypes as C

import numpy as np

import tests.paged_ref as pr


def f16(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def poison(cache, table, lens):
    """NaN into every slot past a sequence's end."""
    for s, n in enumerate(lens):
        if n % 32 == 0:
            continue
        p = table[s, n // 32]
        for h in range(cache.n_kv):
            for v in (0, 1):
                part = cache.pool[p, h, v]
                if cache.fmt == pr.FP16:
                    part.view(np.uint16)[pr.element(cache.fmt, cache.hd, v)[n % 32:].reshape(-1)] = 0x7E01
                else:
                    i, _ = pr.scale_index(cache.fmt, cache.hd, v)
                    part[(32 if cache.fmt == pr.INT8 else 16) * cache.hd:].view(np.uint16)[i[n % 32:].reshape(-1)] = 0x7E01


def run_case(ia, dev, rng, fmt, nq, nkv, hd, rows, lens, cap=0.0, bias=False, first=None, prefix=None, out_f32=False,
             rotary=None, scale=0.0, say=print):
    n_pages, table, pos = pr.batch(rng, rows, lens)
    M, rotary = len(pos), hd if rotary is None else rotary
    cache = pr.Cache(fmt, nkv, hd, n_pages, rng)
    poison(cache, table, lens)
    q, k, v = f16(rng, M, nq, hd), f16(rng, M, nkv, hd), f16(rng, M, nkv, hd)
    cos, sin = pr.tables(max(lens + [1]), rotary)
    plan = ia.Paged(dev, fmt, nq, nkv, hd, n_pages)
    assert plan.pool_bytes() == cache.pool.nbytes
    plan.set(rows, lens, table, first=first, prefix=prefix)
    bufs = []

    def up(x):
        bufs.append(dev.upload(x))
        return bufs[-1]

    def new(n):
        bufs.append(dev.alloc(n))
        return bufs[-1]

    pool, qd, kd, vd = up(cache.pool), up(q), up(k), up(v)
    qo, ko, vo = new(q.nbytes), new(k.nbytes), new(v.nbytes)
    cd, sd = (up(cos).p, up(sin).p) if rotary else (None, None)
    try:
        plan.append(pool.p, kd.p, vd.p, qd.p, qo.p, cd, sd, rotary, cos.shape[0])
        plan.read(pool.p, ko.p, vo.p)
        kr = pr.rotate(k, pos, cos, sin)
        seq = np.repeat(np.arange(len(rows)), rows)
        for m in range(M):
            cache.append(table[seq[m]], pos[m], kr[m], v[m].astype(np.float32))
        assert np.array_equal(dev.download(pool, np.uint8, cache.pool.shape), cache.pool), "pages"
        assert np.array_equal(dev.download(qo, np.float16, q.shape), pr.rotate(q, pos, cos, sin).astype(np.float16)), "q"
        got = [dev.download(b, np.float16, k.shape).astype(np.float64) for b in (ko, vo)]
        m = 0
        for s, r in enumerate(rows):
            if r:
                held = cache.gather(table[s, :-(-lens[s] // 32)], lens[s])
                for w in (0, 1):
                    assert np.array_equal(got[w][m:m + r], held[w][lens[s] - r:]), ("read", w, s)
            m += r
        slopes = (2.0 ** (-8.0 * np.arange(1, nq + 1) / nq)).astype(np.float32) if bias else None
        sl = up(slopes).p if bias else None
        kind = np.float32 if out_f32 else np.float16
        guard = np.full((M + 1, nq, hd), 7.5, kind)  # a row behind the last one stays as it was
        out = up(guard)
        qr = dev.download(qo, np.float16, q.shape)
        plan.attention(pool.p, qo.p, out.p, out_f32=out_f32, softcap=cap, slopes=sl, scale=scale)
        res = dev.download(out, kind, guard.shape)
        assert (res[M] == 7.5).all()
        want, tol = pr.expect(cache, rows, lens, table, qr, first, prefix, scale, cap, slopes, out_f32)
        off = np.abs(res[:M].astype(np.float64) - want)
        worst = float(np.nanmax(off / np.maximum(tol, 1e-300))) if M else 0.0
        say(f"paged fmt={fmt} {nq}/{nkv}x{hd} rows={rows[:8]} lens={lens[:8]}: worst {worst:.3f} of the bound")
        assert np.isfinite(res[:M]).all()
        assert (off <= tol).all(), (worst, np.unravel_index(np.nanargmax(off / np.maximum(tol, 1e-300)), off.shape))
        return plan.cfg
    finally:
        plan.close()
        for b in bufs:
            b.free()


def refusals(ia, dev):
    """Every refusal of the ifr_paged_* calls, by return code; nothing is launched for any of them."""
    from intfer_amd import _abi
    L = ia.lib()
    H = C.c_void_p()

    def create(*cfg):
        return L.ifr_paged_create(dev.ctx, C.byref(_abi.PagedCfg(*cfg)), C.byref(H))

    for cfg, code in (((3, 4, 2, 128, 8), ia.IFR_EINVAL), ((-1, 4, 2, 128, 8), ia.IFR_EINVAL),
                      ((0, 4, 2, 96, 8), ia.IFR_EDECLINE), ((0, 4, 3, 128, 8), ia.IFR_EINVAL),
                      ((0, 4, 0, 128, 8), ia.IFR_EINVAL), ((0, 0, 1, 128, 8), ia.IFR_EINVAL),
                      ((0, 4, 2, 128, 0), ia.IFR_EINVAL)):
        assert create(*cfg) == code, cfg
        assert not H.value and L.ifr_paged_bytes(C.byref(_abi.PagedCfg(*cfg))) == 0
    assert L.ifr_paged_create(None, C.byref(_abi.PagedCfg(0, 4, 2, 128, 8)), C.byref(H)) == ia.IFR_EINVAL
    assert L.ifr_paged_destroy(None) == ia.IFR_OK
    plan = ia.Paged(dev, ia.KV_INT4, 4, 2, 128, 8)
    pool = dev.alloc(plan.pool_bytes() + 16)
    x = dev.alloc(1 << 16)
    a = x.p.value
    P, I = C.c_void_p, ia.IFR_EINVAL

    def rows(**over):
        d = dict(k=P(a), v=P(a + 4096), k_stride=256, v_stride=256, q=P(a + 8192), q_out=P(a + 16384), q_stride=512,
                 q_out_stride=512, cos=P(a + 32768), sin=P(a + 40960), rotary=128, max_pos=64)
        d.update(over)
        return C.byref(_abi.PagedRows(**d))

    def query(**over):
        d = dict(q=P(a), q_stride=512, out=P(a + 32768), out_stride=512, out_f32=0, scale=0.0, softcap=0.0, slopes=None)
        d.update(over)
        return C.byref(_abi.PagedQuery(**d))

    S = ia._abi.IFR_ESTATE
    assert L.ifr_paged_append(plan.h, pool.p, rows()) == S  # no batch yet
    assert L.ifr_paged_attention(plan.h, pool.p, query()) == S
    assert L.ifr_paged_read(plan.h, pool.p, P(a), P(a + 4096)) == S

    def bad_set(r, n, table, **more):
        try:
            plan.set(r, n, table, **more)
        except ia.IfrError as e:
            return e.code
        return ia.IFR_OK

    t = np.array([[0, 1], [2, 3]], np.int32)
    assert bad_set([1, 1], [40, 65], t) == I          # more pages than the table row has
    assert bad_set([1, 1], [40, 33], np.array([[0, 8], [2, 3]])) == I
    assert bad_set([1, 1], [40, 33], np.array([[0, -1], [2, 3]])) == I
    assert bad_set([-1, 1], [40, 33], t) == I
    assert bad_set([41, 1], [40, 33], t) == I         # more new rows than tokens
    assert bad_set([1, 1], [40, 33], t, prefix=[0, -1]) == I
    assert L.ifr_paged_set(plan.h, None) == I and L.ifr_paged_set(None, C.byref(_abi.PagedBatch())) == I
    for r, n, tb in (([1, 1], [40, 33], t.astype(np.int64) + 2**32), ([1, 1], [40, 2**32 + 33], t), ([1.5, 1], [40, 33], t),
                     ([1], [40, 33], t), ([1, 1], [40, 33], t[0])):
        try:
            plan.set(r, n, tb)
        except ValueError:
            continue
        raise AssertionError((r, n, tb))
    # a sequence without new rows takes no part, whatever stands in its entries
    assert bad_set([1, 0], [40, -3], np.array([[0, 1], [99, -7]])) == ia.IFR_OK
    assert bad_set([], [], np.zeros((0, 0))) == ia.IFR_OK  # an empty batch: calls do nothing
    assert L.ifr_paged_append(plan.h, pool.p, rows()) == ia.IFR_OK
    assert L.ifr_paged_attention(plan.h, pool.p, query()) == ia.IFR_OK
    assert L.ifr_paged_read(plan.h, pool.p, P(a), P(a + 4096)) == ia.IFR_OK
    # one page written by two sequences, or by two entries of one sequence: not appendable, still readable
    for r, n, tb in (([1, 1], [40, 40], [[0, 1], [2, 1]]), ([40], [40], [[5, 5]])):
        assert bad_set(r, n, np.array(tb, np.int32)) == ia.IFR_OK
        assert L.ifr_paged_append(plan.h, pool.p, rows(max_pos=4096)) == I
    plan.set([2, 1], [40, 33], t)
    for over in (dict(k=None), dict(v=None), dict(k=P(a + 2)), dict(v=P(a + 4104)), dict(k_stride=255), dict(k_stride=248),
                 dict(v_stride=260), dict(q=None), dict(q_out=None), dict(q=P(a + 8200)), dict(q_stride=504),
                 dict(q_out_stride=516), dict(cos=None), dict(sin=None), dict(cos=P(a + 32772)),
                 dict(sin=P(a + 40964)), dict(rotary=8), dict(rotary=144), dict(rotary=-16), dict(max_pos=39), dict(q_out=P(a + 8192 + 16)), dict(q_out=P(a)),
                 dict(q_out=P(a + 4096)), dict(k=P(pool.p.value)), dict(v=P(pool.p.value + 4096)),
                 dict(q_out=P(pool.p.value)), dict(q_out=P(a + 32768)), dict(q_out=P(a + 40960)), dict(k_stride=1 << 33),
                 dict(q_out_stride=1 << 33)):
        assert L.ifr_paged_append(plan.h, pool.p, rows(**over)) == I, over
    for over in (dict(q=None), dict(out=None), dict(q=P(a + 8)), dict(out=P(a + 32776)), dict(q_stride=511),
                 dict(q_stride=504), dict(out_stride=508), dict(out_f32=2), dict(scale=-1.0), dict(scale=float("nan")),
                 dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")),
                 dict(softcap=1e-44), dict(softcap=1e-32), dict(softcap=1e31), dict(scale=1e31),
                 dict(slopes=P(a + 32768)), dict(slopes=P(a + 32768 + 1024)), dict(out_stride=1 << 33),
                 dict(out=P(a)), dict(out=P(a + 1024)), dict(out=P(pool.p.value + 64))):
        assert L.ifr_paged_attention(plan.h, pool.p, query(**over)) == I, over
    for k, v in ((None, P(a)), (P(a), None), (P(a + 2), P(a + 4096)), (P(a), P(a + 256)), (P(a), P(pool.p.value))):
        assert L.ifr_paged_read(plan.h, pool.p, k, v) == I
    for f in (L.ifr_paged_append(plan.h, None, rows()), L.ifr_paged_append(plan.h, P(pool.p.value + 8), rows()),
              L.ifr_paged_append(None, pool.p, rows()), L.ifr_paged_append(plan.h, pool.p, None),
              L.ifr_paged_attention(plan.h, None, query()), L.ifr_paged_attention(plan.h, pool.p, None),
              L.ifr_paged_read(plan.h, None, P(a), P(a + 4096))):
        assert f == I
    plan.close()
    x.free()
    pool.free()
