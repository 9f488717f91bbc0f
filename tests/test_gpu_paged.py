"""The caller-owned paged KV cache on the GPU: pages bit for bit, attention within a bound derived from the roundings
(tests/paged_ref.py), and the calls in which such operators go wrong."""
import ctypes as C
import threading

import numpy as np
import pytest

import intfer_amd as ia
import tests.paged_ref as pr
from tests.conftest import announce
from tests.paged_check import f16, refusals, run_case

pytestmark = pytest.mark.gpu

FMT = [ia.KV_FP16, ia.KV_INT8, ia.KV_INT4]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("nq,nkv,hd,rows,lens,more", [
    (16, 8, 128, [1], [1], {}),                                   # one token, nothing cached
    (16, 8, 128, [1, 1, 1, 1], [31, 32, 33, 1000], {}),           # around a page's end
    (8, 2, 256, [1, 3, 2], [64, 65, 300], {"rotary": 64, "cap": 50.0}),
    (16, 16, 64, [1, 1], [97, 2049], {"bias": True, "out_f32": True}),
    (40, 8, 128, [5, 5], [133, 5], {"out_f32": True}),            # verify rows, 25 columns a head
    (9, 3, 64, [7, 0, 2], [50, 90, 35], {"rotary": 32}),          # a sequence that takes no part
    (12, 1, 128, [3, 1], [400, 7], {"scale": 0.25}),              # one kv head
    (32, 1, 64, [1, 2], [77, 64], {"rotary": 0}),                 # 32 columns from one row
    (71, 1, 128, [1, 3], [500, 40], {"cap": 20.0}),               # more: a row's heads over several tiles
    (192, 1, 64, [2], [333], {"bias": True, "out_f32": True}),
    (3, 3, 256, [1, 1, 1], [200, 5, 64], {"prefix": [0, 5, 64]}),  # a head each
])
def test_formats_and_shapes(dev, fmt, nq, nkv, hd, rows, lens, more):
    announce(f"paged fmt={fmt} {nq}/{nkv}x{hd} rows={rows} lens={lens} {more}")
    run_case(ia, dev, np.random.default_rng(nq + hd + fmt), fmt, nq, nkv, hd, rows, lens, **more)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("nq,nkv,hd,rows,lens,more", [
    (4, 2, 128, [150], [150], {}),                                # a whole prompt
    (4, 2, 128, [129, 1, 65], [517, 900, 65], {"cap": 20.0}),     # a chunk inside pages, a decode row, a short prompt
    (2, 2, 64, [200], [333], {"bias": True}),
    (4, 1, 256, [70], [131], {"out_f32": True}),
    (5, 1, 64, [33], [64], {"cap": 30.0, "bias": True, "out_f32": True}),
])
def test_chunks(dev, fmt, nq, nkv, hd, rows, lens, more):
    announce(f"paged chunk fmt={fmt} {nq}/{nkv}x{hd} rows={rows} lens={lens} {more}")
    run_case(ia, dev, np.random.default_rng(nq + hd + fmt), fmt, nq, nkv, hd, rows, lens, **more)


@pytest.mark.parametrize("rows,lens", [([1, 2], [200, 90]), ([90], [140])])
@pytest.mark.parametrize("fmt", FMT)
def test_masks(dev, fmt, rows, lens):
    """Documents, windows, prefixes, and rows that see nothing."""
    rng = np.random.default_rng(fmt)
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    for first, prefix in ((np.maximum(pos - 20, 0), None), (pos, None), (pos + 1, None), (pos // 37 * 37, lens),
                          (None, [n - 7 for n in lens]), (pos + 1, [n + 9 for n in lens]), (pos * 0 - 5, [0] * len(lens)),
                          (np.where(np.arange(len(pos)) % 3 == 0, 1 << 30, pos // 64 * 64), None)):
        announce(f"paged masks fmt={fmt} rows={rows} first={None if first is None else first[:4]} prefix={prefix}")
        run_case(ia, dev, rng, fmt, 4, 2, 128, rows, lens, first=first, prefix=prefix)


@pytest.mark.parametrize("rows,lens", [([1, 4], [400, 77]), ([300], [1700])])
@pytest.mark.parametrize("cap,scale", [(0.7, 0.3), (3.0, 0.0), (1e4, 0.0), (2e6, 0.1), (50.0, 40.0), (1e-3, 1.0),
                                       (1e-29, 1.0), (1e30, 0.0)])
def test_caps(dev, rows, lens, cap, scale):
    """Caps that scores never come near, that all of them are far beyond, and both sides of where the polynomial and
    the exponential share the work."""
    for f32 in (False, True):
        announce(f"paged cap={cap} scale={scale} rows={rows} f32={f32}")
        run_case(ia, dev, np.random.default_rng(3), ia.KV_INT4, 4, 2, 128, rows, lens, cap=cap, scale=scale, out_f32=f32)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("nq,nkv,hd,rows,lens,more", [
    # two tiles by eight waves: 13 to 24 pages, or tiles of like lengths that the CUs hold at once
    (16, 8, 128, [130, 20], [500, 300], {}),
    (4, 2, 128, [99], [757], {"cap": 7.0, "bias": True, "out_f32": True}),
    (32, 32, 128, [250], [1000], {"out_f32": True}),
    (32, 32, 128, [249], [1000], {"prefix": [970], "bias": True}),
    # by four, with splits
    (16, 8, 128, [130], [1000], {}),
    (40, 8, 128, [5] * 6, [900, 30, 400, 2000, 33, 700], {"out_f32": True}),
    (8, 2, 256, [30, 7], [2000, 300], {}),
])
def test_units_of_two_tiles(dev, fmt, nq, nkv, hd, rows, lens, more):
    announce(f"paged units fmt={fmt} {nq}/{nkv}x{hd} rows={rows} {more}")
    run_case(ia, dev, np.random.default_rng(hd), fmt, nq, nkv, hd, rows, lens, **more)


@pytest.mark.parametrize("fmt", FMT)
def test_units_of_two_tiles_masks(dev, fmt):
    pos = np.arange(370, 500)
    rng = np.random.default_rng(fmt)
    for first, prefix in ((np.where(pos % 3 == 0, pos + 1, np.where(pos % 5 == 0, pos // 64 * 64, 0)), None),
                          (np.where(pos % 7 == 0, pos // 100 * 100, 3), [450]),
                          (np.where(pos % 50 == 14, 9, 1 << 30), [500])):
        announce(f"paged units masks fmt={fmt} first={first[:4]} prefix={prefix}")
        run_case(ia, dev, rng, fmt, 16, 8, 128, [130], [500], first=first, prefix=prefix, out_f32=prefix is None)


# Batches with 4096 pages of work and more over their tiles of 128 columns and their kv heads (over fp16 pages 512 tiles
# and more as well): the workgroups that share their pages.
SHARED = [
    (64, 64, 64, [129, 130, 200, 140], [600, 500, 420, 700], {"cap": 12.0, "out_f32": True}),
    (64, 64, 128, [257, 300, 140], [257, 500, 410], {"bias": True}),
    (32, 32, 64, [33, 40, 130, 257], [700, 1000, 1500, 1300], {}),
    (64, 32, 128, [100, 20, 1], [1700, 1500, 60], {"cap": 5.0, "bias": True}),
    (64, 32, 128, [129, 65], [1301, 1665], {"out_f32": True}),
    (32, 16, 64, [300], [2601], {"cap": 0.8, "scale": 1.0, "out_f32": True}),
    (40, 8, 64, [230, 1, 30], [2300, 900, 1000], {"bias": True}),
    (64, 32, 128, [150, 290], [1700, 1600], {"cap": 30.0, "out_f32": True}),
    (32, 4, 64, [530], [2500], {"cap": 30.0}),
    (32, 32, 256, [130, 40], [1500, 1300], {"cap": 30.0}),  # (two-tile units of many columns)
    (32, 32, 256, [150], [2100], {"bias": True, "out_f32": True}),
]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("nq,nkv,hd,rows,lens,more", SHARED)
def test_shared_pages(dev, fmt, nq, nkv, hd, rows, lens, more):
    announce(f"paged shared fmt={fmt} {nq}/{nkv}x{hd} rows={rows} lens={lens} {more}")
    run_case(ia, dev, np.random.default_rng(nq + hd + fmt), fmt, nq, nkv, hd, rows, lens, **more)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("hd", [64, 128])
def test_shared_pages_masks(dev, fmt, hd):
    rows, lens = [270, 250], [500, 600]
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    rng = np.random.default_rng(hd)
    for first, prefix in ((np.where(pos % 3 == 0, pos + 1, np.where(pos % 5 == 0, pos // 64 * 64, 0)), None),
                          (np.where(pos % 7 == 0, pos // 100 * 100, 40), [450, 599]),
                          (np.where(np.arange(len(pos)) % 50 == 14, 9, 1 << 30), lens)):
        announce(f"paged shared masks fmt={fmt} hd={hd} first={first[:4]} prefix={prefix}")
        run_case(ia, dev, rng, fmt, 128, 64, hd, rows, lens, first=first, prefix=prefix, out_f32=hd == 128)


@pytest.mark.parametrize("fmt", FMT)
def test_long_context_is_split(dev, fmt):
    """Splits over a long axis and their join, beside short rows in one batch."""
    announce(f"paged long fmt={fmt}")
    run_case(ia, dev, np.random.default_rng(5), fmt, 4, 2, 64, [1, 1, 40], [9001, 3, 4100], out_f32=True)


def _setup(dev, fmt, nq, nkv, hd, rows, lens, seed=0, edit=None):
    rng = np.random.default_rng(seed)
    n_pages, table, pos = pr.batch(rng, rows, lens)
    cache = pr.Cache(fmt, nkv, hd, n_pages, rng)
    if edit:
        edit(cache, table)
    plan = ia.Paged(dev, fmt, nq, nkv, hd, n_pages)
    q = f16(rng, len(pos), nq, hd)
    return cache, table, plan, q, dev.upload(cache.pool), dev.upload(q), dev.alloc(q.size * 4)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("rows,lens,nkv", [([1, 3], [70, 80], 2), ([100], [150], 2), ([130], [500], 8), ([260, 260], [400, 500], 64)])
def test_values_that_a_row_does_not_see_do_not_reach_it(dev, rows, lens, nkv, value):
    """Infinities and NaN in the K and V of positions that some rows see and others do not: the rows that do not see
    them give what they give without them, the others what the formula gives."""
    fmt, nq, hd = ia.KV_FP16, 2 * nkv, 128
    bad = [(s, lens[s] - rows[s] // 2 - 1, v) for s in range(len(rows)) for v in (0, 1)] + [(0, 5, 1), (0, 6, 0)]

    def edit(cache, table):
        for s, t, v in bad:
            cache.pool[table[s, t // 32], nkv - 1, v].view(np.float16)[pr.element(fmt, hd, v)[t % 32, 3::16]] = value

    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    first = np.full(len(pos), 8)
    announce(f"paged {value} rows={rows}")
    clean = pr.Cache(fmt, nkv, hd, 1, np.random.default_rng(1))
    cache, table, plan, q, pool, qd, out = _setup(dev, fmt, nq, nkv, hd, rows, lens, edit=edit)
    clean.pool = _setup_pool(fmt, nkv, hd, rows, lens)
    plan.set(rows, lens, table, first=first)
    plan.attention(pool.p, qd.p, out.p, out_f32=True)
    got = dev.download(out, np.float32, q.shape).astype(np.float64)
    want, tol = pr.expect(clean, rows, lens, table, q, first, out_f32=True)
    seq = np.repeat(np.arange(len(rows)), rows)
    sees = np.array([[any(s == seq[m] and 8 <= t <= pos[m] and v == w for s, t, v in bad) for w in (0, 1)]
                     for m in range(len(pos))])
    same = ~sees.any(1)
    assert (np.abs(got - want)[same] <= tol[same]).all()
    assert (np.abs(got - want)[:, :-2] <= tol[:, :-2]).all()   # the other kv heads' queries
    hurt = ~np.isfinite(got[:, -2:])
    only_v = sees[:, 1] & ~sees[:, 0]
    dims = np.zeros(hd, bool)
    dims[3::16] = True
    assert hurt[sees[:, 1]][:, :, dims].all() and not hurt[only_v][:, :, ~dims].any()
    if np.isnan(value):
        assert np.isnan(got[sees[:, 0], -2:]).all()
    plan.close()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows,lens,nkv", [([1, 3, 5], [70, 80, 900], 2), ([100], [150], 2), ([130], [500], 8),
                                           ([260, 260], [400, 500], 64)])
def test_queries_that_are_not_finite_stay_in_their_rows(dev, rows, lens, nkv, value):
    for fmt, cap in ((ia.KV_FP16, 0.0), (ia.KV_INT4, 20.0)):
        announce(f"paged query {value} rows={rows} fmt={fmt}")
        nq, hd = 2 * nkv, 128
        cache, table, plan, q, pool, _, out = _setup(dev, fmt, nq, nkv, hd, rows, lens)
        want, tol = pr.expect(cache, rows, lens, table, q, cap=cap, out_f32=True)
        bad = np.zeros(q.shape[:2], bool)
        bad[len(q) // 2, 1] = bad[-1, nq - 1] = True
        q[bad] = value
        qd = dev.upload(q)
        plan.set(rows, lens, table)
        plan.attention(pool.p, qd.p, out.p, out_f32=True, softcap=cap)
        got = dev.download(out, np.float32, q.shape).astype(np.float64)
        assert (np.abs(got - want)[~bad] <= tol[~bad]).all()
        if np.isnan(value):
            assert np.isnan(got[bad]).all()
        plan.close()


@pytest.mark.parametrize("rows,lens,nkv", [([1, 3, 5], [1, 80, 900], 2), ([100], [150], 2), ([130], [500], 8),
                                           ([260, 260], [400, 500], 64)])
def test_scores_of_minus_infinity_only(dev, rows, lens, nkv):
    """The softmax of scores that are all -infinity is not a number; a row that sees nothing still gives zeros."""
    fmt, nq, hd = ia.KV_FP16, 2 * nkv, 128

    def edit(cache, table):
        cache.pool.view(np.uint16)[..., :] &= 0x7FFF  # values of one sign

    announce(f"paged -inf rows={rows}")
    cache, table, plan, q, pool, _, out = _setup(dev, fmt, nq, nkv, hd, rows, lens, edit=edit)
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    first = np.where(np.arange(len(pos)) % 7 == 3, pos + 1, 0)
    bad = np.zeros(q.shape[:2], bool)
    bad[::3, 1] = bad[-1, nq - 1] = True
    want, tol = pr.expect(cache, rows, lens, table, q, first, out_f32=True)
    q[bad] = 0
    q[bad, 5] = -np.inf
    qd = dev.upload(q)
    plan.set(rows, lens, table, first=first)
    plan.attention(pool.p, qd.p, out.p, out_f32=True)
    got = dev.download(out, np.float32, q.shape).astype(np.float64)
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all()
    blind = first > pos
    assert np.isnan(got[bad & ~blind[:, None]]).all() and (got[blind] == 0).all()
    plan.close()


@pytest.mark.parametrize("fmt", [ia.KV_INT8, ia.KV_INT4])
@pytest.mark.parametrize("rows,lens,nkv", [([1, 3], [70, 80], 2), ([100], [150], 2), ([130], [500], 8), ([260, 260], [400, 500], 64)])
def test_quantized_rows_without_a_scale(dev, fmt, rows, lens, nkv):
    """Rows that were stored with a NaN (their scale is NaN) reach only the rows that see them: K the whole head, V its
    group's dims."""
    nq, hd = 2 * nkv, 128
    rng = np.random.default_rng(7)
    n_pages, table, pos = pr.batch(rng, rows, lens)
    M, plan = len(pos), ia.Paged(dev, fmt, nq, nkv, hd, n_pages)
    cache = pr.Cache(fmt, nkv, hd, n_pages, rng)
    pool, q = dev.upload(cache.pool), f16(rng, M, nq, hd)
    k, v = f16(rng, M, nkv, hd), f16(rng, M, nkv, hd)
    bad_k, bad_v = M // 2, M - 1 if M < 5 else 2 * M // 3   # batch rows
    kn, vn = k.copy(), v.copy()
    kn[bad_k, 1, 9] = np.nan
    vn[bad_v, 0, 70] = np.inf
    plan.set(rows, lens, table)
    qd, kd, vd, out = dev.upload(q), dev.upload(kn), dev.upload(vn), dev.alloc(q.size * 4)
    announce(f"paged quantized NaN fmt={fmt} rows={rows}")
    plan.append(pool.p, kd.p, vd.p)
    plan.attention(pool.p, qd.p, out.p, out_f32=True)
    got = dev.download(out, np.float32, q.shape).astype(np.float64)
    seq = np.repeat(np.arange(len(rows)), rows)
    for m in range(M):
        cache.append(table[seq[m]], pos[m], k[m].astype(np.float32), v[m].astype(np.float32))
    want, tol = pr.expect(cache, rows, lens, table, q, out_f32=True)
    sees = lambda b: (seq == seq[b]) & (pos >= pos[b])  # noqa: E731
    hurt = np.zeros(q.shape, bool)
    hurt[sees(bad_k), 2:4] = True
    hurt[sees(bad_v), :2, slice(64, 128) if fmt == ia.KV_INT4 else slice(0, 128)] = True
    assert np.isnan(got[hurt]).all()
    assert (np.abs(got - want)[~hurt] <= tol[~hurt]).all()
    plan.close()


def _setup_pool(fmt, nkv, hd, rows, lens):
    rng = np.random.default_rng(0)
    n_pages, _, _ = pr.batch(rng, rows, lens)
    return pr.Cache(fmt, nkv, hd, n_pages, rng).pool


@pytest.mark.parametrize("fmt", FMT)
def test_append_of_values_without_a_scale(dev, fmt):
    """Rows of zeros, constant rows, the largest and smallest fp16, NaN and infinities: stored by the format's rule."""
    nkv, hd, rng = 2, 128, np.random.default_rng(1)
    rows = f16(rng, 9, nkv, hd)
    rows[0] = 0
    rows[1] = 2.5
    rows[2] = np.where(rng.random(rows[2].shape) < 0.5, 65504, -65504)
    rows[3] = np.float16(6e-8)
    rows[4, 0, 5] = np.nan
    rows[5, 1, 70] = np.inf
    rows[6, 0, 100] = -np.inf
    rows[7] = 100 + rows[7] * 0.01
    cache = pr.Cache(fmt, nkv, hd, 2, fill=0xA5)
    plan = ia.Paged(dev, fmt, 2, nkv, hd, 2)
    plan.set([9], [36], np.array([[1, 0]]))
    pool, kd, vd = dev.upload(cache.pool), dev.upload(rows), dev.upload(rows[::-1].copy())
    ko, vo = dev.alloc(rows.nbytes), dev.alloc(rows.nbytes)
    announce(f"paged append of odd values fmt={fmt}")
    plan.append(pool.p, kd.p, vd.p)
    plan.read(pool.p, ko.p, vo.p)
    for i in range(9):
        pos = 27 + i
        cache.append([1, 0], pos, rows[i].astype(np.float32), rows[8 - i].astype(np.float32))
    got = dev.download(pool, np.uint8, cache.pool.shape)
    if fmt == ia.KV_FP16:  # (which NaN a NaN becomes is nobody's)
        a, b = got.view(np.float16), cache.pool.view(np.float16)
        assert ((a == b) | (np.isnan(a) & np.isnan(b)) | (got.view(np.uint16) == cache.pool.view(np.uint16))).all()
    else:
        assert np.array_equal(got, cache.pool)
    for b, w in ((ko, 0), (vo, 1)):
        x = dev.download(b, np.float16, rows.shape).astype(np.float64)
        assert np.array_equal(x, cache.gather([1, 0], 36)[w][27:], equal_nan=True)
    plan.close()


@pytest.mark.parametrize("fmt", FMT)
def test_slices_of_a_fused_buffer(dev, fmt):
    """Q, K and V as slices of one QKV buffer, Q rotated in place; the output in rows of another width."""
    nq, nkv, hd, rows, lens = 4, 2, 128, [1, 40, 2], [50, 70, 2]
    rng = np.random.default_rng(4)
    n_pages, table, pos = pr.batch(rng, rows, lens)
    M, wide = len(pos), (nq + 2 * nkv) * hd + 24
    qkv = f16(rng, M, wide)
    cos, sin = pr.tables(100, hd)
    cache = pr.Cache(fmt, nkv, hd, n_pages, rng)
    plan = ia.Paged(dev, fmt, nq, nkv, hd, n_pages)
    plan.set(rows, lens, table)
    pool, buf, cd, sd = dev.upload(cache.pool), dev.upload(qkv), dev.upload(cos), dev.upload(sin)
    k0, v0 = nq * hd * 2, (nq + nkv) * hd * 2
    at = lambda o: C.c_void_p(buf.p.value + o)  # noqa: E731
    announce(f"paged fused slices fmt={fmt}")
    plan.append(pool.p, at(k0), at(v0), at(0), at(0), cd.p, sd.p, hd, 100, wide, wide, wide, wide)
    q, k, v = (qkv[:, o:o + n * hd].reshape(M, n, hd) for o, n in ((0, nq), (nq * hd, nkv), ((nq + nkv) * hd, nkv)))
    qr, kr = pr.rotate(q, pos, cos, sin).astype(np.float16), pr.rotate(k, pos, cos, sin)
    seq = np.repeat(np.arange(3), rows)
    for m in range(M):
        cache.append(table[seq[m]], pos[m], kr[m], v[m].astype(np.float32))
    assert np.array_equal(dev.download(pool, np.uint8, cache.pool.shape), cache.pool)
    want = qkv.copy()
    want[:, :nq * hd] = qr.reshape(M, -1)
    assert np.array_equal(dev.download(buf, np.float16, qkv.shape), want)
    ow = nq * hd + 40
    out = dev.upload(np.full((M, ow), 3.25, np.float32))
    plan.attention(pool.p, at(0), out.p, out_f32=True, q_stride=wide, out_stride=ow)
    got = dev.download(out, np.float32, (M, ow))
    ref, tol = pr.expect(cache, rows, lens, table, qr, out_f32=True)
    assert (got[:, nq * hd:] == 3.25).all()
    assert (np.abs(got[:, :nq * hd].reshape(ref.shape) - ref) <= tol).all()
    plan.close()


def test_pages_shared_for_reading(dev):
    """Two sequences over one prefix's pages, each with its own last page."""
    fmt, nq, nkv, hd = ia.KV_INT4, 4, 2, 128
    rng = np.random.default_rng(2)
    cache = pr.Cache(fmt, nkv, hd, 6, rng)
    table, rows, lens = np.array([[4, 2, 0], [4, 2, 5]], np.int32), [1, 3], [70, 80]
    plan = ia.Paged(dev, fmt, nq, nkv, hd, 6)
    plan.set(rows, lens, table)
    q, k, v = f16(rng, 4, nq, hd), f16(rng, 4, nkv, hd), f16(rng, 4, nkv, hd)
    pool, qd, kd, vd, out = dev.upload(cache.pool), dev.upload(q), dev.upload(k), dev.upload(v), dev.alloc(q.nbytes)
    announce("paged shared prefix")
    plan.append(pool.p, kd.p, vd.p)
    plan.attention(pool.p, qd.p, out.p)
    for m, (s, p) in enumerate(((0, 69), (1, 77), (1, 78), (1, 79))):
        cache.append(table[s], p, k[m].astype(np.float32), v[m].astype(np.float32))
    want, tol = pr.expect(cache, rows, lens, table, q)
    assert (np.abs(dev.download(out, np.float16, q.shape) - want) <= tol).all()
    plan.close()


def test_a_row_has_the_same_bits_again(dev):
    """No sum's order depends on timing: the same batch twice, between other batches of the same plan."""
    fmt, nq, nkv, hd = ia.KV_INT4, 8, 2, 128
    rows, lens = [1, 1, 60, 5], [5000, 40, 200, 900]
    cache, table, plan, q, pool, qd, out = _setup(dev, fmt, nq, nkv, hd, rows, lens)
    res = []
    announce("paged: the same batch again")
    for i in range(4):
        plan.set(rows, lens, table)
        plan.attention(pool.p, qd.p, out.p, out_f32=True)
        res.append(dev.download(out, np.float32, q.shape))
        plan.set([3, 1], [77, 500], table[:2])  # a smaller batch in the same buffers
        plan.attention(pool.p, qd.p, out.p, out_f32=True)
    assert all(np.array_equal(r.view(np.uint32), res[0].view(np.uint32)) for r in res)
    plan.close()


def test_batches_set_while_the_one_before_runs(dev):
    """ifr_paged_set does not disturb calls that are queued: eight batches of growing size without a wait."""
    fmt, nq, nkv, hd = ia.KV_INT8, 4, 2, 64
    rng = np.random.default_rng(8)
    cache = pr.Cache(fmt, nkv, hd, 400, rng)
    plan = ia.Paged(dev, fmt, nq, nkv, hd, 400)
    pool, jobs = dev.upload(cache.pool), []
    announce("paged: batches set one after the other")
    for i in range(8):
        rows, lens = [1] * (i + 1) + [3 + 9 * i], [200 * (j + 1) for j in range(i + 1)] + [40 + 50 * i]
        table = rng.integers(0, 400, (len(rows), 60)).astype(np.int32)
        q = f16(rng, sum(rows), nq, hd)
        qd, out = dev.upload(q), dev.alloc(q.nbytes * 2)
        plan.set(rows, lens, table)
        plan.attention(pool.p, qd.p, out.p, out_f32=True)
        jobs.append((rows, lens, table, q, out))
    for rows, lens, table, q, out in jobs:
        want, tol = pr.expect(cache, rows, lens, table, q, out_f32=True)
        assert (np.abs(dev.download(out, np.float32, q.shape) - want) <= tol).all()
    plan.close()


@pytest.mark.parametrize("fmt", FMT)
def test_pool_offsets_past_32_bits(dev, fmt):
    """Pages behind the first 4 GiB of a pool."""
    nq, nkv, hd, rows, lens = 8, 4, 128, [2, 40], [100, 40]
    n_pages = (5 << 30) // (2 * nkv * pr.part_bytes(fmt, hd))
    rng = np.random.default_rng(6)
    cache = pr.Cache(fmt, nkv, hd, 6, rng)
    plan = ia.Paged(dev, fmt, nq, nkv, hd, n_pages)
    assert plan.pool_bytes() > 1 << 32
    small = np.array([[0, 1, 2, 3], [4, 5, 0, 0]], np.int32)
    table = n_pages - 6 + small
    pool, page = dev.alloc(plan.pool_bytes()), cache.pool[0].nbytes
    ia.check(ia.lib().ifr_h2d(dev.ctx, C.c_void_p(pool.p.value + (n_pages - 6) * page),
                              cache.pool.ctypes.data_as(C.c_void_p), cache.pool.nbytes), "ifr_h2d")
    q, k, v = f16(rng, 42, nq, hd), f16(rng, 42, nkv, hd), f16(rng, 42, nkv, hd)
    qd, kd, vd, out = dev.upload(q), dev.upload(k), dev.upload(v), dev.alloc(q.nbytes)
    plan.set(rows, lens, table)
    announce(f"paged far pages fmt={fmt}")
    plan.append(pool.p, kd.p, vd.p)
    plan.attention(pool.p, qd.p, out.p)
    for m in range(42):
        s, p = (0, 98 + m) if m < 2 else (1, m - 2)
        cache.append(small[s], p, k[m].astype(np.float32), v[m].astype(np.float32))
    want, tol = pr.expect(cache, rows, lens, small, q)
    assert (np.abs(dev.download(out, np.float16, q.shape) - want) <= tol).all()
    plan.close()
    pool.free()


def test_captured_calls_replay(dev):
    """Append and attention captured into a graph, replayed between eager calls of another plan; the captured plan
    refuses another batch, and a batch cannot be set inside a capture."""
    hip = C.CDLL("libamdhip64.so")
    st = C.c_void_p(dev.stream())
    fmt, nq, nkv, hd, rows, lens = ia.KV_INT4, 4, 2, 128, [1, 1, 50], [700, 33, 90]
    rng = np.random.default_rng(3)
    cache, table, plan, q, pool, qd, out = _setup(dev, fmt, nq, nkv, hd, rows, lens)
    k, v = f16(rng, 52, nkv, hd), f16(rng, 52, nkv, hd)
    kd, vd = dev.upload(k), dev.upload(v)
    other = _setup(dev, ia.KV_FP16, nq, nkv, hd, [5, 1], [400, 90], seed=1)
    plan.set(rows, lens, table)
    other[2].set([5, 1], [400, 90], other[1])
    announce("paged: capture and replay")
    plan.append(pool.p, kd.p, vd.p)
    plan.attention(pool.p, qd.p, out.p, out_f32=True)
    eager = dev.download(out, np.float32, q.shape)
    graph, ex = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(st, 2) == 0  # relaxed
    try:
        with pytest.raises(ia.IfrError) as e:
            plan.set(rows, lens, table)
        assert e.value.code == ia._abi.IFR_ESTATE
        plan.append(pool.p, kd.p, vd.p)
        plan.attention(pool.p, qd.p, out.p, out_f32=True)
    finally:
        assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    with pytest.raises(ia.IfrError) as e:
        plan.set(rows, lens, table)
    assert e.value.code == ia._abi.IFR_ESTATE
    for i in range(4):
        ia.check(ia.lib().ifr_memset(dev.ctx, out.p, 0, q.size * 4), "ifr_memset")
        other[2].attention(other[4].p, other[5].p, other[6].p)
        assert hip.hipGraphLaunch(ex, st) == 0
        other[2].attention(other[4].p, other[5].p, other[6].p)
        got = dev.download(out, np.float32, q.shape)
        assert np.array_equal(got.view(np.uint32), eager.view(np.uint32)), i
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    plan.close()
    other[2].close()


def test_two_contexts_at_once():
    """Two contexts, a thread each, with plans of their own."""
    devs, errors = [ia.Device(0), ia.Device(0)], []
    jobs = []
    for i, d in enumerate(devs):
        rows, lens = [1, 20 + i, 1], [900, 100, 40 + 300 * i]
        cache, table, plan, q, pool, qd, out = _setup(d, FMT[2 - i], 4, 2, 128, rows, lens, seed=i)
        plan.set(rows, lens, table)
        jobs.append((d, plan, pool, qd, out, q, pr.expect(cache, rows, lens, table, q)))

    def run(d, plan, pool, qd, out, q, ref):
        for _ in range(10):
            plan.attention(pool.p, qd.p, out.p)
            if not (np.abs(d.download(out, np.float16, q.shape) - ref[0]) <= ref[1]).all():
                errors.append(d)

    announce("paged: two contexts, two threads")
    th = [threading.Thread(target=run, args=j) for j in jobs]
    for t in th:
        t.start()
    for t in th:
        t.join()
    for j in jobs:
        j[1].close()
    for d in devs:
        d.close()
    assert not errors


def test_a_layer_step(dev):
    """The calls of one layer together: rotated append, attention in fp32, and the quantizer that the O projection
    takes its rows from."""
    fmt, nq, nkv, hd, rows, lens = ia.KV_INT4, 8, 4, 128, [1, 1, 30], [400, 65, 93]
    rng = np.random.default_rng(12)
    cache, table, plan, q, pool, qd, out = _setup(dev, fmt, nq, nkv, hd, rows, lens)
    M = len(q)
    k, v = f16(rng, M, nkv, hd), f16(rng, M, nkv, hd)
    cos, sin = pr.tables(512, hd)
    kd, vd, cd, sd = dev.upload(k), dev.upload(v), dev.upload(cos), dev.upload(sin)
    codes, sc = dev.alloc((M + 15) // 16 * 16 * nq * hd), dev.alloc(M * 4)
    plan.set(rows, lens, table)
    announce("paged: a layer's step")
    plan.append(pool.p, kd.p, vd.p, qd.p, qd.p, cd.p, sd.p, hd, 512)
    plan.attention(pool.p, qd.p, out.p, out_f32=True)
    ia.check(ia.lib().ifr_act_quant(dev.ctx, out.p, M, nq * hd, None, 0.0, 0, 0, 0, codes.p, sc.p, None), "ifr_act_quant")
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
    kr, qr = pr.rotate(k, pos, cos, sin), pr.rotate(q, pos, cos, sin).astype(np.float16)
    seq = np.repeat(np.arange(3), rows)
    for m in range(M):
        cache.append(table[seq[m]], pos[m], kr[m], v[m].astype(np.float32))
    want, tol = pr.expect(cache, rows, lens, table, qr, out_f32=True)
    got = ia.untile(dev.download(codes, np.int8, ((M + 15) // 16 * 16 * nq * hd,)), M, nq * hd)
    s = dev.download(sc, np.float32, (M,)).astype(np.float64)
    # a code is off by half a step and by the attention's own bound; its scale's bound follows the largest value
    off = np.abs(got * s[:, None] - want.reshape(M, -1))
    assert (off <= 0.5001 * s[:, None] + 2 * tol.reshape(M, -1).max(1, keepdims=True)).all()
    plan.close()


def test_refusals(dev):
    announce("paged refusals")
    refusals(ia, dev)
