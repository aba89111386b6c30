"""GPU: the operators over 8-bit pages and shared beginnings under bounds that scale with what each row sees, and at the inputs where their roundings go wrong first.

Tolerances of attention (`close_attention`): what is rounded to fp16 in front of the second product are the weights w_j = 2^(s_j - m) v_scale_j (fp16 pages: v_scale = 1), m at most the largest
s_j + log2(v_scale_j) of the positions that the row sees; a rounding is off by 2^-11 of the weight, and by 2^-25 among fp16's smallest numbers, that is 2^-25 of the row's largest contribution."""
import numpy as np
import pytest

from spy_b200 import backend as B
from test_gpu_paged import Device, Pool, be, dev  # noqa: F401
from test_gpu_paged_more import TYPES, BytePool, attend, plain_norm, scale_above

pytestmark = pytest.mark.gpu


def close_attention(q, kb, vb, sk, sv, first, scale, causal, window, there):
    """q [rows][heads][e]; kb, vb [positions][kv heads][e] and their scales [positions][kv heads], f64. The output, and how far the kernels may be from it (without the output's own rounding)."""
    rows, h, hd = q.shape
    n, h_kv, _ = kb.shape
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    per = scale / np.log(2)
    for g in range(h_kv):
        heads = np.arange(g * (h // h_kv), (g + 1) * (h // h_kv))
        s_all = np.einsum("rhe,ne->rhn", q[:, heads], kb[:, g]) * (sk[:, g] * per)
        a_all = np.einsum("rhe,ne->rhn", np.abs(q[:, heads]), np.abs(kb[:, g])) * np.abs(sk[:, g] * per)
        for i in range(rows):
            j = np.arange(n)
            seen = there.copy()
            if causal:
                seen &= j <= first + i
                if window:
                    seen &= j > first + i - window
            if not seen.any():
                continue
            v, v_scale = vb[seen, g], np.abs(sv[seen, g])
            for x, head in enumerate(heads):
                s, a = s_all[i, x, seen], a_all[i, x, seen]
                p = np.exp2(s - s.max())
                w = p * v_scale
                top = (p * np.maximum(v_scale, 2.0 ** -24)).max()
                # an exponent: head_dim exact products summed in f32 (a truncation each: 2^-23 of the sum of magnitudes), by a scale that is rounded three times, beside a maximum that is moved up a few times
                d = np.log(2) * (hd * 2.0 ** -23 * a + 8 * 2.0 ** -24 * (np.abs(s) + np.abs(s).max() + 40))
                # weights to fp16; powers of two and joins; f32 sums, 16 terms a step
                rel = 2.0 ** -11 + 2.0 ** -20 + (len(s) / 16 + 60) * 2.0 ** -23
                out[i, head] = (p * sv[seen, g]) @ v / p.sum()
                off[i, head] = ((rel + d) * w) @ np.abs(v) + 2.0 ** -25 * top * np.abs(v).sum(0) + np.abs(out[i, head]) * (d @ p + rel * p.sum())
                off[i, head] /= p.sum()
    return out, off


def held(pool, s, n):
    """What pages hold of a sequence: whole numbers (or values) and scales of K and V, and which positions are there."""
    pos = np.arange(n)
    pages = pool.table[s, pos // pool.page]
    there = (pages >= 0) & (pages < pool.n_pages)
    at = (np.where(there, pages, 0), pos % pool.page)
    k, v = (np.where(there[:, None, None], pool.view(x)[at], 0).astype(np.float64) for x in (pool.k, pool.v))
    if not isinstance(pool, BytePool):
        return k, v, np.ones(k.shape[:2]), np.ones(k.shape[:2]), there
    sc = np.where(there[:, None, None], pool.scale_view()[at], 0).astype(np.float64)
    return k, v, sc[..., 0], sc[..., 1], there


def check_close(got, pool, starts, rows, q, scale=None, causal=True, window=0, room=None, show=None):
    """All rows of all sequences; `room`: the largest share of a typical output that the bound may be, so that it says something."""
    hd = q.shape[2]
    for s, n in enumerate(pool.n_kv):
        a, b = starts[s], starts[s + 1]
        if b == a:
            continue
        want, off = close_attention(q[a:b].astype(np.float64), *held(pool, s, n)[:4], n - rows[s], hd ** -0.5 if scale is None else scale, causal, window, held(pool, s, n)[4])
        if room is not None:
            assert np.median(off) <= room * np.sqrt((want ** 2).mean()), (float(np.median(off)), float(np.sqrt((want ** 2).mean())))
        tol = off + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if got.dtype == np.float16 else np.abs(want) * 2.0 ** -24)
        err = np.abs(got[a:b].astype(np.float64) - want)
        assert (err <= tol).all(), (s, float((err / np.maximum(tol, 1e-300)).max()), np.unravel_index(np.argmax(err / np.maximum(tol, 1e-300)), err.shape))


def make_pool(rng, n_kv, h_kv, hd, page, eight=True, sizes=0.5, token_major=False, groups=None):
    pool = BytePool(rng, n_kv, h_kv, hd, page, token_major) if eight else Pool(rng, n_kv, h_kv, hd, page, token_major)
    x = [rng.standard_normal((2, n, h_kv, hd)) * np.exp(sizes * rng.standard_normal((2, n, h_kv, 1))) for n in n_kv]
    for g, n in enumerate(groups[1] if groups else []):
        a, b = groups[0][g], groups[0][g + 1]
        longest = max(range(a, b), key=lambda i: n_kv[i])
        for i in range(a, b):
            m = min(n, n_kv[i])
            x[i][:, :m] = x[longest][:, :m]
            pool.table[i, :m // page] = pool.table[longest, :m // page]
    for s in range(len(n_kv)):
        pool.put(s, *(x[s].astype(np.float16)))
    return pool


# ---------------------------------------------------------------------------------------------- V's scales
@pytest.mark.parametrize("rows", [1, 2, 6, 100])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("large", [32.0, 515.5, 65504.0])
def test_a_position_of_no_weight_and_a_large_scale_takes_nothing_from_the_others(be, dev, rows, hd, large):
    """4000 positions of scale 0.03 and, at the start, in the middle and near the end, one whose score is some 40 below theirs and whose V is thousands of times larger."""
    rng = np.random.default_rng(rows + hd)
    n, h, h_kv = 4000, 4, 2
    pool = make_pool(rng, [n], h_kv, hd, 16, sizes=0.1)
    q = (1 + 0.1 * rng.standard_normal((rows, h, hd))).astype(np.float16)
    at = lambda j: (pool.table[0, j // 16], j % 16)  # noqa: E731
    pool.scale_view()[(pool.table[0, np.arange(n) // 16], np.arange(n) % 16)] = (0.03 / 16, 0.03)
    for j in (3, 2222, n - rows - 5):
        pool.view(pool.k)[at(j)] = -100
        pool.scale_view()[at(j)] = (40 / 100 * hd ** -0.5, large)
    got = attend(be, dev, pool, [0, rows], q, np.zeros(q.shape, dtype=np.float32))
    check_close(got, pool, [0, rows], [rows], q, room=0.15)


@pytest.mark.parametrize("rows", [2, 6, 100])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_scales_of_positions_that_a_row_does_not_see_take_nothing_from_it(be, dev, rows, hd):
    """The last row's position has K and V of any scale: the rows in front of it are as near as without it, and in the kernel for few rows, where a row's maximum is its own alone, the same bits."""
    rng = np.random.default_rng(rows + hd)
    n, h, h_kv = 500 + rows, 6, 2
    pool = make_pool(rng, [n], h_kv, hd, 16)
    q, out0, last = rng.standard_normal((rows, h, hd)).astype(np.float16), np.zeros((rows, h, hd), dtype=np.float32), (pool.table[0, (n - 1) // 16], (n - 1) % 16)
    got = []
    for pair in ((1e-3, 1e-3), (5.0, 515.5), (65504.0, 65504.0), (0.0, 2.0 ** -24)):
        pool.scale_view()[last] = pair
        got.append(attend(be, dev, pool, [0, rows], q, out0)[:rows - 1])
        pool.scale_view()[last] = 1
        front = pool.n_kv
        pool.n_kv = [n - 1]
        check_close(got[-1], pool, [0, rows - 1], [rows - 1], q[:rows - 1], room=0.05)
        pool.n_kv = front
    assert rows == 100 or all(np.array_equal(got[0].view(np.uint32), x.view(np.uint32)) for x in got[1:])


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_that_are_zero_negative_or_the_smallest(be, dev, rows, hd):
    rng = np.random.default_rng(rows * hd)
    n, h, h_kv = 600, 4, 2
    for kind in range(4):
        pool = make_pool(rng, [n], h_kv, hd, 16)
        where = (pool.table[0, np.arange(n) // 16], np.arange(n) % 16, slice(None), 1)
        v = pool.scale_view()[where].copy()
        pool.scale_view()[where] = (0 * v, np.where(rng.random(v.shape) < 0.5, -v, v), 0 * v + 2.0 ** -24, np.where(rng.random(v.shape) < 0.5, 0, v))[kind]
        q = (2 * rng.standard_normal((rows, h, hd))).astype(np.float16)
        check_close(attend(be, dev, pool, [0, rows], q, np.zeros(q.shape, dtype=np.float32)), pool, [0, rows], [rows], q)


# ---------------------------------------------------------------------------------------------- long contexts, scores and scales of all sizes
@pytest.mark.parametrize("rows,n_kv,h,h_kv,hd,page", [([1], [40000], 2, 1, 64, 64), ([1], [30011], 4, 2, 128, 24), ([3], [30000], 4, 1, 128, 16), ([40], [9000], 2, 1, 128, 64), ([33], [12000], 3, 1, 64, 16),
                                                      ([5, 1], [20000, 700], 4, 2, 96, 16), ([1, 6], [9000, 12001], 4, 4, 32, 32)])
@pytest.mark.parametrize("spread,sizes", [(0.05, 0.2), (1.0, 0.5), (1.0, 2.0)])
def test_cut_items_of_all_scores_and_scales(be, dev, rows, n_kv, h, h_kv, hd, page, spread, sizes):
    """Items that many CTAs share, whose pieces have maxima and scales of their own."""
    rng = np.random.default_rng(n_kv[0] + hd)
    pool = make_pool(rng, n_kv, h_kv, hd, page, sizes=sizes)
    starts = np.concatenate([[0], np.cumsum(rows)])
    q = (spread * rng.standard_normal((starts[-1], h, hd))).astype(np.float16)
    check_close(attend(be, dev, pool, starts, q, np.zeros(q.shape, dtype=np.float32)), pool, starts, rows, q, room=0.3)


@pytest.mark.parametrize("rows", [1, 4, 33, 300])
@pytest.mark.parametrize("hd", [64, 128])
def test_sharp_rows_and_scales_of_all_sizes_by_what_each_row_sees(be, dev, rows, hd):
    rng = np.random.default_rng(rows)
    for spread, sizes in ((2.0, 0.2), (0.05, 2.5)):
        pool = make_pool(rng, [900, rows], 2, hd, 16, sizes=sizes)
        q = (spread * rng.standard_normal((2 * rows, 8, hd))).astype(np.float16)
        check_close(attend(be, dev, pool, [0, rows, 2 * rows], q, np.zeros(q.shape, dtype=np.float32)), pool, [0, rows, 2 * rows], [rows, rows], q, room=0.3)


# ---------------------------------------------------------------------------------------------- shared beginnings
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("shared", [128, 290, 299, 300, 500, 100000])
@pytest.mark.parametrize("rows", [1, 2, 12])
def test_what_is_shared_is_cut_to_what_all_rows_see(be, dev, eight, shared, rows):
    """The shortest sequence of three has 300 positions in front of its rows: of more than that only these are shared, whatever the caller says."""
    rng = np.random.default_rng(shared + rows)
    for hd, page, causal in ((64, 16, True), (128, 24, True), (96, 16, True), (128, 32, False)):
        n_kv, starts = [900 + rows, 300 + rows, 640 + rows], [0, rows, 2 * rows, 3 * rows]
        pool = make_pool(rng, n_kv, 2, hd, page, eight, groups=([0, 3], [min(shared, 900)]))
        q = rng.standard_normal((3 * rows, 4, hd)).astype(np.float16)
        got = attend(be, dev, pool, starts, q, np.zeros(q.shape, dtype=np.float32), ([0, 3], [shared]), causal=causal)
        check_close(got, pool, starts, [rows] * 3, q, causal=causal, room=0.05)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_groups_of_any_order_give_what_no_groups_give(be, dev, eight, hd):
    """Rows enough for the kernel on tensor memory in the first pass, sequences whose first 304 positions are all the same, and groups that are not ascending, overlap or leave the batch: whatever is
    made of them, what a row sees does not change, and nothing outside the described buffers is touched."""
    rng = np.random.default_rng(hd)
    n_seq, rows, h, h_kv, common = 6, 9, 4, 2, 304
    n_kv = [common + rows + 50 * i for i in range(n_seq)]
    pool = make_pool(rng, n_kv, h_kv, hd, 16, eight, groups=([0, n_seq], [common]))
    starts = np.arange(n_seq + 1) * rows
    q = rng.standard_normal((n_seq * rows, h, hd)).astype(np.float16)
    size = B.paged_attend_workspace(n_seq, n_seq * rows, h, hd)
    margin = np.full((3 * n_seq * rows, h, hd), 3.0, dtype=np.float32)
    po = dev(margin)
    b = B.paged_batch(dev(starts.astype(np.int32)), dev(np.array(n_kv, np.int32)), dev(pool.table), n_seq, n_seq * rows, pool.table.shape[1])
    a = B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), b, dev(q), po + n_seq * rows * h * hd * 4, h, out_type=B.FP32)
    sc = pool.of_scales(dev(pool.scales)) if eight else None
    kinds = [[2, 0, 6], [0, 2, 1, 6], [0, 4, 2, 6], [5, 1, 3], [-7, 3, 2, 90], [6, 5, 4, 3, 2, 1, 0], [0, 0, 6, 6], [1, 6, 0, 4, 2, 9], [0, 1 << 30], [0, 6]] + [rng.integers(-2, 9, 5).tolist() for _ in range(12)]
    for start in kinds:
        for fill in (0x33, 0xff, 0x7f):
            room = dev(np.full(size + 64, fill, np.uint8))
            be.paged_attend(B.paged_attend_desc(a, sc, group_start=dev(np.array(start, np.int64).astype(np.int32)), n_shared=dev(np.full(len(start) - 1, common, np.int32)), n_group=len(start) - 1, workspace=room,
                                                workspace_bytes=size))
            got = dev.back(po, margin)
            assert (got[:n_seq * rows] == 3).all() and (got[2 * n_seq * rows:] == 3).all()
            assert (dev.back(room, np.zeros(size + 64, np.uint8))[size:] == fill).all()
            check_close(got[n_seq * rows:2 * n_seq * rows], pool, starts, [rows] * n_seq, q, room=0.05)


@pytest.mark.parametrize("eight", [False, True])
def test_groups_over_rows_that_make_no_sense_touch_nothing_else(be, dev, eight):
    """Rows' beginnings that are not ascending, negative or behind the last row, under one group: answered inside the described buffers."""
    rng = np.random.default_rng(3)
    n_seq, n_rows, h, hd, common = 5, 60, 4, 64, 304
    n_kv = [common + 60] * n_seq
    pool = make_pool(rng, n_kv, 2, hd, 16, eight, groups=([0, n_seq], [common]))
    q = rng.standard_normal((n_rows, h, hd)).astype(np.float16)
    size = B.paged_attend_workspace(n_seq, n_rows, h, hd)
    margin = np.full((3 * n_rows, h, hd), 3.0, dtype=np.float32)
    po, c, pq, pn, pt = dev(margin), pool.cache(dev(pool.k), dev(pool.v)), dev(q), dev(np.array(n_kv, np.int32)), dev(pool.table)
    sc = pool.of_scales(dev(pool.scales)) if eight else None
    for start in ([0, 20, 10, 40, 30, 60], [50, 40, 30, 20, 10, 0], [-9, 5, 70, 20, 65, 1 << 20], [0, 60, 0, 60, 0, 60], [10, 30, 5, 50, 2, 40], [0, 30, 12, 13, 14, 20]):
        room = dev(np.full(size + 64, 0x33, np.uint8))
        a = B.paged_attention_desc(c, B.paged_batch(dev(np.array(start, np.int32)), pn, pt, n_seq, n_rows, pool.table.shape[1]), pq, po + n_rows * h * hd * 4, h, out_type=B.FP32)
        be.paged_attend(B.paged_attend_desc(a, sc, group_start=dev(np.array([0, n_seq], np.int32)), n_shared=dev(np.array([common], np.int32)), n_group=1, workspace=room, workspace_bytes=size))
        got = dev.back(po, margin)
        assert (got[:n_rows] == 3).all() and (got[2 * n_rows:] == 3).all()
        assert (dev.back(room, np.zeros(size + 64, np.uint8))[size:] == 0x33).all()


# ---------------------------------------------------------------------------------------------- store
def store_values(be, dev, values, dtype=np.float32, **norms):
    """K and V (the same values, [rows][head_dim]) into 8-bit pages, without rotation: bytes and scales of V, of K."""
    n, hd = values.shape
    pool = BytePool(np.random.default_rng(0), [n], 1, hd, 16)
    pk, pv, ps, px = dev(pool.k), dev(pool.v), dev(pool.scales), dev(values.astype(dtype))
    batch = B.paged_batch(dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), dev(pool.table), 1, n, pool.table.shape[1])
    be.paged_store(B.paged_store_desc(B.paged_append_desc(pool.cache(pk, pv), batch, None, px, px, None, 0, in_type=TYPES[dtype], rope_mode=B.ROPE_NONE), pool.of_scales(ps), **norms))
    at = (pool.table[0, np.arange(n) // 16], np.arange(n) % 16)
    k, v, sc = dev.back(pk, pool.k), dev.back(pv, pool.v), pool.scale_view(dev.back(ps, pool.scales))[at][:, 0]
    return (pool.view(v)[at][:, 0], sc[:, 1]), (pool.view(k)[at][:, 0], sc[:, 0])


def nearest_even(x, scale):
    """x / scale to the nearest whole number, a half to the even one, without an error on the way: twice the quotient is compared as whole numbers of 2^-200."""
    from fractions import Fraction
    got = np.zeros(x.shape, np.int64)
    for i, row in enumerate(x):
        unit = Fraction(float(scale[i]))
        got[i] = [round(Fraction(float(e)) / unit) if unit else 0 for e in row]      # (Python rounds a half to the even one)
    return got


@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_are_the_nearest_and_a_half_goes_to_the_even_one(be, dev, hd):
    """Elements that are k + 1/2 scales to the last bit, or a bit beside it, for scales of all mantissas: K and V the same bytes, which are the nearest."""
    rng = np.random.default_rng(hd)
    n = 700
    scale = (1 + rng.integers(0, 1024, n) / 1024) * 2.0 ** rng.integers(-14, 8, n)                    # (of 11 bits, as fp16's)
    k = rng.integers(-126, 126, (n, hd))
    x = (scale[:, None] * (k + 0.5)).astype(np.float32)                                               # exact: 11 bits by 8
    beside = rng.integers(0, 3, (n, hd))
    x = np.where(beside == 0, x, np.nextafter(x, np.where(beside == 1, np.float32(np.inf), np.float32(-np.inf)))).astype(np.float32)
    x[:, 5] = (127 * scale).astype(np.float32)                                                        # exact: the largest magnitude
    for bytes_, got in store_values(be, dev, x):
        assert np.array_equal(got.astype(np.float64), scale)
        assert np.array_equal(bytes_.astype(np.int64), nearest_even(x, scale))


def test_a_scale_is_not_below_its_largest_magnitude_by_127(be, dev):
    """Largest magnitudes a bit above 127 fp16 numbers: their quotients lie between f32 numbers beside these."""
    rng = np.random.default_rng(11)
    n, hd = 900, 64
    h = (1 + rng.integers(0, 1024, n) / 1024) * 2.0 ** rng.integers(-14, 8, n)
    most = np.nextafter((127 * h).astype(np.float32), np.float32(np.inf))
    x = (rng.uniform(-1, 1, (n, hd)) * most[:, None]).astype(np.float32)
    x[np.arange(n), rng.integers(0, hd, n)] = most
    want = scale_above(most.astype(np.float64) / 127)
    assert (want > h).all()
    for bytes_, got in store_values(be, dev, x):
        assert np.array_equal(got, want)
        assert np.array_equal(bytes_.astype(np.int64), nearest_even(x, got.astype(np.float64)))


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("size", [1e18, 1e10, 1e-5, 1e-15])
@pytest.mark.parametrize("hd", [24, 128, 256])
def test_norms_of_very_large_and_very_small_heads(be, dev, eps, size, hd):
    """Squares at either end of f32."""
    rng = np.random.default_rng(hd)
    n, h = 9, 3
    x = (size * rng.uniform(-1, 1, (n, h, hd))).astype(np.float32)
    x[:, 1] = rng.standard_normal((n, hd))                                                            # (an ordinary head beside them)
    w = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    one = (hd + 15) // 16 * 16
    pool = Pool(rng, [n], 1, hd, 16, strides=(16 * one, one, 16 * one), fill=0)
    px, pq, q0 = dev(x), None, np.zeros((n, h, hd), np.float32)
    pq = dev(q0)
    batch = B.paged_batch(dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), dev(pool.table), 1, n, pool.table.shape[1])
    zeros = dev(np.zeros((n, hd), np.float32))
    append = B.paged_append_desc(pool.cache(dev(pool.k), dev(pool.v)), batch, px, zeros, zeros, pq, h, q_out_type=B.FP32, rope_mode=B.ROPE_NONE)
    be.paged_store(B.paged_store_desc(append, q_norm=dev(w), norm_eps=eps))
    want = plain_norm(x.astype(np.float64), w.astype(np.float64), np.float64(np.float32(eps)))
    err = np.abs(dev.back(pq, q0).astype(np.float64) - want)
    # a sum of head_dim squares (half its relative error), a reciprocal square root of 2 steps, two products, each a bit among the smallest numbers
    assert (err <= np.abs(want) * ((hd + 2) / 2 + 4 + 2) * 2.0 ** -24 + 3 * 2.0 ** -149).all(), float((err / np.maximum(np.abs(want), 1e-300)).max())
