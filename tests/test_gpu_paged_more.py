"""GPU: storing with norms and in bytes, reading back, attention over 8-bit pages and over shared beginnings, against plain numpy in 64 bits.

Tolerances: a rounding is off by half a step at most, relative 2^-11 for fp16 (2^-25 absolutely among its smallest values) and 2^-24 for f32; an element of an 8-bit head is off by half the head's
scale. What follows from these is derived where it is used."""
import numpy as np
import pytest

from spy_b200 import backend as B
from test_gpu_paged import Device, Pool, be, dev, plain_attention, plain_rope, rope_off  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = {np.float32: B.FP32, np.float16: B.FP16}


def scale_above(x):
    """The smallest fp16 that is not below x (f64, not negative)."""
    h = x.astype(np.float16)
    return np.where(h.astype(np.float64) < x, np.nextafter(h, np.float16(np.inf)), h)


class BytePool(Pool):
    """Pages of bytes: free places hold 127 and a NaN scale. `scale_strides`: (page, position, head), in pairs."""

    def __init__(self, rng, n_kv, heads, head_dim, page, token_major=False, strides=None, scale_strides=None, spare=2):
        super().__init__(rng, n_kv, heads, head_dim, page, token_major, strides, spare, fill=0)
        self.k, self.v = (np.full(self.size, 127, dtype=np.int8) for _ in range(2))
        self.ss = scale_strides or ((page * heads, heads, 1) if token_major else (page * heads, 1, page))
        self.scales = np.full(2 * (self.n_pages * self.ss[0] + page * self.ss[1] + heads * self.ss[2] + 1), np.nan, dtype=np.float16)

    def view(self, a):
        return np.lib.stride_tricks.as_strided(a, (self.n_pages, self.page, self.heads, self.hd), self.strides + (1,))

    def scale_view(self, a=None):
        return np.lib.stride_tricks.as_strided(self.scales if a is None else a, (self.n_pages, self.page, self.heads, 2), tuple(4 * s for s in self.ss) + (2,))

    def put(self, s, k, v):
        """Floats, as bytes; returns the values that are kept."""
        pos = np.arange(len(k))
        at, kept = (self.table[s, pos // self.page], pos % self.page), []
        for i, (a, x) in enumerate(((self.k, k), (self.v, v))):
            scale = scale_above(np.abs(x.astype(np.float64)).max(-1, initial=0) / 127)
            step = np.where(scale > 0, scale, 1).astype(np.float64)[..., None]
            b = np.rint(x / step)
            self.view(a)[at] = b
            self.scale_view()[at + (slice(None), i)] = scale
            kept.append(b * scale.astype(np.float64)[..., None])
        return kept

    def values(self, s, n, k=None, v=None, scales=None):
        pos = np.arange(n)
        pages = self.table[s, pos // self.page]
        there = (pages >= 0) & (pages < self.n_pages)
        at = (np.where(there, pages, 0), pos % self.page)
        sc = self.scale_view(scales)[at].astype(np.float64)
        return [self.view(a)[at].astype(np.float64) * sc[..., i:i + 1] for i, a in enumerate((self.k if k is None else k, self.v if v is None else v))], there, np.abs(sc)

    def cache(self, pk, pv):
        return B.paged_cache(pk, pv, self.n_pages, self.page, self.heads, self.hd, strides=self.strides, number_type=B.INT8)

    def of_scales(self, p):
        return B.paged_scales(p, self.page, self.heads, strides=self.ss)


# ---------------------------------------------------------------------------------------------- store
def plain_norm(x, weight, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight


def check_store(be, dev, rng, rows, n_kv, h, h_kv, hd, page, eight, mode=B.ROPE_HALVES, rot=None, base=1e6, dtype=np.float32, q_type=np.float16, token_major=False, pad=0, in_place=False, drop=0,
                norms="qk", eps=1e-6, size=1.0, strides=None, scale_strides=None):
    rot = hd if rot is None else rot
    pool = BytePool(rng, n_kv, h_kv, hd, page, token_major, strides, scale_strides) if eight else Pool(rng, n_kv, h_kv, hd, page, token_major, fill=0.25)
    if drop:
        pool.table[rng.random(pool.table.shape) < drop] = -1
        pool.table[rng.random(pool.table.shape) < drop / 2] = pool.n_pages
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n_rows, width = int(starts[-1]) + pad, (h + 2 * h_kv) * hd + 8
    x = (size * rng.standard_normal((n_rows, width)) * np.exp(rng.standard_normal((n_rows, 1)))).astype(dtype)
    weights = (1 + 0.3 * rng.standard_normal((2, hd))).astype(np.float32)
    px, pk, pv = dev(x), dev(pool.k), dev(pool.v)
    ps = dev(pool.scales) if eight else None
    q0 = np.full((n_rows, h, hd), -9, dtype=q_type)
    pq = px if in_place else dev(q0)
    e = x.itemsize * hd
    a = B.paged_append_desc(pool.cache(pk, pv), B.paged_batch(dev(starts), dev(np.array(n_kv, dtype=np.int32)), dev(pool.table), len(rows), n_rows, pool.table.shape[1]),
                            px if h else None, px + h * e, px + (h + h_kv) * e, pq if h else None, h, in_type=TYPES[dtype], q_out_type=TYPES[q_type], row_stride=width,
                            q_out_stride=width if in_place else None, rope_mode=mode, rope_dim=rot, freq_base=base)
    be.paged_store(B.paged_store_desc(a, pool.of_scales(ps) if eight else None, q_norm=dev(weights[0]) if "q" in norms and h else None, k_norm=dev(weights[1]) if "k" in norms else None, norm_eps=eps))
    got_k, got_v = dev.back(pk, pool.k), dev.back(pv, pool.v)
    got_s = dev.back(ps, pool.scales) if eight else None
    got_q = dev.back(px, x)[:, :h * hd].reshape(n_rows, h, hd) if in_place else dev.back(pq, q0)
    want_k, want_v, want_s = pool.k.copy(), pool.v.copy(), pool.scales.copy() if eight else None
    untouched = np.ones((n_rows,), dtype=bool)
    half = lambda a: np.abs(a) * 2.0 ** -11 + 2.0 ** -25  # noqa: E731
    for s, n in enumerate(n_kv):
        a, b = starts[s], starts[s + 1]
        pos = np.arange(n - rows[s], n)
        full = x[a:b, :(h + 2 * h_kv) * hd].reshape(b - a, h + 2 * h_kv, hd).astype(np.float64)
        off = np.zeros(full.shape)
        for lo, hi, name, w in ((0, h, "q", weights[0]), (h, h + h_kv, "k", weights[1])):
            if name in norms:
                full[:, lo:hi] = plain_norm(full[:, lo:hi], w.astype(np.float64), np.float64(np.float32(eps)))
                # a sum of head_dim squares and eps (half its relative error), a reciprocal square root of 2 steps, two products
                off[:, lo:hi] = np.abs(full[:, lo:hi]) * ((hd + 2) / 2 + 4 + 2) * 2.0 ** -24
        if mode == B.ROPE_NONE:
            turned = full
        else:
            turned, spread = plain_rope(full, pos, mode, rot, base, 1.0), rope_off(full, mode, rot)
            i = np.arange(rot // 2)
            u, w = (2 * i, 2 * i + 1) if mode == B.ROPE_PAIRS else (i, i + rot // 2)
            off[..., u] = off[..., w] = off[..., u] + off[..., w]
            off += spread
        ok = pos >= 0
        untouched[a:b] = ~ok
        if h:
            err = np.abs(got_q[a:b][ok].astype(np.float64) - turned[ok, :h])
            tol = off[ok, :h] + (half(turned[ok, :h]) if q_type == np.float16 else np.abs(turned[ok, :h]) * 2.0 ** -24)
            assert (err <= tol).all(), float((err / tol).max())
        pages = pool.table[s, pos[ok] // page] if ok.any() else np.zeros(0, dtype=int)
        there = (pages >= 0) & (pages < pool.n_pages)
        at = (pages[there], pos[ok][there] % page)
        for i, (got, want, lo, exact) in enumerate(((got_k, want_k, h, False), (got_v, want_v, h + h_kv, True))):
            value = (x[a:b, :(h + 2 * h_kv) * hd].reshape(b - a, h + 2 * h_kv, hd).astype(np.float64) if exact else turned)[ok][there][:, lo:lo + h_kv]
            slack = 0 * value if exact else off[ok][there][:, lo:lo + h_kv]
            kept = pool.view(got)[at].astype(np.float64)
            if eight:
                scale = pool.scale_view(got_s)[at][..., i].astype(np.float64)
                most, more = np.abs(value).max(-1, initial=0), slack.max(-1, initial=0)
                # the largest magnitude / 127, rounded in f32, and up to fp16
                lo_most, hi_most = (np.maximum(most - more, 0) / 127 * (1 - 2.0 ** -23), (most + more) / 127 * (1 + 2.0 ** -23))
                assert (scale >= scale_above(lo_most)).all() and (scale <= scale_above(hi_most)).all()
                # half a scale, and what a product with 1 / scale in f32 is off: 2^-23 of up to 127.5 scales
                assert (np.abs(kept * scale[..., None] - value) <= slack + scale[..., None] * (0.5 + 128 * 2.0 ** -23)).all()
                assert (np.abs(kept) <= 127).all()
                pool.scale_view(want_s)[at + (slice(None), i)] = pool.scale_view(got_s)[at + (slice(None), i)]
            else:
                assert (np.abs(kept - value) <= half(value) + slack).all()
            pool.view(want)[at] = pool.view(got)[at]
    assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)         # nothing else was stored
    assert got_s is None or np.array_equal(got_s.view(np.uint16), want_s.view(np.uint16))
    untouched[starts[-1]:] = True
    if h:
        before = x[:, :h * hd].reshape(n_rows, h, hd) if in_place else q0
        assert np.array_equal(got_q[untouched], before[untouched])


@pytest.mark.parametrize("mode", [B.ROPE_NONE, B.ROPE_PAIRS, B.ROPE_HALVES])
@pytest.mark.parametrize("hd,rot", [(32, 16), (64, 64), (96, 48), (128, 128), (256, 256)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_store(be, dev, mode, hd, rot, eight, dtype):
    rng = np.random.default_rng(hd + rot)
    check_store(be, dev, rng, [1, 20, 0, 3], [400, 20, 7, 100001], 6, 2, hd, 16, eight, mode=mode, rot=rot, dtype=dtype, pad=2)
    check_store(be, dev, rng, [1], [33], 3, 3, hd, 5, eight, mode=mode, rot=rot, dtype=dtype, q_type=np.float32, token_major=True, base=500000.0, eps=1e-3)


@pytest.mark.parametrize("norms", ["", "q", "k"])
@pytest.mark.parametrize("eight", [False, True])
def test_store_with_some_norms(be, dev, norms, eight):
    rng = np.random.default_rng(21)
    check_store(be, dev, rng, [9, 2], [40, 2], 5, 5, 64, 16, eight, norms=norms, mode=B.ROPE_PAIRS)
    check_store(be, dev, rng, [9, 2], [40, 2], 0, 2, 128, 16, eight, norms=norms)


@pytest.mark.parametrize("eight", [False, True])
def test_store_in_place_with_missing_pages_small_and_large_values(be, dev, eight):
    rng = np.random.default_rng(22)
    check_store(be, dev, rng, [5, 2], [50, 2], 4, 2, 64, 16, eight, q_type=np.float32, in_place=True)
    check_store(be, dev, rng, [5, 2], [50, 2], 4, 2, 64, 16, eight, mode=B.ROPE_PAIRS, dtype=np.float16, in_place=True)
    check_store(be, dev, rng, [40, 30], [300, 30], 4, 2, 64, 8, eight, drop=0.5)
    check_store(be, dev, rng, [6, 1], [4, 0], 4, 2, 64, 8, eight)                          # rows with negative positions
    check_store(be, dev, rng, [30], [30], 4, 2, 64, 8, eight, size=1e-4)                   # (eps counts)
    check_store(be, dev, rng, [30], [30], 4, 2, 64, 8, eight, size=500.0)


def test_store_many_sequences_and_other_strides(be, dev):
    rng = np.random.default_rng(23)
    rows = rng.integers(0, 4, 1500).tolist()
    check_store(be, dev, rng, rows, [r + int(x) for r, x in zip(rows, rng.integers(0, 30, 1500))], 2, 1, 64, 16, True, pad=5)
    check_store(be, dev, rng, [7, 50], [100, 50], 4, 2, 64, 16, True, strides=(16 * 2 * 96 + 48, 80 + 80, 80), scale_strides=(16 * 7 + 3, 7, 3))


@pytest.mark.parametrize("hd", [24, 40, 96, 200])
@pytest.mark.parametrize("eight", [False, True])
def test_store_heads_that_fill_no_power_of_two_in_several_rows_of_a_block(be, dev, hd, eight):
    rng = np.random.default_rng(hd)
    one = (hd + 15) // 16 * 16                                                              # (strides of bytes are multiples of 16)
    strides = lambda n: (16 * n * one, n * one, one) if eight else None  # noqa: E731
    check_store(be, dev, rng, [1300, 0, 1], [1350, 0, 9], 5, 2, hd, 16, eight, mode=B.ROPE_PAIRS, strides=strides(2))
    check_store(be, dev, rng, [900], [900], 30, 12, hd, 16, eight, mode=B.ROPE_HALVES, strides=strides(12))      # (several turns of heads, the last one of few)


def test_store_heads_of_all_kinds(be, dev):
    """Zeros, one value, the smallest numbers, the largest that bytes take and the next, infinities and NaN; what is read back, and what is kept."""
    hd = 64
    rows = np.zeros((11, hd), dtype=np.float32)
    rows[1] = -3.5
    rows[2, 5] = 1e-30
    rows[3, :] = 2.0 ** -24
    rows[4, 7] = 65468.0
    rows[5, 7] = np.nextafter(np.float32(65468.0), np.float32(1e9))
    rows[6, 1], rows[6, 2] = 1.0, np.inf
    rows[7, 1], rows[7, 2] = 1.0, -np.inf
    rows[8, 1], rows[8, 63] = 1.0, np.nan
    rows[9] = np.linspace(-127, 127, hd)
    rows[10] = 12345.678 * np.linspace(-1, 1, hd)
    n = len(rows)
    pool = BytePool(np.random.default_rng(0), [n], 1, hd, 4)
    pk, pv, ps, px = dev(pool.k), dev(pool.v), dev(pool.scales), dev(rows)
    batch = B.paged_batch(dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), dev(pool.table), 1, n, pool.table.shape[1])
    append = B.paged_append_desc(pool.cache(pk, pv), batch, None, px, px, None, 0, rope_mode=B.ROPE_NONE)
    be.paged_store(B.paged_store_desc(append, pool.of_scales(ps)))
    k, v, scales = dev.back(pk, pool.k), dev.back(pv, pool.v), dev.back(ps, pool.scales)
    (got_k, got_v), _, _ = pool.values(0, n, k, v, scales)
    sc = pool.scale_view(scales)[pool.table[0, np.arange(n) // 4], np.arange(n) % 4, 0]
    assert np.array_equal(sc[:, 0], sc[:, 1], equal_nan=True)
    for i in range(n):
        assert np.array_equal(got_k[i], got_v[i], equal_nan=True)
        if i in (5, 6, 7, 8):
            assert np.isnan(sc[i, 0]) and np.isnan(got_k[i]).all()
            continue
        assert sc[i, 0] == scale_above(np.float64(np.float32(np.abs(rows[i]).max() / np.float32(127))))
        assert (np.abs(got_k[i, 0] - rows[i]) <= np.float64(sc[i, 0]) * (0.5 + 2.0 ** -16)).all()
    assert sc[0, 0] == 0 and sc[2, 0] == 2.0 ** -24 and sc[4, 0] == 515.5
    for dtype in (np.float32, np.float16):
        out0 = np.full((n, 1, hd), -7, dtype=dtype)
        po, pw = dev(out0), dev(out0)
        be.paged_load(B.paged_load_desc(pool.cache(pk, pv), batch, po, pw, pool.of_scales(ps), out_type=TYPES[dtype]))
        for p in (po, pw):
            assert np.array_equal(dev.back(p, out0), got_k.astype(np.float32).astype(dtype), equal_nan=True)


# ---------------------------------------------------------------------------------------------- load
@pytest.mark.parametrize("hd", [8, 64, 96, 128, 256])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("out", [np.float16, np.float32])
def test_load(be, dev, hd, heads, eight, out):
    """Whole sequences, ends of some, none of one; pages that are not there, rows in front of the first position, rows of nobody, rows with room between them."""
    rng = np.random.default_rng(hd + heads)
    rows, n_kv, page = [70, 3, 0, 1, 5], [70, 40, 9, 1, 3], 8
    wide = hd if hd % 16 == 0 else 16
    strides = (page * heads * wide, wide, page * wide)
    pool = BytePool(rng, n_kv, heads, hd, page, strides=strides) if eight else Pool(rng, n_kv, heads, hd, page, strides=strides)
    for s, n in enumerate(n_kv):
        pool.put(s, *rng.standard_normal((2, n, heads, hd)).astype(np.float16))
    pool.table[0, 3], pool.table[1, 4] = -1, pool.n_pages
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n_rows, stride = int(starts[-1]) + 3, heads * hd + 8
    out0 = np.full((n_rows, stride), 3, dtype=out)
    c = pool.cache(dev(pool.k), dev(pool.v))
    b = B.paged_batch(dev(starts), dev(np.array(n_kv, np.int32)), dev(pool.table), len(rows), n_rows, pool.table.shape[1])
    sc = pool.of_scales(dev(pool.scales)) if eight else None
    for which in ("kv", "k", "v"):
        pk, pv = dev(out0), dev(out0)
        be.paged_load(B.paged_load_desc(c, b, pk if "k" in which else None, pv if "v" in which else None, sc, out_type=TYPES[out], k_stride=stride, v_stride=stride))
        for i, p in enumerate((pk, pv)):
            want = out0.copy()
            for s, n in enumerate(n_kv):
                if "kv"[i] not in which:
                    continue
                if eight:
                    (values, there, _) = pool.values(s, n)
                    x = np.where(there[:, None, None], values[i], 0)
                else:
                    there = (pool.table[s, np.arange(n) // page] >= 0) & (pool.table[s, np.arange(n) // page] < pool.n_pages)
                    safe = np.where(there, pool.table[s, np.arange(n) // page], 0)
                    x = np.where(there[:, None, None], pool.view((pool.k, pool.v)[i])[safe, np.arange(n) % page], 0).astype(np.float64)
                first = n - rows[s]
                x = np.concatenate([np.zeros((max(0, -first),) + x.shape[1:]), x[max(0, first):]])
                want[starts[s]:starts[s + 1], :heads * hd] = x.reshape(rows[s], heads * hd).astype(np.float32).astype(out)
            assert np.array_equal(dev.back(p, out0), want)


def test_load_more_rows_than_a_grid_has_at_once(be, dev):
    """20 000 positions in pages by token, other pages beside them; a copy through f32 gives the same as through fp16 (bytes x scales are no fp16 numbers: rounded once)."""
    rng = np.random.default_rng(5)
    n, heads, hd = 20000, 2, 64
    pool = BytePool(rng, [n, 50], heads, hd, 24, token_major=True)
    pool.put(0, *rng.standard_normal((2, n, heads, hd)))
    pool.put(1, *rng.standard_normal((2, 50, heads, hd)))
    b = B.paged_batch(dev(np.array([0, n, n + 2], np.int32)), dev(np.array([n, 50], np.int32)), dev(pool.table), 2, n + 2, pool.table.shape[1])
    c, sc = pool.cache(dev(pool.k), dev(pool.v)), pool.of_scales(dev(pool.scales))
    want = [np.concatenate([pool.values(0, n)[0][i], pool.values(1, 50)[0][i][48:]]).astype(np.float32) for i in range(2)]
    for out in (np.float32, np.float16):
        out0 = np.zeros((n + 2, heads, hd), dtype=out)
        pk, pv = dev(out0), dev(out0)
        be.paged_load(B.paged_load_desc(c, b, pk, pv, sc, out_type=TYPES[out]))
        assert np.array_equal(dev.back(pk, out0), want[0].astype(out)) and np.array_equal(dev.back(pv, out0), want[1].astype(out))


# ---------------------------------------------------------------------------------------------- attend
def attend(be, dev, pool, starts, q, out0, groups=None, max_rows=0, **kw):
    """groups: (group_start, n_shared). The same bits twice."""
    n_rows, h, hd = q.shape
    eight = isinstance(pool, BytePool)
    starts = np.asarray(starts, dtype=np.int32)
    b = B.paged_batch(dev(starts), dev(np.array(pool.n_kv, dtype=np.int32)), dev(pool.table), len(pool.n_kv), n_rows, pool.table.shape[1], max_rows)
    po = dev(out0)
    a = B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), b, dev(q), po, h, out_type=TYPES[out0.dtype.type], **kw)
    more = {}
    if groups is not None:
        size = B.paged_attend_workspace(len(pool.n_kv), n_rows, h, hd)
        more = dict(group_start=dev(np.asarray(groups[0], np.int32)), n_shared=dev(np.asarray(groups[1], np.int32)), n_group=len(groups[1]), workspace=dev(np.full(size, 0xff, np.uint8)), workspace_bytes=size)
    d = B.paged_attend_desc(a, pool.of_scales(dev(pool.scales)) if eight else None, **more)
    be.paged_attend(d)
    got = dev.back(po, out0)
    be.paged_attend(d)
    assert np.array_equal(got.view(np.uint8), dev.back(po, out0).view(np.uint8))
    return got


def check_rows(got, q, k, v, first, scale, causal, window, there, scales, out):
    """One sequence's rows. `scales`: of its positions, None for fp16."""
    want, off = plain_attention(q, k, v, first, scale, causal, window, there)
    h_kv = k.shape[1]
    if scales is not None:
        # a probability times its scale is held against the largest scale rounded up: 2^-25 of twice 127 of these among fp16's smallest
        for x in range(q.shape[1]):
            g = x // (q.shape[1] // h_kv)
            if there.any():
                off[:, x] += there.sum() * 2.0 ** -24 * 127 * scales[there][:, g, 1].max()
    tol = off + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if out == np.float16 else np.abs(want) * 2.0 ** -24)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (float((err / np.maximum(tol, 1e-30)).max()), np.unravel_index(np.argmax(err - tol), err.shape))
    assert (got[~np.any(want != 0, axis=2)] == 0).all()


def check_attend(be, dev, rng, rows, n_kv, h, h_kv, hd, page, eight=True, causal=True, window=0, scale=0.0, out=np.float16, token_major=False, pad=0, spread=1.0, max_rows=0, drop=None, strides=None,
                 scale_strides=None, groups=None, by_value=False, sizes=0.5, q_pad=0):
    """groups: (group_start, n_shared); what is shared lies in the same pages, or (by_value) in pages of its own with the same values."""
    pool = BytePool(rng, n_kv, h_kv, hd, page, token_major, strides, scale_strides) if eight else Pool(rng, n_kv, h_kv, hd, page, token_major, strides)
    starts = np.concatenate([[0], np.cumsum(rows)])
    x = [rng.standard_normal((2, max(0, n), h_kv, hd)) * np.exp(sizes * rng.standard_normal((2, max(0, n), h_kv, 1))) for n in n_kv]
    for g, n in enumerate(groups[1] if groups else []):
        a, b = groups[0][g], min(groups[0][g + 1], len(n_kv))
        longest = max(range(a, b), key=lambda i: n_kv[i]) if b > a else a
        for i in range(a, b):
            m = min(n, max(0, n_kv[i]))
            x[i][:, :m] = x[longest][:, :m]
            if not by_value and i != longest:
                pool.table[i, :m // page] = pool.table[longest, :m // page]
    for s in range(len(n_kv)):
        pool.put(s, *(x[s].astype(np.float16)))
    if drop is not None:
        for s in range(len(n_kv)):                                    # (what is shared is missing for all)
            gone = rng.random(pool.table.shape[1]) < drop
            common = max([n for g, n in enumerate(groups[1]) if groups[0][g] <= s < groups[0][g + 1]] + [0]) // page + 1 if groups else 0
            gone[:common] = (np.arange(common) % 3 == 1)[:len(gone)] if common else gone[:common]
            pool.table[s, gone] = [-1, pool.n_pages + 5][s % 2]
    q = (spread * rng.standard_normal((starts[-1] + pad, h, hd))).astype(np.float16)
    out0 = np.full(q.shape, 7.5, dtype=out)
    got = attend(be, dev, pool, starts, q, out0, groups, max_rows, causal=causal, window=window, scale=scale)
    for s, n in enumerate(n_kv):
        n = max(0, n)
        if eight:
            (k, v), there, sc = pool.values(s, n)
            k, v = (np.where(there[:, None, None], a, 0) for a in (k, v))
        else:
            pages = pool.table[s, np.arange(n) // page]
            there, sc = (pages >= 0) & (pages < pool.n_pages), None
            safe = np.where(there, pages, 0)
            k, v = (np.where(there[:, None, None], pool.view(a)[safe, np.arange(n) % page], 0).astype(np.float64) for a in (pool.k, pool.v))
        a, b = starts[s], starts[s + 1]
        if b > a:
            check_rows(got[a:b], q[a:b].astype(np.float64), k, v, n - rows[s] if n_kv[s] >= 0 else -rows[s], scale or hd ** -0.5, causal, window, there, sc, out)
    assert (got[starts[-1]:] == 7.5).all()                   # rows behind the last sequence


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("h,h_kv", [(4, 4), (6, 2), (5, 1), (8, 1), (20, 1)])
def test_bytes_single_tokens(be, dev, hd, h, h_kv):
    rng = np.random.default_rng(hd * 100 + h * 10 + h_kv)
    check_attend(be, dev, rng, [1] * 7, [1, 2, 15, 16, 17, 300, 1031], h, h_kv, hd, 16, pad=2, max_rows=1)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 200, 256])
@pytest.mark.parametrize("token_major", [False, True])
def test_bytes_pages_of_all_sizes(be, dev, page, token_major):
    rng = np.random.default_rng(page)
    check_attend(be, dev, rng, [1, 3, 40, 0, 1], [77, 130, 290, 55, 1], 4, 2, 64, page, token_major=token_major)
    check_attend(be, dev, rng, [140, 2], [333, 64], 4, 1, 128, page, token_major=token_major)


@pytest.mark.parametrize("rows,n_kv", [([1], [0]), ([0], [5]), ([3], [2]), ([5, 1, 0, 2], [5, 0, 9, 1]), ([130], [130]), ([129], [500]), ([257], [260]), ([64, 1, 64], [64, 700, 200])])
@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_short_and_empty(be, dev, rows, n_kv, hd):
    rng = np.random.default_rng(len(rows) + rows[0])
    check_attend(be, dev, rng, rows, n_kv, 4, 2, hd, 16, pad=3)


@pytest.mark.parametrize("window", [1, 17, 128, 129, 1000])
@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_windows(be, dev, window, rows, hd):
    rng = np.random.default_rng(window)
    check_attend(be, dev, rng, [rows, 1, rows], [700, 90, rows], 6, 2, hd, 16, window=window)
    for page in (32, 64, 192):                               # (a window that begins in the middle of a page)
        check_attend(be, dev, rng, [1, 2, 1, 1], [700, 590, 333, 64], 6, 2, hd, page, window=window)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("rows", [1, 9, 200])
def test_bytes_without_causal_order_and_with_other_scales(be, dev, hd, rows):
    rng = np.random.default_rng(hd + rows)
    check_attend(be, dev, rng, [rows, rows], [310, 40], 4, 2, hd, 32, causal=False, scale=0.3)
    check_attend(be, dev, rng, [rows], [310], 4, 4, hd, 32, scale=-0.1, out=np.float32)


@pytest.mark.parametrize("rows", [1, 4, 33, 300])
@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_sharp_rows_and_scales_of_all_sizes(be, dev, rows, hd):
    """Scales over five orders of magnitude; f32 outputs."""
    rng = np.random.default_rng(rows)
    check_attend(be, dev, rng, [rows, rows], [900, rows], 8, 2, hd, 16, out=np.float32, spread=2.0, sizes=0.2)
    check_attend(be, dev, rng, [rows, rows], [900, rows], 8, 2, hd, 16, out=np.float32, spread=0.05, sizes=2.5)


@pytest.mark.parametrize("rows", [1, 6, 160])
@pytest.mark.parametrize("hd", [64, 128])
def test_bytes_pages_that_are_not_there(be, dev, rows, hd):
    rng = np.random.default_rng(rows * hd)
    for drop in (0.3, 0.9, 1.0):
        check_attend(be, dev, rng, [rows, rows, 1], [400, 170, 333], 4, 2, hd, 16, drop=drop)


@pytest.mark.parametrize("rows", [2, 30, 200])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_bytes_scales_that_are_not_finite_reach_only_who_sees_them(be, dev, rows, hd, value):
    """A scale of a later position, of one outside the window, behind the sequence's end or in a free page has no influence."""
    rng = np.random.default_rng(rows + hd)
    n, h, h_kv, window = 230 + rows, 4, 2, 90
    pool = BytePool(rng, [n], h_kv, hd, 16)
    pool.scales[:] = value
    k, v = pool.put(0, *rng.standard_normal((2, n, h_kv, hd)))
    bad_v, bad_k, old = n - rows + rows // 2, n - 1, n - rows - window - 3       # seen by the rows behind it in its window, by the last one, by nobody
    at = lambda j: (pool.table[0, j // 16], j % 16)  # noqa: E731
    pool.scale_view()[at(bad_v) + (0, 1)] = value
    pool.scale_view()[at(bad_k) + (1, 0)] = value
    pool.scale_view()[at(old)] = value
    q = rng.standard_normal((rows, h, hd)).astype(np.float16)
    got = attend(be, dev, pool, [0, rows], q, np.zeros(q.shape, dtype=np.float32), window=window)
    first = n - rows
    sees_v = np.arange(first, n) >= bad_v
    sees_v &= np.arange(first, n) < bad_v + window
    sees_k = np.arange(first, n) >= bad_k
    v[bad_v, 0] = 0
    k[bad_k, 1] = 0
    ok = np.ones((rows, h), dtype=bool)
    ok[sees_v, :2] = False
    ok[sees_k, 2:] = False
    want, off = plain_attention(q.astype(np.float64), k, v, first, hd ** -0.5, True, window, np.ones(n, dtype=bool))
    err = np.abs(got - want)
    assert np.isfinite(got[ok]).all()
    assert (err[ok] <= (off + n * 2.0 ** -24 * 2 * np.abs(v).max() + np.abs(want) * 2.0 ** -24)[ok]).all()
    assert not np.isfinite(got[sees_v][:, :2]).all(axis=2).any() and not np.isfinite(got[sees_k][:, 2:]).all(axis=2).any()


@pytest.mark.parametrize("rows", [1, 2, 6, 100])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_bytes_the_largest_scale_in_front_of_the_window_has_no_influence(be, dev, rows, hd):
    rng = np.random.default_rng(rows + hd)
    n, h, h_kv, window = 230 + rows, 4, 2, 90
    pool = BytePool(rng, [n], h_kv, hd, 16)
    k, v = pool.put(0, *rng.standard_normal((2, n, h_kv, hd)))
    q = rng.standard_normal((rows, h, hd)).astype(np.float16)
    out0 = np.zeros(q.shape, dtype=np.float32)
    before = attend(be, dev, pool, [0, rows], q, out0, window=window)
    for j in range(n - rows - window + 1):
        pool.scale_view()[pool.table[0, j // 16], j % 16] = 65504
    assert np.array_equal(before, attend(be, dev, pool, [0, rows], q, out0, window=window))


def test_bytes_whole_chip_on_one_head_and_cut_items(be, dev):
    rng = np.random.default_rng(5)
    check_attend(be, dev, rng, [1], [40000], 2, 1, 64, 64, max_rows=1)
    check_attend(be, dev, rng, [3], [30000], 4, 1, 128, 16)
    check_attend(be, dev, rng, [40], [9000], 2, 1, 128, 64)


def test_bytes_other_strides(be, dev):
    rng = np.random.default_rng(7)
    check_attend(be, dev, rng, [1, 50], [200, 150], 4, 2, 64, 16, strides=(16 * 2 * 96 + 48, 80 + 80, 80), scale_strides=(16 * 7 + 3, 7, 3))


def test_bytes_many_sequences(be, dev):
    rng = np.random.default_rng(6)
    n = 700
    rows = rng.integers(0, 3, n).tolist()
    check_attend(be, dev, rng, rows, [int(x) for x in rng.integers(0, 60, n)], 2, 1, 32, 16)
    check_attend(be, dev, rng, rows, [int(x) for x in rng.integers(0, 60, n)], 24, 1, 64, 16)


# ---------------------------------------------------------------------------------------------- shared beginnings
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("h,h_kv,rows", [(4, 4, 1), (8, 2, 1), (6, 2, 3), (5, 1, 40)])
def test_shared(be, dev, eight, hd, h, h_kv, rows):
    """Groups of all kinds: three sequences, one with a single sequence, one whose beginning is too short to share, sequences in no group in front of, between and behind them."""
    rng = np.random.default_rng(hd + h + rows)
    n_kv = [300, 900 + rows, 700 + rows, 768 + rows, 50 + rows, 500 + rows, 450 + rows, 77 + rows, 1000 + rows, 640]
    check_attend(be, dev, rng, [rows] * 9 + [1], n_kv, h, h_kv, hd, 16, eight, groups=([1, 4, 5, 7, 9], [700, 40, 130, 60]), pad=3)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 127, 128, 129, 500, 100000])
def test_shared_more_than_all_see(be, dev, eight, shared):
    """What is shared is cut to what all rows of the group see: 260 positions, or with rows in front of the first position none."""
    rng = np.random.default_rng(shared)
    n_kv = [400, 263, 1000]
    check_attend(be, dev, rng, [1, 3, 2], n_kv, 4, 2, 64, 16, eight, groups=([0, 3], [min(shared, 260) if shared <= 500 else 260]), out=np.float32)
    pool_kv = [300, 300, 300]
    check_attend(be, dev, rng, [2, 300, 1], pool_kv, 4, 2, 64, 16, eight, groups=([0, 3], [shared if shared < 300 else 300]))


@pytest.mark.parametrize("eight", [False, True])
def test_shared_values_in_other_pages_and_odd_ones(be, dev, eight):
    rng = np.random.default_rng(31)
    check_attend(be, dev, rng, [1, 2, 1, 1], [600, 700, 520, 512], 4, 2, 128, 24, eight, groups=([0, 2, 4], [515, 510]), by_value=True, token_major=True)
    check_attend(be, dev, rng, [1, 2, 1, 1], [600, 700, 520, 512], 4, 2, 64, 7, eight, groups=([0, 4], [505]))
    check_attend(be, dev, rng, [5, 2, 1, 9], [600, 700, 520, 530], 10, 2, 64, 32, eight, groups=([0, 4], [505]), causal=False, scale=0.2, out=np.float32)
    check_attend(be, dev, rng, [5, 2, 1, 9], [600, 700, 520, 530], 10, 2, 64, 32, eight, groups=([0, 4], [505]), window=100)
    check_attend(be, dev, rng, [5, 2, 1, 9], [600, 700, 520, 530], 10, 2, 128, 16, eight, groups=([0, 4], [505]), drop=0.3)


@pytest.mark.parametrize("eight", [False, True])
def test_shared_without_rows(be, dev, eight):
    """Groups whose first sequence has no rows, whose sequences have none, and with nothing that is the sequence's own."""
    rng = np.random.default_rng(32)
    check_attend(be, dev, rng, [0, 1, 1, 0, 0, 3, 1], [0, 400, 300, 20, 30, 300, 257], 8, 2, 128, 16, eight, groups=([0, 3, 5, 7], [290, 16, 256]))
    check_attend(be, dev, rng, [1, 1], [257, 257], 2, 2, 64, 16, eight, groups=([0, 2], [256]))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_shared_large_groups(be, dev, eight, hd):
    rng = np.random.default_rng(33)
    check_attend(be, dev, rng, [1] * 90, [1500 + 7 * i for i in range(90)], 8, 2, hd, 16, eight, groups=([0, 90], [1500]), max_rows=1)
    check_attend(be, dev, rng, [2] * 40, [800 + 7 * i for i in range(40)], 24, 1, hd, 64, eight, groups=([0, 20, 40], [790, 650]))


def test_shared_groups_that_make_no_sense_touch_nothing_else(be, dev):
    """Negative groups, groups behind the last sequence, not ascending: answered inside the described buffers (margins around them stay), and the sequences that they leave alone are right."""
    rng = np.random.default_rng(34)
    n_kv, h, hd = [300, 300, 300, 40], 4, 64
    pool = Pool(rng, n_kv, 2, hd, 16)
    for s, n in enumerate(n_kv):
        pool.put(s, *rng.standard_normal((2, n, 2, hd)).astype(np.float16))
    q = rng.standard_normal((4, h, hd)).astype(np.float16)
    margin = np.full((4 + 4 + 4, h, hd), 3.0, dtype=np.float16)
    po = dev(margin)
    size = B.paged_attend_workspace(4, 4, h, hd)
    room = dev(np.full(size + 64, 0x33, np.uint8))
    b = B.paged_batch(dev(np.arange(5, dtype=np.int32)), dev(np.array(n_kv, dtype=np.int32)), dev(pool.table), 4, 4, pool.table.shape[1])
    a = B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), b, dev(q), po + 4 * h * hd * 2, h)
    for start, shared in (([-7, 2, 90], [1 << 30, -5]), ([3, 1, 0], [256, 256]), ([5, 9, 2], [256, 1 << 30]), ([-(1 << 31), (1 << 31) - 1], [(1 << 31) - 1])):
        be.paged_attend(B.paged_attend_desc(a, None, group_start=dev(np.array(start, np.int64).astype(np.int32)), n_shared=dev(np.array(shared, np.int64).astype(np.int32)), n_group=len(shared), workspace=room,
                                            workspace_bytes=size))
        got = dev.back(po, margin)
        assert (got[:4] == 3).all() and (got[8:] == 3).all()
        assert (dev.back(room, np.zeros(size + 64, np.uint8))[size:] == 0x33).all()
        if start[0] in (3, 5):                                        # (no sequence is in any group)
            for s, n in enumerate(n_kv):
                k, v = (pool.get(x, s).astype(np.float64) for x in (pool.k, pool.v))
                check_rows(got[4 + s:5 + s], q[s:s + 1].astype(np.float64), k, v, n - 1, hd ** -0.5, True, 0, np.ones(n, dtype=bool), None, np.float16)


def test_nothing_to_do(be, dev):
    c = B.paged_cache(dev(np.zeros(4096, np.int8)), dev(np.zeros(4096, np.int8)), 2, 16, 1, 64, number_type=B.INT8)
    z = dev(np.zeros(64, np.float32))
    sc = B.paged_scales(z, 16, 1)
    for n_seq, n_rows in ((0, 3), (2, 0)):
        b = B.paged_batch(z, z, z, n_seq, n_rows, 1)
        be.paged_attend(B.paged_attend_desc(B.paged_attention_desc(c, b, z, z, 1), sc, z, z, 1, z, 1 << 20))
        be.paged_store(B.paged_store_desc(B.paged_append_desc(c, b, z, z, z, z, 1), sc, z, z))
        be.paged_load(B.paged_load_desc(c, b, z, z, sc))
    be.sync()


# ---------------------------------------------------------------------------------------------- every position, by counting
def check_counts(be, dev, rng, rows, n_kv, h, h_kv, hd, page, eight=True, causal=True, window=0, max_rows=0, groups=None, out=np.float32, q_pad=0, out_pad=0):
    """All keys 0: a row's output is the mean of the values that it sees. Values are small whole numbers (bytes of scale 1), so that every sum on the way (below 2^24, or half of that) is exact and the
    output is one quotient, rounded to f32 twice (2^-23 of it): a position that is left out, seen twice, by both passes or by none, or another head's shows."""
    n_kv = [max(r, n) for r, n in zip(rows, n_kv)]
    pool = BytePool(rng, n_kv, h_kv, hd, page) if eight else Pool(rng, n_kv, h_kv, hd, page, fill=0.0)
    values = [rng.integers(-9, 10, (n, h_kv, hd)) for n in n_kv]
    for g, common in enumerate(groups[1] if groups else []):
        a, b = groups[0][g], groups[0][g + 1]
        longest = max(range(a, b), key=lambda i: n_kv[i])
        for i in range(a, b):
            m = min(common, n_kv[i])
            values[i][:m] = values[longest][:m]
            pool.table[i, :m // page] = pool.table[longest, :m // page]
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n_rows, sums = int(starts[-1]), []
    for s, n in enumerate(n_kv):
        at = (pool.table[s, np.arange(n) // page], np.arange(n) % page)
        pool.view(pool.k)[at] = 0
        pool.view(pool.v)[at] = values[s]
        if eight:
            pool.scale_view()[at] = 1
        sums.append(np.concatenate([np.zeros((1, h_kv, hd), np.int64), np.cumsum(values[s], axis=0)]))
        assert np.abs(sums[-1]).max() + 9 * n < 2 ** 23
    q_stride, out_stride = h * hd + q_pad, h * hd + out_pad
    q = np.full((n_rows, q_stride), np.nan, np.float16)
    q[:, :h * hd] = rng.standard_normal((n_rows, h * hd))
    out0 = np.full((n_rows, out_stride), 7.5, out)
    po = dev(out0)
    batch = B.paged_batch(dev(starts), dev(np.array(n_kv, np.int32)), dev(pool.table), len(rows), n_rows, pool.table.shape[1], max_rows)
    a = B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), batch, dev(q), po, h, out_type=TYPES[out], causal=causal, window=window, q_stride=q_stride, out_stride=out_stride)
    more = {}
    if groups:
        size = B.paged_attend_workspace(len(rows), n_rows, h, hd)
        more = dict(group_start=dev(np.array(groups[0], np.int32)), n_shared=dev(np.array(groups[1], np.int32)), n_group=len(groups[1]), workspace=dev(np.full(size, 0xff, np.uint8)), workspace_bytes=size)
    be.paged_attend(B.paged_attend_desc(a, pool.of_scales(dev(pool.scales)) if eight else None, **more))
    got = dev.back(po, out0)
    assert (got[:, h * hd:] == 7.5).all()                    # between the rows
    got = got[:, :h * hd].reshape(n_rows, h, hd).astype(np.float64)
    heads = np.arange(h) // (h // h_kv)
    for s, n in enumerate(n_kv):
        hi = np.arange(n - rows[s], n) + 1 if causal else np.full(rows[s], n)
        lo = np.maximum(0, hi - window) if window else np.zeros(rows[s], int)
        total, count = (sums[s][hi] - sums[s][lo])[:, heads], (hi - lo)[:, None, None]
        want = total / count
        tol = np.abs(want) * 2.0 ** -23 if out == np.float32 else np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25
        assert (np.abs(got[starts[s]:starts[s + 1]] - want) <= tol).all(), s


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_every_position_of_long_contexts(be, dev, hd):
    rng = np.random.default_rng(hd)
    check_counts(be, dev, rng, [1], [40000], 2, 1, hd, 64, max_rows=1)
    check_counts(be, dev, rng, [1], [65537], 1, 1, hd, 24, max_rows=1)
    check_counts(be, dev, rng, [3, 1], [50001, 20011], 4, 1, hd, 16)
    check_counts(be, dev, rng, [7, 1, 30], [30000, 11, 9001], 5, 1, hd, 32)
    check_counts(be, dev, rng, [40], [9000], 2, 1, hd, 64)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("n_seq", [1, 2, 5, 6, 13, 160, 161, 512, 513, 800])
def test_every_position_of_many_sequences(be, dev, n_seq, hd):
    """As many sequences as warps, as threads, and more than either; of no rows, single rows, a few and many."""
    rng = np.random.default_rng(n_seq)
    rows = rng.choice([0, 1, 1, 2, 5, 40], n_seq)
    rows[0] = 3
    if n_seq <= 13:
        rows[-1] = 300
    n_kv = [int(x) for x in rng.integers(1, 400 if n_seq > 20 else 4000, n_seq)]
    check_counts(be, dev, rng, rows.tolist(), n_kv, 6, 2, hd, 16)
    check_counts(be, dev, rng, np.minimum(rows, 1).tolist(), n_kv, 6, 2, hd, 16, max_rows=1)
    check_counts(be, dev, rng, np.minimum(rows, 2).tolist(), n_kv, 9, 1, hd, 64, max_rows=2)
    check_counts(be, dev, rng, rows.tolist(), n_kv, 2, 1, hd, 8, window=90)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("out", [np.float32, np.float16])
def test_every_position_with_room_between_rows_many_tiles_and_many_heads(be, dev, hd, out):
    rng = np.random.default_rng(hd)
    for rows, n_kv in (([1, 1, 3], [300, 41, 90]), ([200, 1, 33], [900, 41, 33]), ([20], [6000])):
        check_counts(be, dev, rng, rows, n_kv, 4, 2, hd, 16, q_pad=8, out_pad=hd, out=out)
        check_counts(be, dev, rng, rows, n_kv, 3, 1, hd, 16, q_pad=2 * hd + 24, out_pad=8, out=out, eight=False, groups=([0, len(rows)], [31]))
    check_counts(be, dev, rng, [1300, 2, 1100], [1400, 900, 1100], 2, 2, hd, 16, out=out)
    check_counts(be, dev, rng, [2300, 700], [2300, 900], 8, 1, hd, 3, out=out)
    for group in (24, 25, 127, 129, 300):
        check_counts(be, dev, rng, [1, 5, 20], [300, 41, 700], group, 1, hd, 16, out=out)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [8, 16, 24, 64, 128])
def test_every_position_of_shared_beginnings(be, dev, eight, hd, page):
    """Whole pages are shared, or what the last rows see in common; of one row a sequence to many, on both passes' kernels, with cut items and without."""
    rng = np.random.default_rng(hd + page)
    for rows, h, h_kv in (([1] * 12, 4, 2), ([3] * 12, 10, 1), ([1, 2, 1, 40, 1, 0, 5, 1, 1, 30, 1, 1], 4, 4)):
        n_kv = [1500 + r + int(x) for r, x in zip(rows, rng.integers(0, 700, 12))]
        check_counts(be, dev, rng, rows, n_kv, h, h_kv, hd, page, eight, groups=([0, 4, 5, 12], [1500, 900, 1333]))
        check_counts(be, dev, rng, rows, n_kv, h, h_kv, hd, page, eight, groups=([1, 6, 11], [128 + page, 1499]), causal=False, out=np.float16)


@pytest.mark.parametrize("eight", [False, True])
def test_every_position_of_many_groups(be, dev, eight):
    rng = np.random.default_rng(77)
    n = 600
    rows = rng.choice([0, 1, 1, 1, 3], n).tolist()
    n_kv = [400 + r + int(x) for r, x in zip(rows, rng.integers(0, 50, n))]
    starts = np.unique(np.concatenate([[0, n], rng.integers(0, n, 200)])).tolist()
    check_counts(be, dev, rng, rows, n_kv, 4, 1, 64, 16, eight, groups=(starts, rng.integers(0, 400, len(starts) - 1).tolist()))
    check_counts(be, dev, rng, [1] * 300, [9000 + i for i in range(300)], 2, 1, 128, 64, eight, groups=([0, 300], [9000]), max_rows=1)


# ---------------------------------------------------------------------------------------------- together, and beside others
def test_a_serving_loop_on_bytes(be, dev):
    """Requests behind one system prompt come in chunks: normalised, rotated and stored in bytes, attended over what they share and what is theirs; what is read back is what attention saw."""
    rng = np.random.default_rng(51)
    h, h_kv, hd, page, common = 4, 2, 64, 16, 300
    d, width = 96, (h + 2 * h_kv) * hd
    w_qkv, norms = rng.standard_normal((d, width)) * d ** -0.5, (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    system, own = rng.standard_normal((common, d)), [rng.standard_normal((n, d)) for n in (60, 1, 37, 90)]
    texts = [np.concatenate([system, x]) for x in own]
    n_seq = len(texts)
    pool = BytePool(rng, [len(t) + 4 for t in texts], h_kv, hd, page)
    pool.table[1:, :common // page] = pool.table[0, :common // page]
    pk, pv, ps, pt, pn = dev(pool.k), dev(pool.v), dev(pool.scales), dev(pool.table), dev(norms)
    groups = dict(group_start=dev(np.array([0, n_seq], np.int32)), n_shared=dev(np.array([common], np.int32)), n_group=1)
    # the first request brings the system prompt, the others begin behind it with the part of a page that is not whole
    done = [0] + [common // page * page] * (n_seq - 1)
    for step in range(7):
        rows = [0 if step == 0 and s > 0 else min(common if step == 0 else 32, len(t) - n) for s, (t, n) in enumerate(zip(texts, done))]
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        n_kv = np.array([n + r for n, r in zip(done, rows)], dtype=np.int32)
        x = (np.concatenate([t[n:n + r] for t, n, r in zip(texts, done, rows)]) @ w_qkv).astype(np.float32)
        n_rows = int(starts[-1])
        if n_rows == 0:
            break
        px, pq, po = dev(x), dev(np.zeros((n_rows, h, hd), np.float16)), dev(np.zeros((n_rows, h, hd), np.float32))
        batch = B.paged_batch(dev(starts), dev(n_kv), pt, n_seq, n_rows, pool.table.shape[1], max(rows))
        cache, scales = pool.cache(pk, pv), pool.of_scales(ps)
        append = B.paged_append_desc(cache, batch, px, px + 4 * h * hd, px + 4 * (h + h_kv) * hd, pq, h, row_stride=width, rope_mode=B.ROPE_HALVES)
        be.paged_store(B.paged_store_desc(append, scales, q_norm=pn, k_norm=pn + 4 * hd, norm_eps=1e-6))
        size = B.paged_attend_workspace(n_seq, n_rows, h, hd)
        be.paged_attend(B.paged_attend_desc(B.paged_attention_desc(cache, batch, pq, po, h, out_type=B.FP32), scales, workspace=dev(np.zeros(size, np.uint8)), workspace_bytes=size, **groups))
        # every position of every sequence, read back
        whole = np.concatenate([[0], np.cumsum(n_kv)]).astype(np.int32)
        out0 = np.zeros((int(whole[-1]), h_kv, hd), np.float32)
        rk, rv = dev(out0), dev(out0)
        be.paged_load(B.paged_load_desc(cache, B.paged_batch(dev(whole), dev(n_kv), pt, n_seq, int(whole[-1]), pool.table.shape[1]), rk, rv, scales, out_type=B.FP32))
        k, v, q, out = dev.back(rk, out0).astype(np.float64), dev.back(rv, out0).astype(np.float64), dev.back(pq, np.zeros((n_rows, h, hd), np.float16)), dev.back(po, np.zeros((n_rows, h, hd), np.float32))
        for s in range(n_seq):
            a, b, c, e = starts[s], starts[s + 1], whole[s], whole[s + 1]
            if b > a:
                largest = np.abs(np.concatenate([k[c:e], v[c:e]], -1)).max((0, 2)) / 127 * (1 + 2.0 ** -9) + 2.0 ** -24
                check_rows(out[a:b], q[a:b].astype(np.float64), k[c:e], v[c:e], done[s], hd ** -0.5, True, 0, np.ones(n_kv[s], dtype=bool),
                           np.broadcast_to(largest[None, :, None], (n_kv[s], h_kv, 2)), np.float32)
                full = x[a:b].reshape(-1, h + 2 * h_kv, hd).astype(np.float64)
                turned = plain_rope(plain_norm(full[:, h:h + h_kv], norms[1].astype(np.float64), np.float64(np.float32(1e-6))), np.arange(done[s], n_kv[s]), B.ROPE_HALVES, hd, 10000.0, 1.0)
                for got, want in ((k[c + done[s]:e], turned), (v[c + done[s]:e], full[:, h + h_kv:])):
                    step_size = np.abs(want).max(-1, keepdims=True) / 127 * (1 + 2.0 ** -10) + 2.0 ** -24
                    assert (np.abs(got - want) <= step_size * 0.501 + np.abs(want).max() * 2.0 ** -17).all()
            done[s] = int(n_kv[s])
    assert done == [len(t) for t in texts]


def test_results_do_not_depend_on_programmatic_launch(dev):
    got = []
    for pdl in (True, False):
        b = B.B200Backend(0, use_pdl=pdl)
        d, rng = Device(b), np.random.default_rng(31)
        pool = BytePool(rng, [600, 500, 490], 2, 64, 16)
        pool.table[1:, :28] = pool.table[0, :28]
        pool.put(0, *rng.standard_normal((2, 599, 2, 64)))
        batch = B.paged_batch(d(np.array([0, 1, 21, 60], np.int32)), d(np.array([600, 500, 490], np.int32)), d(pool.table), 3, 60, pool.table.shape[1])
        cache, scales = pool.cache(d(pool.k), d(pool.v)), pool.of_scales(d(pool.scales))
        x = d(rng.standard_normal((60, 8 * 64)).astype(np.float32))
        q, o, kv = d(np.zeros((60, 4, 64), np.float16)), np.zeros((60, 4 * 64), np.float32), np.zeros((60, 2, 64), np.float16)
        po, pk, pv, size = d(o), d(kv), d(kv), B.paged_attend_workspace(3, 60, 4, 64)
        room, start, common, norm = d(np.zeros(size, np.uint8)), d(np.array([0, 3], np.int32)), d(np.array([448], np.int32)), d(np.ones(64, np.float32))
        for _ in range(20):
            b.paged_store(B.paged_store_desc(B.paged_append_desc(cache, batch, x, x + 4 * 256, x + 4 * 384, q, 4, row_stride=512), scales, q_norm=norm, k_norm=norm))
            b.paged_attend(B.paged_attend_desc(B.paged_attention_desc(cache, batch, q, po, 4, out_type=B.FP32), scales, start, common, 1, room, size))
            b.paged_load(B.paged_load_desc(cache, batch, pk, pv, scales))
        got.append((d.back(po, o), d.back(pk, kv), d.back(pv, kv)))
        d.free()
        b.close()
    assert got[0][0].any() and all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(*got))   # (bits: what was never stored is NaN)


@pytest.mark.parametrize("hd,h", [(128, 2), (64, 4), (96, 2)])
def test_bytes_beyond_32_bits(be, dev, hd, h):
    """Bytes and scales more than 2^32 behind the pools' first: the same bits as with pages side by side."""
    import torch

    rng = np.random.default_rng(hd)
    n, page, far = 40, 16, (1 << 32) + 64
    table = np.array([[2, 0, 1]], np.int32)
    x, q = rng.standard_normal((n, (h + 2) * hd)).astype(np.float32), rng.standard_normal((n, h, hd)).astype(np.float16)
    store = torch.full((2 * far + (1 << 18),), 3, dtype=torch.uint8, device="cuda")
    pairs = torch.full((2 * far + 64,), 0, dtype=torch.int16, device="cuda")     # (pairs of 4 bytes, far / 2 a page and more)
    torch.cuda.synchronize()
    px, pq, pt = dev(x), dev(q), dev(table)
    near = B.paged_cache(dev(np.full(3 * page * hd, 3, np.int8)), dev(np.full(3 * page * hd, 3, np.int8)), 3, page, 1, hd, number_type=B.INT8)
    base, got = store.data_ptr(), []
    for c, sc in ((near, B.paged_scales(dev(np.zeros(2 * 3 * page, np.float16)), page, 1)),
                  (B.paged_cache(base, base + (1 << 17), 3, page, 1, hd, strides=(far, hd, page * hd), number_type=B.INT8), B.paged_scales(pairs.data_ptr(), page, 1, strides=(far // 2, 1, page)))):
        batch = B.paged_batch(dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), pt, 1, n, 3)
        turned, out, kv = dev(np.zeros((n, h, hd), np.float16)), np.zeros((n + 1, h, hd), np.float32), np.zeros((n, 1, hd), np.float32)
        be.paged_store(B.paged_store_desc(B.paged_append_desc(c, batch, px, px + 4 * h * hd, px + 4 * (h + 1) * hd, turned, h, row_stride=(h + 2) * hd), sc))
        po, pk, pv = dev(out), dev(kv), dev(kv)
        be.paged_attend(B.paged_attend_desc(B.paged_attention_desc(c, batch, pq, po, h, out_type=B.FP32), sc))
        one = B.paged_batch(dev(np.array([0, 1], np.int32)), dev(np.array([n], np.int32)), pt, 1, 1, 3)
        be.paged_attend(B.paged_attend_desc(B.paged_attention_desc(c, one, pq, po + 4 * n * h * hd, h, out_type=B.FP32), sc))
        be.paged_load(B.paged_load_desc(c, batch, pk, pv, sc, out_type=B.FP32))
        got.append((dev.back(po, out), dev.back(pk, kv), dev.back(pv, kv)))
    assert got[0][0].any(axis=(1, 2)).all() and got[0][1].any() and all(np.array_equal(a.view(np.uint32), b.view(np.uint32)) for a, b in zip(*got))


def test_two_backends_at_once(dev):
    import threading

    rng = np.random.default_rng(9)
    n_kv = [1700, 1660, 3000, 1500]
    pool = BytePool(rng, n_kv, 2, 128, 16)
    pool.table[1:, :90] = pool.table[0, :90]
    for s, n in enumerate(n_kv):
        pool.put(s, *rng.standard_normal((2, n, 2, 128)))
    q = rng.standard_normal((142, 8, 128)).astype(np.float16)
    results = [None] * 3

    def work(i):
        b = B.B200Backend(0)
        d = Device(b)
        cache, scales = pool.cache(d(pool.k), d(pool.v)), pool.of_scales(d(pool.scales))
        po, size = d(np.zeros(q.shape, np.float16)), B.paged_attend_workspace(4, 142, 8, 128)
        room, pq = d(np.zeros(size, np.uint8)), d(q)
        batch = B.paged_batch(d(np.array([0, 130, 140, 141, 142], np.int32)), d(np.array(n_kv, np.int32)), d(pool.table), 4, 142, pool.table.shape[1])
        few = B.paged_batch(d(np.array([0, 1, 3, 4, 6], np.int32)), d(np.array(n_kv, np.int32)), d(pool.table), 4, 6, pool.table.shape[1], 2)
        shared = dict(group_start=d(np.array([0, 4], np.int32)), n_shared=d(np.array([1440], np.int32)), n_group=1, workspace=room, workspace_bytes=size)
        calls = [B.paged_attend_desc(B.paged_attention_desc(cache, x, pq, po, 8), scales, **k) for x in (batch, few) for k in ({}, shared)]
        for _ in range(60):
            for c in calls:
                b.paged_attend(c)
        got = []
        for c in calls:
            b.paged_attend(c)
            got.append(d.back(po, np.zeros(q.shape, np.float16)))
        results[i] = got
        d.free()
        b.close()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    work(2)
    assert all(np.array_equal(x, y) for r in results[:2] for x, y in zip(r, results[2]))


def test_first_calls_beside_a_stream_capture(dev):
    """A backend's first calls while another library captures a stream: nothing is allocated in them."""
    import torch

    rng = np.random.default_rng(41)
    pool = BytePool(rng, [700, 690], 2, 64, 16)
    pool.table[1, :40] = pool.table[0, :40]
    for s, n in enumerate((700, 690)):
        pool.put(s, *rng.standard_normal((2, n, 2, 64)))
    b = B.B200Backend(0)
    d = Device(b)
    cache, scales = pool.cache(d(pool.k), d(pool.v)), pool.of_scales(d(pool.scales))
    many = B.paged_batch(d(np.array([0, 140, 141], np.int32)), d(np.array([700, 690], np.int32)), d(pool.table), 2, 141, pool.table.shape[1])
    one = B.paged_batch(d(np.array([0, 1, 2], np.int32)), d(np.array([700, 690], np.int32)), d(pool.table), 2, 2, pool.table.shape[1], 1)
    px, pq, size = d(rng.standard_normal((141, 8 * 64)).astype(np.float32)), d(np.zeros((141, 4, 64), np.float16)), B.paged_attend_workspace(2, 141, 4, 64)
    out, kv = np.zeros((141, 4, 64), np.float32), np.zeros((141, 2, 64), np.float16)
    po, pk, pv, room, start, common = d(out), d(kv), d(kv), d(np.zeros(size, np.uint8)), d(np.array([0, 2], np.int32)), d(np.array([640], np.int32))

    def calls():
        got = []
        for batch in (many, one):
            b.paged_store(B.paged_store_desc(B.paged_append_desc(cache, batch, px, px + 4 * 256, px + 4 * 384, pq, 4, row_stride=512), scales))
            for groups in ({}, dict(group_start=start, n_shared=common, n_group=1, workspace=room, workspace_bytes=size)):
                b.paged_attend(B.paged_attend_desc(B.paged_attention_desc(cache, batch, pq, po, 4, out_type=B.FP32), scales, **groups))
            b.paged_load(B.paged_load_desc(cache, batch, pk, pv, scales))
        return got

    x = torch.zeros(1000, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        calls()
    during = d.back(po, out), d.back(pk, kv), d.back(pv, kv)
    calls()
    assert during[0].any() and all(np.array_equal(a, d.back(p, a)) for a, p in zip(during, (po, pk, pv)))
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all()
    d.free()
    b.close()


@pytest.mark.parametrize("who", [1, 2, 3, 4])
def test_roles_that_come_late(dev, who):
    """Roles microseconds behind change nothing; copies three limits late are given up on: the kernels end by themselves with the copies landed, the status says so, and later launches on the backend are right."""
    b = B.B200Backend(0)
    assert b.paged_selftest_late(who, 1_000_000_000 if who == 1 else 2_000_000) == (0 if who == 1 else 7)
    assert b.paged_selftest_late(1, 1_000_000_000) == 0
    d = Device(b)
    rng = np.random.default_rng(who)
    for hd in (64, 128):
        check_attend(b, d, rng, [150, 1, 40], [700, 2000, 90], 4, 2, hd, 16)
        check_attend(b, d, rng, [2, 1, 3], [700, 2000, 600], 6, 2, hd, 16, groups=([0, 3], [590]))
    d.free()
    b.close()
