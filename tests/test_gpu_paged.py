"""GPU: the operators over paged caches and the sampler against plain numpy in 64 bits.

Tolerances: a rounding is off by half a step at most, relative 2^-11 for fp16 (2^-25 absolutely among its smallest values) and 2^-24 for f32; what follows from it
is derived where it is used."""
import numpy as np
import pytest

from spy_b200 import backend as B
from spy_b200 import gguf_io, quants

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.B200Backend(0)
    yield b
    b.close()


class Device:
    """Arrays on the device that go when the test is over."""

    def __init__(self, be):
        self.be, self.held = be, []

    def __call__(self, a):
        a = np.ascontiguousarray(a)
        p = self.be.upload(a)
        self.held.append((p, max(1, a.nbytes)))
        return p

    def back(self, p, like):
        return self.be.download(p, like.shape, like.dtype)

    def free(self):
        self.be.sync()
        for p, n in self.held:
            self.be.dealloc_memory(p, n)


@pytest.fixture
def dev(be):
    d = Device(be)
    yield d
    d.free()


class Pool:
    """Pages in random order with NaN wherever nothing is stored; `k` and `v`: what each sequence has stored, [position][head][element]."""

    def __init__(self, rng, n_kv, heads, head_dim, page, token_major=False, strides=None, spare=2, fill=np.nan):
        self.page, self.heads, self.hd, self.n_kv, self.token_major = page, heads, head_dim, list(n_kv), token_major
        need = [-(-max(0, n) // page) for n in n_kv]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(n_kv), max(1, max(need))), -1, dtype=np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        if strides is None:
            strides = (page * heads * head_dim, heads * head_dim, head_dim) if token_major else (page * heads * head_dim, head_dim, page * head_dim)
        self.strides = strides
        self.size = self.n_pages * strides[0] + (page - 1) * strides[1] + (heads - 1) * strides[2] + head_dim
        self.k, self.v = (np.full(self.size, fill, dtype=np.float16) for _ in range(2))

    def view(self, a):
        return np.lib.stride_tricks.as_strided(a, (self.n_pages, self.page, self.heads, self.hd), tuple(2 * s for s in self.strides) + (2,))

    def put(self, s, k, v):
        pos = np.arange(len(k))
        for a, x in ((self.k, k), (self.v, v)):
            self.view(a)[self.table[s, pos // self.page], pos % self.page] = x

    def get(self, a, s, n=None):
        n = max(0, self.n_kv[s]) if n is None else n
        pos = np.arange(n)
        return self.view(a)[self.table[s, pos // self.page], pos % self.page]

    def cache(self, pk, pv):
        return B.paged_cache(pk, pv, self.n_pages, self.page, self.heads, self.hd, strides=self.strides)


def plain_attention(q, k, v, first, scale, causal, window, there):
    """q [rows][heads][e]; k, v [positions][kv heads][e], f64. Returns out, and per element how far fp16 probabilities and f32 sums may move it."""
    rows, h, hd = q.shape
    n, h_kv, _ = k.shape
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(rows):
        j = np.arange(n)
        seen = there.copy()
        if causal:
            seen &= j <= first + i
            if window:
                seen &= j > first + i - window
        if not seen.any():
            continue
        for x in range(h):
            kk, vv = k[seen][:, x // (h // h_kv)], v[seen][:, x // (h // h_kv)]
            t = kk @ q[i, x] * scale
            w = np.exp(t - t.max())
            w /= w.sum()
            out[i, x] = w @ vv
            with np.errstate(invalid="ignore"):
                # scores: f32 sums of exact products (head_dim terms), scaled, subtracted, 2^x: relative error of a probability
                d_score = (hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[i, x])).max() * abs(scale) + 2.0 ** -20
                # probabilities to fp16, twice (sum and product use the same ones), their smallest absolutely; f32 sums
                rel = 2 * (2.0 ** -11 + d_score) + (len(w) / 16 + 40) * 2.0 ** -24
                off[i, x] = rel * (w @ np.abs(vv)) + len(w) * 2.0 ** -24 * np.abs(vv).max()
    return out, off


def run_attention(be, dev, pool, row_start, q, out0, **kw):
    n_rows, h, hd = q.shape
    row_start = np.asarray(row_start, dtype=np.int32)
    c = pool.cache(dev(pool.k), dev(pool.v))
    b = B.paged_batch(dev(row_start), dev(np.array(pool.n_kv, dtype=np.int32)), dev(pool.table), len(pool.n_kv), n_rows, pool.table.shape[1], kw.pop("max_rows", 0))
    po = dev(out0)
    d = B.paged_attention_desc(c, b, dev(q), po, h, out_type=B.FP32 if out0.dtype == np.float32 else B.FP16, **kw)
    be.paged_attention(d)
    got = dev.back(po, out0)
    be.paged_attention(d)                                    # the same bits every time
    again = dev.back(po, out0)
    assert np.array_equal(got.view(np.uint8), again.view(np.uint8))
    return got


def check_attention(be, dev, rng, rows, n_kv, h, h_kv, hd, page, causal=True, window=0, scale=0.0, out=np.float16, token_major=False, pad=0, spread=1.0, max_rows=0, drop=None, strides=None, share=0):
    pool = Pool(rng, n_kv, h_kv, hd, page, token_major, strides)
    for s, n in enumerate(n_kv):
        pool.put(s, *(rng.standard_normal((2, max(0, n), h_kv, hd)).astype(np.float16)))
    pool.table[1:, :share] = pool.table[0, :share]             # (a common beginning)
    if drop is not None:
        pool.table[rng.random(pool.table.shape) < drop] = -1
        pool.table[rng.random(pool.table.shape) < drop / 2] = pool.n_pages + 5
    starts = np.concatenate([[0], np.cumsum(rows)])
    q = (spread * rng.standard_normal((starts[-1] + pad, h, hd))).astype(np.float16)
    out0 = np.full(q.shape, 7.5, dtype=out)
    got = run_attention(be, dev, pool, starts, q, out0, causal=causal, window=window, scale=scale, max_rows=max_rows)
    for s, n in enumerate(n_kv):
        pos = np.arange(max(0, n))
        pages = pool.table[s, pos // page]
        there = (pages >= 0) & (pages < pool.n_pages)
        safe = np.where(there, pages, 0)
        k, v = (np.where(there[:, None, None], pool.view(a)[safe, pos % page], 0).astype(np.float64) for a in (pool.k, pool.v))
        a, b = starts[s], starts[s + 1]
        want, off = plain_attention(q[a:b].astype(np.float64), k, v, n - rows[s], scale or hd ** -0.5, causal, window, there)
        tol = off + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if out == np.float16 else np.abs(want) * 2.0 ** -24)
        err = np.abs(got[a:b].astype(np.float64) - want)
        assert (err <= tol).all(), (s, float((err / np.maximum(tol, 1e-30)).max()), np.unravel_index(np.argmax(err - tol), err.shape))
        assert (got[a:b][~np.any(off > 0, axis=2)] == 0).all()
    assert (got[starts[-1]:] == 7.5).all()                   # rows behind the last sequence


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("h,h_kv", [(4, 4), (6, 2), (5, 1), (8, 1)])
def test_single_tokens(be, dev, hd, h, h_kv):
    rng = np.random.default_rng(hd * 100 + h * 10 + h_kv)
    check_attention(be, dev, rng, [1] * 7, [1, 2, 15, 16, 17, 300, 1031], h, h_kv, hd, 16, pad=2, max_rows=1)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 200, 256])
@pytest.mark.parametrize("token_major", [False, True])
def test_pages_of_all_sizes(be, dev, page, token_major):
    rng = np.random.default_rng(page)
    check_attention(be, dev, rng, [1, 3, 40, 0, 1], [77, 130, 290, 55, 1], 4, 2, 64, page, token_major=token_major)
    check_attention(be, dev, rng, [140, 2], [333, 64], 4, 1, 128, page, token_major=token_major)


@pytest.mark.parametrize("rows,n_kv", [([1], [0]), ([0], [5]), ([3], [2]), ([5, 1, 0, 2], [5, 0, 9, 1]), ([130], [130]), ([129], [500]), ([257], [260]), ([64, 1, 64], [64, 700, 200])])
@pytest.mark.parametrize("hd", [64, 128])
def test_short_and_empty(be, dev, rows, n_kv, hd):
    """No positions at all, more rows than positions (rows without a key are zeros), no rows, whole prompts."""
    rng = np.random.default_rng(len(rows) + rows[0])
    check_attention(be, dev, rng, rows, n_kv, 4, 2, hd, 16, pad=3)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 128, 129, 1000])
@pytest.mark.parametrize("rows", [1, 5, 150])
def test_windows(be, dev, window, rows):
    rng = np.random.default_rng(window)
    check_attention(be, dev, rng, [rows, 1, rows], [700, 90, rows], 6, 2, 64, 16, window=window)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("rows", [1, 9, 200])
def test_without_causal_order_and_with_other_scales(be, dev, hd, rows):
    rng = np.random.default_rng(hd + rows)
    check_attention(be, dev, rng, [rows, rows], [310, 40], 4, 2, hd, 32, causal=False, scale=0.3)
    check_attention(be, dev, rng, [rows], [310], 4, 4, hd, 32, scale=-0.1, out=np.float32)


@pytest.mark.parametrize("rows", [1, 4, 33, 300])
@pytest.mark.parametrize("hd", [64, 128])
def test_f32_outputs_and_sharp_rows(be, dev, rows, hd):
    rng = np.random.default_rng(rows)
    check_attention(be, dev, rng, [rows, rows], [900, rows], 8, 2, hd, 16, out=np.float32, spread=6.0)


@pytest.mark.parametrize("rows", [1, 6, 160])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_that_are_not_there(be, dev, rows, hd):
    rng = np.random.default_rng(rows * hd)
    for drop in (0.3, 0.9, 1.0):
        check_attention(be, dev, rng, [rows, rows, 1], [400, 170, 333], 4, 2, hd, 16, drop=drop)


@pytest.mark.parametrize("rows", [2, 30, 200])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite_reach_only_who_sees_them(be, dev, rows, hd, value):
    """A K or V element of a later position, of one outside the window, behind the sequence's end or in a free page has no influence."""
    rng = np.random.default_rng(rows + hd)
    n, h, h_kv, window = 230 + rows, 4, 2, 90
    pool = Pool(rng, [n], h_kv, hd, 16, fill=value)
    k, v = rng.standard_normal((2, n, h_kv, hd)).astype(np.float16)
    bad_v, bad_k, old = n - rows + rows // 2, n - 1, n - rows - window - 3       # seen by the rows behind it in its window, by the last one, by nobody
    v[bad_v, 0, 5] = value
    k[bad_k, 1, 3] = value
    v[old, :, :] = value
    k[old, :, :] = value
    pool.put(0, k, v)
    q = rng.standard_normal((rows, h, hd)).astype(np.float16)
    got = run_attention(be, dev, pool, [0, rows], q, np.zeros(q.shape, dtype=np.float32), window=window)
    first = n - rows
    good_k, good_v = k.astype(np.float64), v.astype(np.float64)
    for a in (good_k, good_v):
        a[~np.isfinite(a)] = 0
    want, off = plain_attention(q.astype(np.float64), good_k, good_v, first, hd ** -0.5, True, window, np.ones(n, dtype=bool))
    err = np.abs(got - want)
    clean = np.ones(q.shape, dtype=bool)
    seeing = slice(bad_v - first, bad_v - first + window)
    clean[seeing, :2, 5] = False                              # the rows that see the bad V, in that element
    clean[rows - 1, 2:, :] = False                            # the row that sees the bad K
    assert (err[clean] <= (off + np.abs(want) * 2.0 ** -24)[clean]).all()
    dirty = got[seeing, :2, 5]
    assert (np.isnan(dirty) if np.isnan(value) else (dirty == value) | np.isnan(dirty)).all()


def test_whole_chip_on_one_head_and_cut_items(be, dev):
    """One K/V head and a long context: every CTA has a piece of the same item."""
    rng = np.random.default_rng(5)
    check_attention(be, dev, rng, [1], [40000], 2, 1, 64, 64, max_rows=1)
    check_attention(be, dev, rng, [40], [9000], 2, 1, 128, 64)


@pytest.mark.parametrize("hd", [64, 128])
def test_items_with_one_tile_between_others(be, dev, hd):
    """Many items a CTA, every other one with a second tile that has no rows or sees nothing: the order of the stretches' hand-overs, over and over."""
    rng = np.random.default_rng(hd)
    rows, n_kv, h = [300, 60, 513, 40, 300], [300, 700, 513, 40, 20], 40
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    pool = Pool(rng, n_kv, h, hd, 16, fill=0.0)
    for s, n in enumerate(n_kv):
        pool.put(s, *rng.standard_normal((2, n, h, hd)).astype(np.float16))
    q = rng.standard_normal((starts[-1], h, hd)).astype(np.float16)
    out = np.zeros(q.shape, dtype=np.float16)
    po = dev(out)
    d = B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), B.paged_batch(dev(starts), dev(np.array(n_kv, np.int32)), dev(pool.table), 5, int(starts[-1]), pool.table.shape[1]), dev(q), po, h, window=200)
    for _ in range(300):
        be.paged_attention(d)
    got = dev.back(po, out)
    for s in (0, 2, 4):
        k, v = (pool.get(a, s).astype(np.float64)[:, :2] for a in (pool.k, pool.v))
        want, off = plain_attention(q[starts[s]:starts[s + 1], :2].astype(np.float64), k, v, n_kv[s] - rows[s], hd ** -0.5, True, 200, np.ones(n_kv[s], dtype=bool))
        assert (np.abs(got[starts[s]:starts[s + 1], :2] - want) <= off + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()


def test_long_contexts_over_and_over(be, dev):
    """Copies from cold memory land in any order: no role may take one phase of a ring slot for another (a wait that ran out shows as an error)."""
    import torch

    n, h_kv, hd, page = 90000, 8, 128, 64
    pools = torch.randn((2, n // page + 1, h_kv, page, hd), device="cuda", dtype=torch.float16)
    q = torch.randn((5, 40, hd), device="cuda", dtype=torch.float16)
    out = torch.empty((8,) + tuple(q.shape), device="cuda", dtype=torch.float16)
    table = torch.randperm(pools.shape[1], device="cuda").int()
    start, n_kv = torch.tensor([0, 5], device="cuda", dtype=torch.int32), torch.tensor([n], device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    c = B.paged_cache(pools[0].data_ptr(), pools[1].data_ptr(), pools.shape[1], page, h_kv, hd)
    b = B.paged_batch(start.data_ptr(), n_kv.data_ptr(), table.data_ptr(), 1, 5, table.numel())
    d = [B.paged_attention_desc(c, b, q.data_ptr(), o.data_ptr(), 40) for o in out]
    for i in range(600):
        be.paged_attention(d[i % 8])
    be.sync()
    assert all(torch.equal(o, out[0]) for o in out)


def test_more_sequences_than_threads(be, dev):
    rng = np.random.default_rng(6)
    n = 700
    rows = rng.integers(0, 3, n).tolist()
    check_attention(be, dev, rng, rows, [int(x) for x in rng.integers(0, 60, n)], 2, 1, 32, 16)
    check_attention(be, dev, rng, rows, [int(x) for x in rng.integers(0, 60, n)], 24, 1, 64, 16)


def test_shared_pages_and_other_strides(be, dev):
    """Two sequences with the same first pages; heads and positions with room between them."""
    rng = np.random.default_rng(7)
    check_attention(be, dev, rng, [1, 50], [200, 150], 4, 2, 64, 16, strides=(16 * 2 * 96 + 40, 72 + 72, 72))
    pool = Pool(rng, [100, 100], 2, 64, 16)
    pool.table[1, :4] = pool.table[0, :4]
    k, v = rng.standard_normal((2, 100, 2, 64)).astype(np.float16)
    pool.put(1, k, v)
    pool.put(0, k, v)
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    q[1] = q[0]
    got = run_attention(be, dev, pool, [0, 1, 2], q, np.zeros(q.shape, dtype=np.float16))
    assert np.array_equal(got[0], got[1])


def test_lengths_that_make_no_sense_touch_nothing_else(be, dev):
    """Negative lengths, lengths beyond the table, rows beyond the buffer: answered inside the described buffers (margins around them stay)."""
    rng = np.random.default_rng(8)
    pool = Pool(rng, [64, 64, 64], 2, 64, 16, fill=0.5)
    pool.n_kv = [-5, 100000, 70]
    margin = np.full((4 + 6 + 4, 4, 64), 3.0, dtype=np.float16)
    po = dev(margin)
    b = B.paged_batch(dev(np.array([0, 2, 5, 50], dtype=np.int32)), dev(np.array(pool.n_kv, dtype=np.int32)), dev(pool.table), 3, 6, pool.table.shape[1])
    c = pool.cache(dev(pool.k), dev(pool.v))
    be.paged_attention(B.paged_attention_desc(c, b, dev(rng.standard_normal((6, 4, 64)).astype(np.float16)), po + 4 * 4 * 64 * 2, 4))
    got = dev.back(po, margin)
    assert (got[:4] == 3).all() and (got[10:] == 3).all()
    assert (got[4:6] == 0).all()                              # no positions
    assert np.allclose(got[6:9], 0.5, atol=2.0 ** -11)


# ---------------------------------------------------------------------------------------------- append
def plain_rope(x, pos, mode, rot, base, scale):
    out = x.copy()
    i = np.arange(rot // 2)
    angle = (pos[:, None] * (scale * np.float64(np.float32(base)) ** (-2.0 * i / rot)))[:, None, :]
    a, b = (2 * i, 2 * i + 1) if mode == B.ROPE_PAIRS else (i, i + rot // 2)
    out[..., a] = x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle)
    out[..., b] = x[..., a] * np.sin(angle) + x[..., b] * np.cos(angle)
    return out


def rope_off(x, mode, rot):
    """|a| + |b| of an element's pair: angle to 2^-26 of a circle, sine, cosine and the two products to f32."""
    s = np.abs(x).copy()
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if mode == B.ROPE_PAIRS else (i, i + rot // 2)
    s[..., a] = s[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return s * (2 * np.pi * 2.0 ** -26 + 4 * 2.0 ** -24)


def check_append(be, dev, rng, rows, n_kv, h, h_kv, hd, page, mode=B.ROPE_PAIRS, rot=None, base=10000.0, scale=1.0, dtype=np.float32, q_type=np.float16, token_major=False, pad=0, in_place=False, drop=0):
    rot = hd if rot is None else rot
    pool = Pool(rng, n_kv, h_kv, hd, page, token_major, fill=0.25)
    if drop:
        pool.table[rng.random(pool.table.shape) < drop] = -1
        pool.table[rng.random(pool.table.shape) < drop / 2] = pool.n_pages
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n_rows, width = int(starts[-1]) + pad, (h + 2 * h_kv) * hd + 8
    x = rng.standard_normal((n_rows, width)).astype(dtype)
    px, pk, pv = dev(x), dev(pool.k), dev(pool.v)
    q0 = np.full((n_rows, h, hd), -9, dtype=q_type)
    pq = px if in_place else dev(q0)
    e = x.itemsize * hd
    types = {np.float32: B.FP32, np.float16: B.FP16}
    d = B.paged_append_desc(pool.cache(pk, pv), B.paged_batch(dev(starts), dev(np.array(n_kv, dtype=np.int32)), dev(pool.table), len(rows), n_rows, pool.table.shape[1]),
                            px if h else None, px + h * e, px + (h + h_kv) * e, pq if h else None, h, in_type=types[dtype], q_out_type=types[q_type], row_stride=width,
                            q_out_stride=width if in_place else None, rope_mode=mode, rope_dim=rot, freq_base=base, freq_scale=scale)
    be.paged_append(d)
    got_k, got_v = dev.back(pk, pool.k), dev.back(pv, pool.v)
    got_q = dev.back(px, x)[:, :h * hd].reshape(n_rows, h, hd) if in_place else dev.back(pq, q0)
    want_k, want_v = pool.k.copy(), pool.v.copy()
    untouched = np.ones((n_rows,), dtype=bool)
    half = lambda a: np.abs(a) * 2.0 ** -11 + 2.0 ** -25  # noqa: E731
    for s, n in enumerate(n_kv):
        a, b = starts[s], starts[s + 1]
        pos = np.arange(n - rows[s], n)
        full = x[a:b, :(h + 2 * h_kv) * hd].reshape(b - a, h + 2 * h_kv, hd).astype(np.float64)
        turned = full if mode == B.ROPE_NONE else plain_rope(full, pos, mode, rot, base, scale)
        off = 0 * full if mode == B.ROPE_NONE else rope_off(full, mode, rot)
        ok = pos >= 0
        untouched[a:b] = ~ok
        if h:
            err = np.abs(got_q[a:b][ok].astype(np.float64) - turned[ok, :h])
            tol = off[ok, :h] + (half(turned[ok, :h]) if q_type == np.float16 else np.abs(turned[ok, :h]) * 2.0 ** -24)
            assert (err <= tol).all(), float((err / tol).max())
        pages = pool.table[s, pos[ok] // page] if ok.any() else np.zeros(0, dtype=int)
        there = (pages >= 0) & (pages < pool.n_pages)
        at = (pages[there], pos[ok][there] % page)
        for got, want, lo, exact in ((got_k, want_k, h, False), (got_v, want_v, h + h_kv, True)):
            value = (full if exact else turned)[ok][there][:, lo:lo + h_kv]
            have = pool.view(got)[at].astype(np.float64)
            assert (np.abs(have - value) <= half(value) + (0 if exact else off[ok][there][:, lo:lo + h_kv])).all()
            pool.view(want)[at] = pool.view(got)[at]
    assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)         # nothing else was stored
    untouched[starts[-1]:] = True
    if h:
        before = x[:, :h * hd].reshape(n_rows, h, hd) if in_place else q0
        assert np.array_equal(got_q[untouched], before[untouched])


@pytest.mark.parametrize("mode", [B.ROPE_NONE, B.ROPE_PAIRS, B.ROPE_HALVES])
@pytest.mark.parametrize("hd,rot", [(8, 8), (24, 16), (64, 64), (96, 48), (128, 128), (256, 256)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_append(be, dev, mode, hd, rot, dtype):
    rng = np.random.default_rng(hd + rot)
    check_append(be, dev, rng, [1, 20, 0, 3], [400, 20, 7, 100001], 6, 2, hd, 16, mode=mode, rot=rot, dtype=dtype, pad=2)
    check_append(be, dev, rng, [1], [33], 3, 3, hd, 5, mode=mode, rot=rot, dtype=dtype, q_type=np.float32, token_major=True, base=500000.0, scale=0.25)


def test_append_in_place_without_q_and_with_missing_pages(be, dev):
    rng = np.random.default_rng(11)
    check_append(be, dev, rng, [5, 2], [50, 2], 4, 2, 64, 16, q_type=np.float32, in_place=True)
    check_append(be, dev, rng, [5, 2], [50, 2], 4, 2, 64, 16, mode=B.ROPE_HALVES, dtype=np.float16, in_place=True)
    check_append(be, dev, rng, [5, 2], [50, 2], 0, 2, 64, 16)
    check_append(be, dev, rng, [40, 30], [300, 30], 4, 2, 64, 8, drop=0.5)
    check_append(be, dev, rng, [6, 1], [4, 0], 4, 2, 64, 8)                              # rows with negative positions


def test_append_of_many_sequences(be, dev):
    rng = np.random.default_rng(12)
    rows = rng.integers(0, 4, 1500).tolist()
    check_append(be, dev, rng, rows, [r + int(x) for r, x in zip(rows, rng.integers(0, 30, 1500))], 2, 1, 64, 16, pad=5)


def test_nothing_to_do(be, dev):
    """No sequences, no rows."""
    c = B.paged_cache(dev(np.zeros(4096, np.float16)), dev(np.zeros(4096, np.float16)), 2, 16, 1, 64)
    z = dev(np.zeros(64, np.float32))
    for n_seq, n_rows in ((0, 3), (2, 0)):
        b = B.paged_batch(z, z, z, n_seq, n_rows, 1)
        be.paged_attention(B.paged_attention_desc(c, b, z, z, 1))
        be.paged_append(B.paged_append_desc(c, b, z, z, z, z, 1))
    be.sample(B.sample_desc(z, B.FP32, 0, 5, z))
    be.sync()


# ---------------------------------------------------------------------------------------------- sample
def plain_sample(x, t, k, p, least, u):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    if x.max() == np.inf:
        x = np.where(x == np.inf, 0.0, -np.inf)
    with np.errstate(invalid="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / np.float64(t)))
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        sums = np.concatenate([[0.0], np.cumsum(w[order])])
        stay = sums[:-1] < np.float64(p) * sums[-1]
        stay[0] = True
        order = order[stay]
    if least > 0:
        order = order[w[order] >= min(np.float64(least), 1.0)]
    order = np.sort(order)
    sums = np.cumsum(w[order])
    at = int(np.searchsorted(sums, np.float64(max(u, 0.0)) * sums[-1], side="right"))
    at = min(at, int(np.nonzero(w[order] > 0)[0][-1]))
    return int(order[at]), float(w[order][at] / sums[-1])


def check_sample(be, dev, x, t=None, k=None, p=None, least=None, u=None, stride=None, offset=0):
    n, v = x.shape
    store = np.full(n * (stride or v) + offset, 50.0, dtype=x.dtype)
    for r in range(n):
        store[offset + r * (stride or v):][:v] = x[r]
    arrays = {"temperature": (t, np.float32), "top_k": (k, np.int32), "top_p": (p, np.float32), "min_p": (least, np.float32), "uniform": (u, np.float32)}
    host = {name: None if a is None else np.broadcast_to(np.asarray(a, dtype=dt), (n,)).copy() for name, (a, dt) in arrays.items()}
    ids, probs = np.full(n + 1, -77, dtype=np.int32), np.full(n + 1, -77, dtype=np.float32)
    pi, pp = dev(ids), dev(probs)
    d = B.sample_desc(dev(store) + offset * x.itemsize, B.FP32 if x.dtype == np.float32 else B.FP16, n, v, pi, probs=pp, row_stride=stride, **{m: None if a is None else dev(a) for m, a in host.items()})
    be.sample(d)
    got_i, got_p = dev.back(pi, ids), dev.back(pp, probs)
    default = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "uniform": 0.0}
    for r in range(n):
        with np.errstate(over="ignore"):
            want = plain_sample(x[r], *(default[m] if host[m] is None else host[m][r] for m in ("temperature", "top_k", "top_p", "min_p", "uniform")))
        assert got_i[r] == want[0], (r, got_i[r], want)
        assert abs(got_p[r] - want[1]) <= 2.0 ** -23 * want[1]                        # one rounding to f32, weights to 2^-40
    assert got_i[n] == -77 and got_p[n] == -77


@pytest.mark.parametrize("v", [1, 2, 31, 100, 1000, 4097, 32000, 50001])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_sample_settings(be, dev, v, dtype):
    rng = np.random.default_rng(v)
    n = 24
    x = (3 * rng.standard_normal((n, v))).astype(dtype)
    u = rng.random(n).astype(np.float32)
    r = np.arange(n)
    check_sample(be, dev, x, u=u)
    check_sample(be, dev, x, t=np.where(r % 3 == 0, 0, 0.5 + r / 20), u=u)
    check_sample(be, dev, x, t=0.8, k=r * r, u=u)
    check_sample(be, dev, x, t=1.1, p=(r + 1) / n, u=u)
    check_sample(be, dev, x, least=r / n, u=u)
    check_sample(be, dev, x, t=0.3 + r / 10, k=np.where(r % 2, 0, 40), p=np.where(r % 3, 0.9, 1.0), least=np.where(r % 5, 0.02, 0), u=u, stride=v + 3, offset=1)


def test_sample_many_candidates(be, dev):
    """Candidates that do not fit a list: a large top_k, flat rows, ties by the thousand."""
    rng = np.random.default_rng(3)
    u = rng.random(6).astype(np.float32)
    x = (2 * rng.standard_normal((6, 20000))).astype(np.float32)
    check_sample(be, dev, x, k=[1023, 1024, 1025, 5000, 19999, 20000], u=u)
    check_sample(be, dev, x, k=[1023, 1024, 1025, 5000, 19999, 20000], p=0.6, least=1e-4, u=u)
    check_sample(be, dev, 1e-3 * x, p=[0.01, 0.2, 0.5, 0.9, 0.999, 0.3], t=3.0, u=u)
    ties = np.round(x)
    check_sample(be, dev, ties, p=[0.01, 0.25, 0.5, 0.9, 0.999, 0.3], u=u)
    check_sample(be, dev, ties, k=[1, 2, 500, 3000, 9000, 15000], u=u)
    check_sample(be, dev, np.zeros_like(x), p=0.5, u=u)
    check_sample(be, dev, np.zeros_like(x), k=7, u=u)
    check_sample(be, dev, np.zeros_like(x), k=3000, p=0.5, least=0.5, u=u)


def test_sample_what_is_not_finite(be, dev):
    inf, nan = np.inf, np.nan
    rows = [[1, 2, nan, 0], [-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [-inf, 3, -inf, 3], [inf, 1, inf, -inf], [inf, nan, inf, inf], [-1e30, -1e30, 1e30, 1e30], [3e38, -3e38, 3e38, 0]]
    x = np.array(rows, dtype=np.float32)
    for u in (0.0, 0.4, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, -1.0, nan):
        check_sample(be, dev, x, u=0.0 if u != u else u) if u == u else None
        for extra in ({}, {"t": 0.0}, {"t": 1e-3}, {"t": 1e3}, {"k": 1}, {"k": 3, "p": 0.5}, {"p": 0.0}, {"p": 0.7}, {"least": 1.0}, {"least": 5.0}):
            check_sample(be, dev, x, u=0.0 if u != u else u, **extra)


def test_sample_large_vocabulary(be, dev):
    """Slices that do not stay in shared memory."""
    rng = np.random.default_rng(4)
    x = (3 * rng.standard_normal((2, (1 << 20) - 5))).astype(np.float32)
    u = rng.random(2).astype(np.float32)
    for k in ({}, {"t": 0.0}, {"k": 50, "p": 0.9}, {"p": 0.8}, {"least": 0.01}):
        check_sample(be, dev, x, u=u, **k)


def test_sample_draws_by_weight(be, dev):
    """Evenly spaced numbers draw each token by its share."""
    x = np.log(np.array([0.5, 0.25, 0.125, 0.125], dtype=np.float64)).astype(np.float32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    ids = np.zeros(n, dtype=np.int32)
    pi = dev(ids)
    be.sample(B.sample_desc(dev(np.broadcast_to(x, (n, 4)).copy()), B.FP32, n, 4, pi, uniform=dev(u)))
    count = np.bincount(dev.back(pi, ids), minlength=4)
    assert np.abs(count - np.array([2048, 1024, 512, 512])).max() <= 1


# ---------------------------------------------------------------------------------------------- together
def test_a_serving_loop(be, dev):
    """Requests of different lengths come in chunks beside running ones: append, attend, sample, feed the token back; against one plain cache a request."""
    rng = np.random.default_rng(21)
    h, h_kv, hd, v, page = 4, 2, 64, 500, 16
    d, width = 128, (h + 2 * h_kv) * hd
    embed, w_qkv, w_out = rng.standard_normal((v, d)), rng.standard_normal((d, width)) * d ** -0.5, rng.standard_normal((h * hd, v)) * 0.2
    prompts = [rng.integers(0, v, n).tolist() for n in (37, 5, 1, 90)]
    total, n_seq = 128, len(prompts)
    pool = Pool(rng, [total] * n_seq, h_kv, hd, page)
    pk, pv, pt = dev(pool.k), dev(pool.v), dev(pool.table)
    done, history = [0] * n_seq, [([], []) for _ in prompts]
    for step in range(12):
        rows = [min(32, len(t) - n) for t, n in zip(prompts, done)]                    # chunks of at most 32
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        n_kv = np.array([n + r for n, r in zip(done, rows)], dtype=np.int32)
        x = np.concatenate([embed[t[n:n + r]] for t, n, r in zip(prompts, done, rows)]) @ w_qkv
        x = x.astype(np.float32)
        px, n_rows = dev(x), int(starts[-1])
        pq, po = dev(np.zeros((n_rows, h, hd), np.float16)), dev(np.zeros((n_rows, h, hd), np.float32))
        batch = B.paged_batch(dev(starts), dev(n_kv), pt, n_seq, n_rows, pool.table.shape[1], max(rows))
        cache = pool.cache(pk, pv)
        be.paged_append(B.paged_append_desc(cache, batch, px, px + 4 * h * hd, px + 4 * (h + h_kv) * hd, pq, h, row_stride=width))
        be.paged_attention(B.paged_attention_desc(cache, batch, pq, po, h, out_type=B.FP32))
        out = dev.back(po, np.zeros((n_rows, h, hd), np.float32))
        for s in range(n_seq):
            a, b = starts[s], starts[s + 1]
            full = x[a:b].reshape(-1, h + 2 * h_kv, hd).astype(np.float64)
            turned = plain_rope(full, np.arange(done[s], n_kv[s]), B.ROPE_PAIRS, hd, 10000.0, 1.0)
            history[s][0].extend(turned[:, h:h + h_kv])
            history[s][1].extend(full[:, h + h_kv:])
            want, off = plain_attention(turned[:, :h], np.array(history[s][0]), np.array(history[s][1]), done[s], hd ** -0.5, True, 0, np.ones(n_kv[s], dtype=bool))
            # Q, K and V were rounded to fp16 on their way: a score is off by 2 x 2^-11 of the sum of its products' sizes, a probability by twice that, a value by 2^-11
            size = hd ** -0.5 * np.abs(turned[:, :h]).sum(-1).max() * np.abs(np.array(history[s][0])).max()
            assert np.all(np.abs(out[a:b] - want) <= off + (2 * 2 * 2.0 ** -11 * size + 2.0 ** -10) * np.abs(np.array(history[s][1])).max())
        last = starts[1:] - 1
        logits = (out.reshape(n_rows, -1)[last] @ w_out).astype(np.float32)
        u = rng.random(n_seq).astype(np.float32)
        pi = dev(np.zeros(n_seq, np.int32))
        be.sample(B.sample_desc(dev(logits), B.FP32, n_seq, v, pi, uniform=dev(u), top_k=dev(np.full(n_seq, 20, np.int32)), temperature=dev(np.full(n_seq, 0.8, np.float32))))
        ids = dev.back(pi, np.zeros(n_seq, np.int32))
        for s in range(n_seq):
            assert ids[s] == plain_sample(logits[s], np.float32(0.8), 20, 1.0, 0.0, u[s])[0]
            done[s] = int(n_kv[s])
            if done[s] == len(prompts[s]):
                prompts[s].append(int(ids[s]))
    assert all(len(t) > n for t, n in zip(prompts, (37, 5, 1, 90)))


def test_results_do_not_depend_on_programmatic_launch(dev):
    """Append, attention and sampling back to back on one stream, with and without kernels that start beside their predecessors."""
    got = []
    for pdl in (True, False):
        b = B.B200Backend(0, use_pdl=pdl)
        d, rng = Device(b), np.random.default_rng(31)
        pool = Pool(rng, [300, 20, 90], 2, 64, 16, fill=0.0)
        pool.put(0, *rng.standard_normal((2, 299, 2, 64)).astype(np.float16))
        cache = pool.cache(d(pool.k), d(pool.v))
        batch = B.paged_batch(d(np.array([0, 1, 21, 60], np.int32)), d(np.array([300, 20, 39], np.int32)), d(pool.table), 3, 60, pool.table.shape[1])
        x = d(rng.standard_normal((60, 8 * 64)).astype(np.float32))
        q, o, ids = d(np.zeros((60, 4, 64), np.float16)), np.zeros((60, 4 * 64), np.float32), np.zeros(60, np.int32)
        po, pi = d(o), d(ids)
        for _ in range(20):
            b.paged_append(B.paged_append_desc(cache, batch, x, x + 4 * 256, x + 4 * 384, q, 4, row_stride=512))
            b.paged_attention(B.paged_attention_desc(cache, batch, q, po, 4, out_type=B.FP32))
            b.sample(B.sample_desc(po, B.FP32, 60, 256, pi))
        got.append((d.back(po, o), d.back(pi, ids)))
        d.free()
        b.close()
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


# ---------------------------------------------------------------------------------------------- a model's decoding loop with drawn tokens
def sampled_model(path, kq=False, nothing=False):
    cfg = gguf_io.LlamaConfig(n_layer=2, d_model=256, n_head=2, n_ff=512, n_vocab=400, weight_std=0.06,
                              **(dict(wtype=quants.Q4_K, overrides={"attn_v": quants.Q6_K, "ffn_down": quants.Q6_K, "output": quants.Q6_K}) if kq else {}))
    gguf_io.make_llama_gguf(path, cfg, seed=61)
    if nothing:                                                                       # every scale of the output matrix is NaN: so are all logits
        blocks = bytes(gguf_io.read_gguf(path)[1]["output.weight"][2])
        raw = np.memmap(path, dtype=np.uint8, mode="r+")
        at = raw.tobytes().find(blocks)
        raw[at:at + len(blocks)].reshape(-1, 18)[:, 0:2] = (0x00, 0x7e)
        raw.flush()
    return cfg


def drawn(logits, uniform, temperature, top_k, top_p, min_p):
    return np.array([plain_sample(x, np.float32(temperature), top_k, np.float32(top_p), np.float32(min_p), u)[0] for x, u in zip(logits, uniform)])


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("kq", [False, True])
def test_model_decode_sampled(use_graph, kq, tmp_models):
    path = str(tmp_models / f"sampled{int(kq)}.gguf")
    cfg = sampled_model(path, kq)
    rng = np.random.default_rng(5)
    prompt, n_steps = rng.integers(3, cfg.n_vocab, size=9), 20
    b = B.B200Backend(0, use_graph=use_graph)
    m = B.LlamaModel(b, path, n_ctx=64)
    first = int(np.argmax(m.eval(prompt, 0)))
    greedy = m.decode(first, 9, n_steps, want_logits=True)
    for settings in ({}, {"temperature": 0.0}):                                       # (temperature 1 and no uniform numbers: the first index with any weight)
        ids, logits = m.decode_sampled(first, 9, n_steps, want_logits=True, **settings)
        if settings:
            assert np.array_equal(ids, greedy[0]) and np.array_equal(logits, greedy[1])
        else:
            assert np.array_equal(ids, drawn(logits, np.zeros(n_steps), 1, 0, 1, 0))
    for t, k, p, least in ((1.0, 0, 1.0, 0.0), (0.7, 30, 0.9, 0.01), (3.0, 0, 0.95, 0.0)):
        u = rng.random(n_steps).astype(np.float32)
        ids, logits = m.decode_sampled(first, 9, n_steps, uniform=u, temperature=t, top_k=k, top_p=p, min_p=least, want_logits=True)
        assert np.array_equal(ids, drawn(logits, u, t, k, p, least))
        again = m.decode_sampled(first, 9, n_steps, uniform=u, temperature=t, top_k=k, top_p=p, min_p=least)[0]
        assert np.array_equal(ids, again)
        last, feed = [], [first, *ids[:-1]]
        for s, token in enumerate(feed):                                              # each step's logits are those of the tokens that were drawn
            last.append(m.eval(np.array([token], dtype=np.int32), 9 + s))
        assert np.array_equal(np.array(last), logits)
        m.eval(prompt, 0)
    again = m.decode(first, 9, n_steps)[0]
    assert np.array_equal(again, greedy[0])
    m.close()
    b.close()


@pytest.mark.parametrize("n_seq", [1, 5, 18])
def test_model_decode_batch_sampled(n_seq, tmp_models):
    """Every sequence draws what it would draw alone, with its own settings; batches on the mat-vec passes and on the GEMMs."""
    path = str(tmp_models / "sampled0.gguf")
    cfg = sampled_model(path)
    rng = np.random.default_rng(n_seq)
    n_prompt, n_steps = 11, 12
    t, k = (0.4 + rng.random(n_seq)).astype(np.float32), rng.integers(0, 50, size=n_seq).astype(np.int32)
    u = rng.random((n_steps, n_seq)).astype(np.float32)
    t[0] = 0
    b = B.B200Backend(0)
    m = B.LlamaModel(b, path, n_ctx=64)
    m.set_sequences(n_seq)
    prompts, first, want = rng.integers(3, cfg.n_vocab, size=(n_seq, n_prompt)), [], []
    for c in range(n_seq):
        m.select_sequence(c)
        first.append(int(np.argmax(m.eval(prompts[c], 0))))
        want.append(m.decode_sampled(first[c], n_prompt, n_steps, uniform=u[:, c], temperature=t[c], top_k=k[c], top_p=0.9, want_logits=True))
    ids, logits = m.decode_batch_sampled(first, n_prompt, n_steps, uniform=u, temperature=t, top_k=k, top_p=0.9, want_logits=True)
    for c in range(n_seq):
        assert np.array_equal(ids[:, c], want[c][0]) and np.array_equal(logits[:, c], want[c][1]), c
        assert np.array_equal(ids[:, c], drawn(logits[:, c], u[:, c], t[c], k[c], 0.9, 0)), c
    m.close()
    b.close()


def test_model_decode_sampled_with_nothing_to_draw(tmp_models):
    path = str(tmp_models / "sampled_nan.gguf")
    sampled_model(path, nothing=True)
    b = B.B200Backend(0)
    m = B.LlamaModel(b, path, n_ctx=32)
    m.set_sequences(2)
    for c in range(2):
        m.select_sequence(c)
        assert np.isnan(m.eval(np.array([5, 6], dtype=np.int32), 0)).all()
        assert np.array_equal(m.decode_sampled(7, 2, 3)[0], [-1] * 3)
    assert np.array_equal(m.decode_batch_sampled([7, 8], 2, 3)[0], [[-1, -1]] * 3)
    m.close()
    b.close()


def test_model_decode_sampled_refuses(tmp_models):
    path = str(tmp_models / "sampled0.gguf")
    cfg = sampled_model(path)
    b = B.B200Backend(0)
    m = B.LlamaModel(b, path, n_ctx=32)
    m.set_sequences(2)
    for bad in (lambda: m.decode_sampled(5, 30, 3), lambda: m.decode_sampled(cfg.n_vocab, 0, 3), lambda: m.decode_batch_sampled([1, 2, 3], 0, 2), lambda: m.decode_batch_sampled([1, -2], 0, 2),
                lambda: m.decode_batch_sampled([1, 2], -1, 2)):
        with pytest.raises(B.SpybError):
            bad()
    ids = np.zeros(3, np.int32)
    assert b._l.spyb_model_decode_sampled(m.h, 5, 0, 3, None, B._np_ptr(ids), None) != B.SUCCESS
    assert m.decode_sampled(5, 0, 3, temperature=0.0)[0].tolist() == m.decode(5, 0, 3)[0].tolist()
    m.close()
    b.close()


# ---------------------------------------------------------------------------------------------- far pages, several backends
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_sequences_that_share_pages(be, dev, hd):
    rng = np.random.default_rng(hd + 1)
    check_attention(be, dev, rng, [1, 1, 1, 1], [200, 130, 64, 300], 4, 2, hd, 16, share=4, max_rows=1)
    check_attention(be, dev, rng, [150, 1, 40, 7], [200, 130, 104, 300], 4, 2, hd, 16, share=4)


@pytest.mark.parametrize("hd,h", [(128, 2), (64, 4), (96, 2)])
def test_pages_beyond_32_bits(be, dev, hd, h):
    """Elements more than 2^32 behind the pool's first: the same bits as with pages side by side."""
    import torch

    rng = np.random.default_rng(hd)
    n, page, far = 40, 16, (1 << 31) + 64
    pool = Pool(rng, [n], 1, hd, page)
    pool.table[0, :3] = [2, 0, 1]
    x = rng.standard_normal((n, (h + 2) * hd)).astype(np.float32)
    q = rng.standard_normal((n, h, hd)).astype(np.float16)
    store = torch.full((2 * far + (1 << 18),), 3.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    px, pq, pt, pk, pv = dev(x), dev(q), dev(pool.table[:, :3].copy()), dev(np.full(3 * page * hd, 3, np.float16)), dev(np.full(3 * page * hd, 3, np.float16))
    near = B.paged_cache(pk, pv, 3, page, 1, hd)
    base = store.data_ptr()
    got = []
    for c in (near, B.paged_cache(base, base + (1 << 18), 3, page, 1, hd, strides=(far, hd, page * hd))):
        batch = B.paged_batch(dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), pt, 1, n, 3)
        turned = dev(np.zeros((n, h, hd), np.float16))
        be.paged_append(B.paged_append_desc(c, batch, px, px + 4 * h * hd, px + 4 * (h + 1) * hd, turned, h, row_stride=(h + 2) * hd))
        out = np.zeros((n + 1, h, hd), np.float32)
        po = dev(out)
        be.paged_attention(B.paged_attention_desc(c, batch, pq, po, h, out_type=B.FP32))
        one = B.paged_batch(dev(np.array([0, 1], np.int32)), dev(np.array([n], np.int32)), pt, 1, 1, 3)
        be.paged_attention(B.paged_attention_desc(c, one, pq, po + 4 * n * h * hd, h, out_type=B.FP32))
        got.append(dev.back(po, out))
    assert got[0].any(axis=(1, 2)).all() and np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
    k = np.empty(3 * page * hd, np.float16)
    assert np.array_equal(store[2 * far:2 * far + page * hd].cpu().numpy(), dev.back(pk, k)[2 * page * hd:])


def test_two_backends_at_once(dev):
    import threading

    rng = np.random.default_rng(9)
    pool = Pool(rng, [700, 60, 3000], 2, 128, 16)
    for s, n in enumerate((700, 60, 3000)):
        pool.put(s, *rng.standard_normal((2, n, 2, 128)).astype(np.float16))
    q = rng.standard_normal((141, 8, 128)).astype(np.float16)
    x = rng.standard_normal((5, 40000)).astype(np.float32)
    results = [None] * 3

    def work(i):
        b = B.B200Backend(0)
        d = Device(b)
        batch = B.paged_batch(d(np.array([0, 130, 140, 141], np.int32)), d(np.array([700, 60, 3000], np.int32)), d(pool.table), 3, 141, pool.table.shape[1])
        po, ids = d(np.zeros(q.shape, np.float16)), d(np.zeros(5, np.int32))
        attention = B.paged_attention_desc(pool.cache(d(pool.k), d(pool.v)), batch, d(q), po, 8)
        sample = B.sample_desc(d(x), B.FP32, 5, 40000, ids, uniform=d(np.linspace(0, 0.9, 5).astype(np.float32)), top_p=d(np.full(5, 0.9, np.float32)))
        for _ in range(100):
            b.paged_attention(attention)
            b.sample(sample)
        results[i] = (d.back(po, np.zeros(q.shape, np.float16)), d.back(ids, np.zeros(5, np.int32)))
        d.free()
        b.close()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    work(2)
    assert all(np.array_equal(r[0], results[2][0]) and np.array_equal(r[1], results[2][1]) for r in results[:2])


# ---------------------------------------------------------------------------------------------- what the descriptors allow at their ends
@pytest.mark.parametrize("rows", [5, 8, 150])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30 + 5, 2 ** 30])
def test_windows_as_long_as_an_int_can_say(be, dev, rows, window):
    """Rows in front of position 0 beside a window that hides nothing: the rows behind see all of their past."""
    rng = np.random.default_rng(rows)
    check_attention(be, dev, rng, [rows, 1, rows], [2, 300, rows - 4], 4, 2, 64, 16, window=window)
    check_attention(be, dev, rng, [rows], [rows // 2], 4, 4, 128, 16, window=window)


def test_numbers_of_steps_beyond_32_bits_are_refused(tmp_models):
    """n_past + n_steps that leaves 32 bits is beyond the context too."""
    path = str(tmp_models / "sampled0.gguf")
    sampled_model(path)
    b = B.B200Backend(0)
    m = B.LlamaModel(b, path, n_ctx=32)
    m.set_sequences(2)
    most, ids, first = 2 ** 31 - 1, np.zeros(8, np.int32), np.array([1, 2], np.int32)
    how, keep = B.LlamaModel._sampling(1, 1, None, 1.0, None, None, None)
    i, f = B._np_ptr(ids), B._np_ptr(first)
    for past in (1, 32, most):
        assert b._l.spyb_model_decode(m.h, 5, past, most, i, None) != B.SUCCESS
        assert b._l.spyb_model_decode_sampled(m.h, 5, past, most, B.C.byref(how), i, None) != B.SUCCESS
        assert b._l.spyb_model_decode_batch(m.h, f, 2, past, most, i, None) != B.SUCCESS
        assert b._l.spyb_model_decode_batch_sampled(m.h, f, 2, past, most, B.C.byref(how), i, None) != B.SUCCESS
        assert b._l.spyb_model_eval(m.h, f, most, past, None) != B.SUCCESS
    with pytest.raises(B.SpybError):
        m.decode(5, 31, 2)
    assert m.decode_sampled(5, 31, 1, temperature=0.0)[0].tolist() == m.decode(5, 31, 1)[0].tolist()
    m.close()
    b.close()


@pytest.mark.parametrize("t", [1.5e-45, 1e-38, 3e-31, 1e-20, 1e20, 1e31, 3e38, np.inf])
def test_sample_temperatures_of_all_sizes(be, dev, t):
    """Logits as many times smaller or larger: weights are those of logit / temperature at ordinary sizes."""
    rng = np.random.default_rng(17)
    n, v = 6, 700
    scale = min(max(t, 2.0 ** -149), 1e38)
    x = np.clip(scale * np.clip(2 * rng.standard_normal((n, v)), -3.3, 3.3), -3.3e38, 3.3e38).astype(np.float32)
    x[0, ::3] = -np.inf
    u = (0.05 + 0.9 * rng.random(n)).astype(np.float32)
    for extra in ({}, {"k": 5}, {"k": 300}, {"k": 650, "p": 0.9}, {"p": 0.3}, {"p": 0.95}, {"least": 0.1}):
        check_sample(be, dev, x, t=t, u=u, **extra)


def check_low(be, dev, x, u, t, **settings):
    """check_sample for numbers near 0: shares down to the smallest that 64 bits hold, rounded to f32."""
    n, v = x.shape
    ids, probs = np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.float32)
    pi, pp = dev(ids), dev(probs)
    types = {"top_k": np.int32}
    host = {m: np.broadcast_to(np.asarray(a, dtype=types.get(m, np.float32)), (n,)).copy() for m, a in dict(settings, temperature=t).items()}
    pu = None if u is None else dev(np.broadcast_to(np.float32(u), (n,)).copy())
    be.sample(B.sample_desc(dev(x), B.FP32 if x.dtype == np.float32 else B.FP16, n, v, pi, probs=pp, uniform=pu, **{m: dev(a) for m, a in host.items()}))
    got_i, got_p = dev.back(pi, ids), dev.back(pp, probs)
    full = dict({"top_k": np.zeros(n, int), "top_p": np.ones(n), "min_p": np.zeros(n)}, **host)
    for r in range(n):
        want = plain_sample(x[r], full["temperature"][r], full["top_k"][r], full["top_p"][r], full["min_p"][r], np.float32(u or 0))
        assert got_i[r] == want[0], (r, got_i[r], want, u, settings)
        assert abs(got_p[r] - want[1]) <= 2.0 ** -23 * want[1] + 2.0 ** -150          # (half a step of the smallest f32)


@pytest.mark.parametrize("v,dtype", [(50, np.float32), (3000, np.float16), (32000, np.float32), (50001, np.float16), ((1 << 20) - 5, np.float32)])
@pytest.mark.parametrize("t", [0.3, 0.5, 1.0, 0.01])
def test_sample_uniform_numbers_near_zero(be, dev, v, dtype, t):
    """A number of 0 falls on the first token that has any weight in 64 bits, however small; numbers near it among weights that are no unit of the integers."""
    rng = np.random.default_rng(v)
    n = 4 if v < 10 ** 6 else 1
    x = (3 * rng.standard_normal((n, v))).astype(dtype)
    x[0, 2:v // 3] -= 40
    for u in (None, 0.0, -1.0, 1e-30, 1e-12, 1e-9, 3e-8, 2.0 ** -24, 9e-7):
        for s in ({}, {"top_k": 7}, {"top_k": min(v - 1, 700)}, {"top_k": v // 2, "min_p": 1e-25}, {"top_p": 0.9}, {"top_p": 1 - 2.0 ** -24}, {"min_p": 1e-20}, {"min_p": 1e-5}, {"top_k": 40, "top_p": 0.95, "min_p": 0.01}):
            if v > 10 ** 6 and (u not in (None, 1e-12) or "top_k" in s and s["top_k"] > 7):
                continue
            check_low(be, dev, x, u, t, **s)


def test_sample_nothing_but_far_tokens_in_front(be, dev):
    """Shares of 1e-30 and of nothing in front of the largest; equal tokens; +inf; -inf."""
    x = np.array([[-600, 0, 1], [-2000, -1000, 0], [-np.inf, -69, 0], [5, 5, 5], [1, np.inf, np.inf], [np.nan, -745, 0]], dtype=np.float32)
    for u in (None, 0.0, 1e-38, 1e-31, 9e-7):
        for s in ({}, {"top_k": 2}, {"top_p": 0.5}, {"min_p": 1e-35}, {"min_p": 1.0}):
            check_low(be, dev, x, u, 1.0, **s)
            check_low(be, dev, x, u, np.inf, **s)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [3, 5, 12])
def test_rows_of_nobody_decide_nothing(be, dev, hd, group):
    """The same bits whatever an earlier kernel left in shared memory (a tile of 128 rows holds whole tokens: groups of 5 leave three rows over), and whatever Q the padding and
    the other sequences have."""
    rng = np.random.default_rng(hd + group)
    rows, n_kv = [130, 9, 61], [900, 400, 61]
    pool = Pool(rng, n_kv, 1, hd, 16, fill=0.0)
    for s, n in enumerate(n_kv):
        pool.put(s, *rng.standard_normal((2, n, 1, hd)).astype(np.float16))
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    q = rng.standard_normal((starts[-1] + 40, group, hd)).astype(np.float16)
    c, pt, pn, ps = pool.cache(dev(pool.k), dev(pool.v)), dev(pool.table), dev(np.array(n_kv, np.int32)), dev(starts)
    out = np.zeros(q.shape, np.float32)

    def run(q):
        po = dev(out)
        be.paged_attention(B.paged_attention_desc(c, B.paged_batch(ps, pn, pt, 3, len(q), pool.table.shape[1]), dev(q), po, group, out_type=B.FP32))
        return dev.back(po, out).view(np.uint32)

    def leave(size):                                         # full tiles of 128 rows with scores of all sizes, in every CTA and buffer
        big = np.full((4096, 4, hd), size, np.float16) * rng.choice([-1, 1], (4096, 4, hd)).astype(np.float16)
        b = B.paged_batch(dev(np.array([0, 4096], np.int32)), dev(np.array([900], np.int32)), pt, 1, 4096, pool.table.shape[1])
        be.paged_attention(B.paged_attention_desc(c, b, dev(big), dev(np.zeros(big.shape, np.float16)), 4, causal=False))

    leave(0.0)
    first = run(q)
    for size in (1.0, 30.0, 3000.0):
        leave(size)
        assert np.array_equal(run(q)[:starts[-1]], first[:starts[-1]]), size
    for size in (0.0, 30.0, 3000.0):
        other = q.copy()
        other[starts[1]:] = size * rng.standard_normal(other[starts[1]:].shape)
        assert np.array_equal(run(other)[:starts[1]], first[:starts[1]]), size
        other[starts[2]:] = q[starts[2]:]
        other[starts[3]:] = size
        assert np.array_equal(run(other)[starts[2]:starts[3]], first[starts[2]:starts[3]]), size


def test_warps_that_come_late_change_nothing():
    """The warps that check V wait for phases of a ring that others drive: however late they come, none is over before they have seen it."""
    b = B.B200Backend(0)
    assert b.paged_selftest_late(1, 1_000_000_000) == 0
    b.close()


@pytest.mark.parametrize("who", [2, 3])
def test_copies_that_come_too_late_are_reported_and_leave_nothing(be, dev, who):
    """Waits of 2 ms for a copy that comes after 6: they give up, the kernel ends by itself with the copy landed, the status says so, and later launches on the backend are right."""
    b = B.B200Backend(0)
    assert b.paged_selftest_late(who, 2_000_000) == 7
    assert b.paged_selftest_late(1, 1_000_000_000) == 0
    d = Device(b)
    rng = np.random.default_rng(who)
    check_attention(b, d, rng, [150, 1, 40], [700, 2000, 90], 4, 2, 128, 16)
    check_attention(b, d, rng, [150, 1, 40], [700, 2000, 90], 6, 2, 64, 16)
    d.free()
    b.close()


def test_first_calls_beside_a_stream_capture(dev):
    """A backend's first attention (both kernels) and sampling while another library captures a stream: nothing is allocated in the calls."""
    import torch

    rng = np.random.default_rng(41)
    pool = Pool(rng, [700, 90], 2, 64, 16, fill=0.0)
    for s, n in enumerate((700, 90)):
        pool.put(s, *rng.standard_normal((2, n, 2, 64)).astype(np.float16))
    q = rng.standard_normal((141, 4, 64)).astype(np.float16)
    b = B.B200Backend(0)
    d = Device(b)
    cache = pool.cache(d(pool.k), d(pool.v))
    many = B.paged_batch(d(np.array([0, 140, 141], np.int32)), d(np.array([700, 90], np.int32)), d(pool.table), 2, 141, pool.table.shape[1])
    one = B.paged_batch(d(np.array([0, 1], np.int32)), d(np.array([700], np.int32)), d(pool.table), 1, 1, pool.table.shape[1])
    pq, po, pi, out = d(q), d(np.zeros(q.shape, np.float32)), d(np.zeros(141, np.int32)), np.zeros(q.shape, np.float32)
    x = torch.zeros(1000, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        b.paged_attention(B.paged_attention_desc(cache, many, pq, po, 4, out_type=B.FP32))
        b.paged_attention(B.paged_attention_desc(cache, one, pq, po, 4, out_type=B.FP32))
        b.sample(B.sample_desc(po, B.FP32, 141, 256, pi))
    during = d.back(po, out)
    b.paged_attention(B.paged_attention_desc(cache, many, pq, po, 4, out_type=B.FP32))
    b.paged_attention(B.paged_attention_desc(cache, one, pq, po, 4, out_type=B.FP32))
    assert during.any() and np.array_equal(during, d.back(po, out))
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all()
    d.free()
    b.close()


@pytest.mark.parametrize("vocab", [1000, 1 << 17, (1 << 17) + 1, 1 << 20])
@pytest.mark.parametrize("c_largest", [0.0, 1.0, -30.0, 640.0, 959.9, -959.9, 960.1, -960.1, 5000.0, -3e5])
def test_weights_of_the_sampler(be, vocab, c_largest):
    """2^S exp((x - largest) / T): to 2^-31.8 of itself (as derived beside the code) and a unit, on both sides of the switch to 64 bits at largest / T log2(e) = 960."""
    bits = min(45, 62 - int(np.ceil(np.log2(vocab))))
    rng = np.random.default_rng(int(abs(c_largest)) + vocab)
    for t in (1.0, 0.37, 1e-3, 2.5e4, 1e-35, 1e33):
        t = np.float32(t)
        largest = np.float32(c_largest * np.log(2.0) * float(t))
        x = (float(largest) - float(t) * np.concatenate([np.linspace(0, 45, 20000), 36 * rng.random(100000), [0, 1e-8, 60, 1e4]])).astype(np.float32)
        x = np.append(np.minimum(x, largest), -np.inf).astype(np.float32)
        w = be.sample_weights(x, largest, t, vocab)
        z = (x.astype(np.longdouble) - np.longdouble(largest)) / np.longdouble(t)
        want = np.exp(z) * np.longdouble(2.0) ** bits
        err = np.abs(w.astype(np.longdouble) - want)
        assert (err <= want * np.longdouble(2.0) ** -31.8 + 1).all(), (t, float((np.maximum(err - 1, 0) / np.maximum(want, 1)).max()))
        assert w[x == largest].min() == w.max() == 2 ** bits and w[-1] == 0


# ---------------------------------------------------------------------------------------------- every position, by counting
def check_counts(be, dev, rng, rows, n_kv, h, h_kv, hd, page, causal=True, window=0, max_rows=0, q_pad=0, out_pad=0, out=np.float32):
    """All keys 0: a row's output is the mean of the values that it sees. Values are small whole numbers, so that every sum on the way (below 2^24) is exact and the output is one
    quotient, rounded to f32 twice (the reciprocal and the product: 2^-23 of it): a position that is left out, seen twice or another head's shows by at least one part in its number."""
    n_kv = [max(r, n) for r, n in zip(rows, n_kv)]
    pool = Pool(rng, n_kv, h_kv, hd, page, fill=0.0)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n_rows = int(starts[-1])
    q_stride, out_stride = h * hd + q_pad, h * hd + out_pad
    q = np.full((n_rows, q_stride), np.nan, np.float16)
    q[:, :h * hd] = rng.standard_normal((n_rows, h * hd))
    out0 = np.full((n_rows, out_stride), 7.5, out)
    sums = []
    for s, n in enumerate(n_kv):
        v = rng.integers(-9, 10, (n, h_kv, hd))
        pool.put(s, np.zeros(v.shape, np.float16), v.astype(np.float16))
        sums.append(np.concatenate([np.zeros((1, h_kv, hd), np.int64), np.cumsum(v, axis=0)]))
        assert np.abs(sums[-1]).max() + 9 * n < 2 ** 24
    po = dev(out0)
    batch = B.paged_batch(dev(starts), dev(np.array(n_kv, np.int32)), dev(pool.table), len(rows), n_rows, pool.table.shape[1], max_rows)
    be.paged_attention(B.paged_attention_desc(pool.cache(dev(pool.k), dev(pool.v)), batch, dev(q), po, h, out_type=B.FP32 if out == np.float32 else B.FP16, causal=causal, window=window,
                                              q_stride=q_stride, out_stride=out_stride))
    got = dev.back(po, out0)
    assert (got[:, h * hd:] == 7.5).all()                    # between the rows
    got = got[:, :h * hd].reshape(n_rows, h, hd).astype(np.float64)
    heads = np.arange(h) // (h // h_kv)
    for s, n in enumerate(n_kv):
        pos = np.arange(n - rows[s], n)
        hi = pos + 1 if causal else np.full(rows[s], n)
        lo = np.maximum(0, hi - window) if window else np.zeros(rows[s], int)
        total, count = (sums[s][hi] - sums[s][lo])[:, heads], (hi - lo)[:, None, None]
        want = total / count
        tol = np.abs(want) * 2.0 ** -23 if out == np.float32 else np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25
        assert (np.abs(got[starts[s]:starts[s + 1]] - want) <= tol).all(), s
        if out == np.float32 and rows[s]:                    # sixteen positions less, anywhere, would show
            at = rng.integers(0, max(1, n - 16), 20)
            for a in at:
                less = total[-1] - (sums[s][np.minimum(a + 16, hi[-1])] - sums[s][np.minimum(a, hi[-1])])[heads]
                assert lo[-1] > a or (np.abs(less / count[-1] - want[-1]) > tol[-1]).any()


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_every_position_of_long_contexts(be, dev, hd):
    """Items that all CTAs have a piece of: one K/V head, one row to a few."""
    rng = np.random.default_rng(hd)
    check_counts(be, dev, rng, [1], [40000], 2, 1, hd, 64, max_rows=1)
    check_counts(be, dev, rng, [1], [65537], 1, 1, hd, 24, max_rows=1)
    check_counts(be, dev, rng, [3, 1], [50001, 20011], 4, 1, hd, 16)
    check_counts(be, dev, rng, [7, 1, 30], [30000, 11, 9001], 5, 1, hd, 32)
    check_counts(be, dev, rng, [40], [9000], 2, 1, hd, 64)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("n_seq", [1, 2, 4, 5, 12, 13, 128, 129, 384, 385, 800])
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
    check_counts(be, dev, rng, rows.tolist(), n_kv, 2, 1, hd, 8, window=90)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_every_position_of_sequences_with_many_tiles(be, dev, hd):
    """More than 32 tiles of rows a sequence, which a CTA finds its place among in several rounds."""
    rng = np.random.default_rng(hd)
    check_counts(be, dev, rng, [1300, 2, 1100], [1400, 900, 1100], 2, 2, hd, 16)
    check_counts(be, dev, rng, [9000], [9100], 1, 1, hd, 64, window=700)
    check_counts(be, dev, rng, [2300, 700], [2300, 900], 8, 1, hd, 3)
    check_counts(be, dev, rng, [1200], [2000], 2, 1, hd, 16, causal=False)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("out", [np.float32, np.float16])
def test_rows_with_room_between_them(be, dev, hd, out):
    """Row strides of Q and of the output that are not the heads' width."""
    rng = np.random.default_rng(hd)
    for rows, n_kv in (([1, 1, 3], [300, 41, 90]), ([200, 1, 33], [900, 41, 33]), ([20], [6000])):
        check_counts(be, dev, rng, rows, n_kv, 4, 2, hd, 16, q_pad=8, out_pad=hd, out=out)
        check_counts(be, dev, rng, rows, n_kv, 3, 1, hd, 16, q_pad=2 * hd + 24, out_pad=8, out=out)


@pytest.mark.parametrize("hd", [64, 128])
def test_more_query_heads_than_a_tile_has_rows(be, dev, hd):
    rng = np.random.default_rng(hd)
    for group in (127, 128, 129, 300):
        check_counts(be, dev, rng, [1, 5, 20], [300, 41, 700], group, 1, hd, 16)
        check_attention(be, dev, rng, [1, 3], [130, 41], group, 1, hd, 16)
