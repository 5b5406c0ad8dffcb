"""A paged cache of keys and values: appending to it, and attention of new tokens over it, against the formulas in 64 bits.

Tolerances are bounds, element by element, from the magnitudes that enter a value: a sum of n products in fp32 is off by at most n * 2^-24 of the
sum of their magnitudes, exp by its argument's error, a weight that is two bfloat16 values by 2^-15, and each rounding to bfloat16 by 2^-8 of what
is rounded."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_attention import E32, STEP, from_bf16, to_bf16

pytestmark = pytest.mark.gpu


def stored(storage, a):
    return np.asarray(a, np.float32) if storage == "f32" else to_bf16(a)


def f64(a):
    return (a if a.dtype == np.float32 else from_bf16(a)).astype(np.float64)


def fn(br, stem, storage):
    return getattr(br.lib, "mi355_%s%s_dev" % (stem, "" if storage == "f32" else "_bf16"))


class Cache:
    """Sequences of the given lengths on pages in no order; entries behind a sequence's last page name no page at all."""

    def __init__(self, storage, kv, hd, page, lengths, seed=0, room=0, spread=1.0, values=True):
        self.storage, self.kv, self.hd, self.page, self.lengths = storage, kv, hd, page, list(lengths)
        rng = np.random.default_rng([seed, kv, hd, page])
        need = [-(-n // page) for n in lengths]
        self.n_pages, self.max_pages = sum(need) + 3, max(need) + room
        ids = rng.permutation(self.n_pages)
        self.pages = rng.choice(np.array([-1, self.n_pages, 2 ** 31 - 1, -2 ** 31], np.int64), (len(need), self.max_pages)).astype(np.int32)
        at = 0
        for i, n in enumerate(need):
            self.pages[i, :n] = ids[at:at + n]
            at += n
        shape = (self.n_pages, kv, page, hd)
        self.k, self.v = ((stored(storage, spread * rng.standard_normal(shape)) if values else stored(storage, np.full(shape, 3.0))) for _ in range(2))

    def to(self, br):
        self.kd, self.vd, self.pd = (br.DevArray.from_numpy(a) for a in (self.k, self.v, self.pages))
        return br.KvCache(self.kd.ptr, self.vd.ptr, self.pd.ptr, self.n_pages, self.page, len(self.pages), self.max_pages, self.kv, self.hd)

    def row(self, seq, pos):
        return int(self.pages[seq, pos // self.page]), pos % self.page

    def rows(self, which, seq, n):
        """[kv][n][hd] of positions that have a page, and which these are."""
        ok = [p for p in range(n) if 0 <= self.pages[seq, p // self.page] < self.n_pages]
        ids = self.pages[seq, np.array(ok, int) // self.page]
        return f64(which)[ids, :, np.array(ok, int) % self.page].transpose(1, 0, 2)


def attend(br, cache, q, seq, pos, heads, scale, fill=7.0, lse=True):
    """q: [batch][heads*hd][S]"""
    B, _, S = q.shape
    D = br.DevArray.from_numpy
    c, qd, pd = cache.to(br), D(q), D(np.asarray(pos, np.int32))
    sd = None if seq is None else D(np.asarray(seq, np.int32))
    o, l = D(stored(cache.storage, np.full(q.shape, fill))), D(np.full((B, heads, S), fill, np.float32))
    br.check(fn(br, "attn_paged", cache.storage)(C.byref(c), o.ptr, l.ptr if lse else None, qd.ptr, sd.ptr if sd else None, pd.ptr, heads, S, B, scale))
    return o.numpy(), l.numpy()


def expected(cache, q, seq, pos, heads, scale):
    """(o, bound of o, lse, bound of lse, columns that are tokens)"""
    B, _, S = q.shape
    hd, kv, G = cache.hd, cache.kv, heads // cache.kv
    eps, extra = STEP[cache.storage], 2.0 ** -15 if cache.storage == "bf16" else 0.0
    pos = np.asarray(pos).reshape(B, S)
    seq = np.arange(B * S).reshape(B, S) if seq is None else np.asarray(seq).reshape(B, S)
    o, ob, le, lb = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, heads, S)), np.zeros((B, heads, S))
    used = np.zeros((B, S), bool)
    for b in range(B):
        for s in range(S):
            i, p = int(seq[b, s]), int(pos[b, s])
            if not (0 <= i < len(cache.pages) and 0 <= p < cache.max_pages * cache.page):
                continue
            K, V = cache.rows(cache.k, i, p + 1), cache.rows(cache.v, i, p + 1)
            n = K.shape[1]
            if n == 0:
                continue
            used[b, s] = True
            for g in range(kv):
                for h in range(g * G, (g + 1) * G):
                    Q = f64(q)[b, h * hd:(h + 1) * hd, s]
                    z = scale * (K[g] @ Q)
                    dz = E32 * (hd + 6) * scale * (np.abs(K[g]) @ np.abs(Q))
                    m = z.max()
                    e = np.exp(z - m)
                    w = e / e.sum()
                    row = 2 * dz.max() + E32 * (n + 32 + 2 * np.abs(z).max())
                    o[b, h * hd:(h + 1) * hd, s] = w @ V[g]
                    ob[b, h * hd:(h + 1) * hd, s] = 1.01 * (w @ np.abs(V[g])) * (2 * row + E32 * (n + 16) + extra) + 1.01 * eps * np.abs(w @ V[g])
                    le[b, h, s] = m + np.log(e.sum())
                    lb[b, h, s] = row + 4 * E32 * (1 + np.abs(le[b, h, s]))
    return o, ob, le, lb, used


def check(got, want, fill=7.0):
    o, l = got
    O, ob, L, lb, used = want
    for a, val, bound in ((f64(o), O, ob), (l.astype(np.float64), L, lb)):
        mask = np.broadcast_to(used[:, None], a.shape)
        assert np.all(a[~mask] == fill), "a column that is no token was written"
        off = np.abs(a - val) - bound
        assert not np.any(~(off[mask] <= 0)), (float(np.nanmax(np.where(mask, off, -np.inf))), np.argwhere(mask & ~(off <= 0))[:3])


SHAPES = [
    # heads, kv, hd, page, lengths, one column to a row of the batch (else all columns side by side)
    (1, 1, 64, 16, [1], True), (2, 1, 64, 16, [2, 1, 3], False), (12, 12, 64, 16, [256], True), (16, 8, 128, 16, [15, 16, 17, 31, 32, 33, 100], False),
    (6, 1, 96, 48, [47, 48, 49, 130], True), (5, 5, 72, 64, [200, 1, 64], False), (4, 2, 8, 16, [40, 7], True), (3, 3, 40, 32, [129, 128, 127], False),
    (16, 1, 128, 16, [300], True), (17, 1, 80, 16, [77, 33], False), (40, 2, 128, 256, [255, 256, 257, 513], True), (64, 2, 64, 16, [90], False),
    (2, 2, 128, 64, [3000], True), (16, 8, 128, 16, [2048, 5, 900], False), (8, 2, 120, 32, [1, 1, 1, 5000], False),
    (2, 1, 64, 16, [1 + 37 * (i % 11) for i in range(300)], False), (1, 1, 16, 16, list(range(1, 66)), True), (130, 130, 24, 16, [70, 20], False),
    (70, 1, 64, 16, [100, 400], True), (130, 2, 32, 16, [33, 500, 1500], False), (48, 1, 128, 16, [700, 64], True), (65, 1, 96, 48, [2000], True),
    (40, 2, 128, 16, [3000, 17, 450], False), (1, 1, 16, 16, [1 + i % 19 for i in range(1500)], False),
]


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(br, i, storage):
    heads, kv, hd, page, lengths, rows = SHAPES[i]
    cache = Cache(storage, kv, hd, page, lengths, seed=i, room=i % 3)
    N, scale = len(lengths), float(np.float32(1.0 / np.sqrt(hd)))
    q = stored(storage, np.random.default_rng(i).standard_normal((N, heads * hd, 1) if rows else (1, heads * hd, N)))
    pos = np.array(lengths) - 1
    got = attend(br, cache, q, None, pos, heads, scale)
    check(got, expected(cache, q, None, pos, heads, scale))
    again = attend(br, cache, q, None, pos, heads, scale)
    assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])
    alone = attend(br, cache, q, None, pos, heads, scale, lse=False)
    assert np.array_equal(alone[0], got[0]) and np.all(alone[1] == 7.0)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(8, 1, 64, 16, [40000]), (6, 1, 96, 48, [20001, 3, 700]), (40, 2, 64, 64, [30000]), (48, 1, 32, 16, [40000, 39000, 1]),
                                   (1, 1, 32, 256, [200000]), (15, 5, 40, 32, [33333, 40]), (20, 1, 128, 16, [25000, 0, 11])])
def test_units_of_many_tiles(br, storage, shape):
    """Few sequences, long ones: cut into fewer pieces than there are workgroups; a length of 0 is a column of no token."""
    heads, kv, hd, page, lengths = shape
    cache = Cache(storage, kv, hd, page, [max(n, 1) for n in lengths], seed=sum(lengths))
    N, scale = len(lengths), float(np.float32(1.0 / np.sqrt(hd)))
    q = stored(storage, np.random.default_rng(N + heads).standard_normal((1, heads * hd, N)))
    pos = np.array(lengths) - 1
    want = expected(cache, q, None, pos, heads, scale)
    got = attend(br, cache, q, None, pos, heads, scale)
    check(got, want)
    again = attend(br, cache, q, None, pos, heads, scale)
    assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_columns_of_no_token_and_several_of_one_sequence(br, storage):
    """[3][C][4]: padded columns, positions in the middle of a sequence, one sequence many times, sequences and positions that are none."""
    cache = Cache(storage, 2, 64, 16, [70, 33, 200], seed=40, room=1)
    seq = np.array([[0, 2, 2, -1], [1, 1, 3, 2], [2 ** 31 - 1, -2 ** 31, 0, 2]], np.int32)
    pos = np.array([[69, 0, 199, 5], [32, -1, 0, 100], [3, 3, -2 ** 31, 14 * 16]], np.int32)
    q = stored(storage, np.random.default_rng(41).standard_normal((3, 4 * 64, 4)))
    got = attend(br, cache, q, seq, pos, 4, 0.125)
    check(got, expected(cache, q, seq, pos, 4, 0.125))
    assert expected(cache, q, seq, pos, 4, 0.125)[4].sum() == 5


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_a_sequences_own_is_not_seen(br, storage, bad):
    """Infinities and NaNs behind a position in its page, in other pages and in other columns leave a result as it is, to the bit."""
    lengths = [1, 13, 16, 37, 64, 250, 1000]
    cache = Cache(storage, 2, 128, 16, lengths, seed=42)
    q = stored(storage, np.random.default_rng(43).standard_normal((1, 4 * 128, 7)))
    pos = np.array(lengths) - 1
    o, l = attend(br, cache, q, None, pos, 4, 0.09)
    for which in ("k", "v"):
        a = getattr(cache, which)
        spoilt = np.full(a.shape, stored(storage, np.full(1, bad))[0], a.dtype)
        for i, n in enumerate(lengths):
            for p in range(n):
                if i != 1:          # one sequence is spoilt throughout
                    page, slot = cache.row(i, p)
                    spoilt[page, :, slot] = a[page, :, slot]
        setattr(cache, which, spoilt)
    q[:, :, 1] = stored(storage, np.full(1, bad))[0]
    o2, l2 = attend(br, cache, q, None, pos, 4, 0.09)
    keep = [0, 2, 3, 4, 5, 6]
    assert np.array_equal(o2[:, :, keep], o[:, :, keep]) and np.array_equal(l2[:, :, keep], l[:, :, keep])


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700])
def test_own_infinities(br, storage, n):
    """A value of a sequence that is no number gives what the formula gives, in its own channel and head alone."""
    hd = 64
    def run(edit):
        cache = Cache(storage, 2, hd, 16, [n], seed=44)
        q = stored(storage, np.random.default_rng(45).standard_normal((1, 4 * hd, 1)))
        edit(cache)
        return f64(attend(br, cache, q, None, [n - 1], 4, 0.125)[0])[0, :, 0].reshape(2, 2, hd)
    def put(which, pos, head, channel, value):
        def edit(cache):
            page, slot = cache.row(0, pos)
            getattr(cache, which)[page, head, slot, channel] = stored(storage, np.full(1, value))[0]
        return edit
    clean = run(lambda c: None)
    rest = [c for c in range(hd) if c != 9]
    for value in (np.inf, -np.inf, np.nan):
        for at in (0, n // 2 + 3, n - 1):
            got = run(put("v", at, 1, 9, value))
            assert np.all(np.isnan(got[1, :, 9]) if value != value else got[1, :, 9] == value), (value, at)
            assert np.array_equal(got[0], clean[0])
            # (the weights of another's channels are the same; a careful second pass may add them up in another order)
            assert np.allclose(got[1][:, rest], clean[1][:, rest], rtol=2.0 ** -7 if storage == "bf16" else n * E32, atol=2.0 ** -7 if storage == "bf16" else 4 * n * E32)
    for value in (np.inf, np.nan):          # a score that is +inf (or NaN) somewhere, -inf for the query of the other sign
        got = run(put("k", n // 2, 0, 5, value))
        assert np.array_equal(got[1], clean[1])
        assert np.all(np.isnan(got[0])) if value != value else np.all(np.isnan(got[0]) | np.isfinite(got[0]))
    both = run(lambda c: (put("v", 3, 0, 9, np.inf)(c), put("v", n - 2, 0, 9, -np.inf)(c)))
    assert np.all(np.isnan(both[0, :, 9])) and np.all(np.isfinite(both[0][:, rest]))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_pages_that_are_none_are_left_out(br, storage):
    cache = Cache(storage, 1, 64, 16, [200, 200, 40, 64], seed=46)
    cache.pages[0, 3], cache.pages[0, 7], cache.pages[1, 0], cache.pages[1, 12] = -1, cache.n_pages, 2 ** 31 - 1, -2 ** 31
    cache.pages[2] = -7
    q = stored(storage, np.random.default_rng(47).standard_normal((4, 2 * 64, 1)))
    pos = np.array([199, 199, 39, 63])
    want = expected(cache, q, None, pos, 2, 0.125)
    assert list(want[4][:, 0]) == [True, True, False, True]
    check(attend(br, cache, q, None, pos, 2, 0.125), want)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_scores_of_any_size(br, storage):
    """Scores whose exponentials overflow or vanish, equal ones, and a largest one at the end of a long cache."""
    cache = Cache(storage, 1, 64, 16, [900, 300, 257], seed=48, spread=9.0)
    q = stored(storage, 9.0 * np.random.default_rng(49).standard_normal((1, 2 * 64, 3)))
    q[:, :, 1] = stored(storage, np.zeros(1))[0]
    pos = np.array([899, 299, 256])
    page, slot = cache.row(2, 256)
    cache.k[page, 0, slot] = stored(storage, 4.0 * f64(q)[0, :64, 2])
    got = attend(br, cache, q, None, pos, 2, 0.125)
    assert np.all(np.isfinite(f64(got[0]))) and np.all(np.isfinite(got[1]))
    check(got, expected(cache, q, None, pos, 2, 0.125))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_scores_beyond_what_fp32_tells_apart(br, storage):
    """Scores of 2^24 to 2^34: the largest one of a row takes all where it is ahead of the others by more than the rounding of its sum; equal ones share."""
    cache = Cache(storage, 1, 64, 16, [500, 40, 33], seed=59, spread=4e4)
    q = stored(storage, 4e4 * np.random.default_rng(60).standard_normal((1, 2 * 64, 3)))
    page, slot = cache.row(1, 7)
    page2, slot2 = cache.row(1, 30)
    cache.k[page2, 0, slot2] = cache.k[page, 0, slot]
    o, l = attend(br, cache, q, None, [499, 39, 32], 2, 0.125)
    assert np.all(np.isfinite(f64(o))) and np.all(np.isfinite(l))
    told = 0
    for i, n in enumerate(cache.lengths):
        K, V = cache.rows(cache.k, i, n)[0], cache.rows(cache.v, i, n)[0]
        for h in range(2):
            Q = f64(q)[0, h * 64:(h + 1) * 64, i]
            z, off = 0.125 * (K @ Q), 0.125 * (np.abs(K) @ np.abs(Q)).max() * E32 * 80
            ahead = np.flatnonzero(z >= z.max() - 2 * off - 40)
            if len({tuple(K[a]) for a in ahead}) > 1:
                continue
            told += 1
            want = V[ahead].mean(0)
            assert np.all(np.abs(f64(o)[0, h * 64:(h + 1) * 64, i] - want) <= (1.01 * STEP[storage] + 2.0 ** -14) * np.abs(V[ahead]).max(0) + 1e-12)
            assert abs(l[0, h, i] - z.max()) <= off + 2 * E32 * abs(z.max()) + 1
    assert told >= 4


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_nothing_but_columns_of_no_token(br, storage):
    cache = Cache(storage, 2, 64, 16, [20, 30], seed=61)
    q = stored(storage, np.ones((1, 4 * 64, 300)))
    for seq, pos in ((np.full(300, -1), np.zeros(300)), (np.zeros(300), np.full(300, -1))):
        o, l = attend(br, cache, q, seq.astype(np.int32), pos.astype(np.int32), 4, 0.1)
        assert np.all(f64(o) == 7.0) and np.all(l == 7.0)
        got = append(br, cache, q, q[:, :128], q[:, 128:], None, None, seq.astype(np.int32), pos.astype(np.int32), 4, None, None, 0.0)
        assert np.all(f64(got[0]) == 5.0) and np.array_equal(got[1], cache.k) and np.array_equal(got[2], cache.v)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_cache_of_more_than_four_gigabytes(br, storage):
    """The last pages of a cache whose values pass 2^31 and whose bytes pass 2^32; all other pages are never touched."""
    kv, hd, page, n = 8, 128, 64, 150
    size = 4 if storage == "f32" else 2
    n_pages = 2 ** 31 // (kv * page * hd) + 40
    big = [br.DevArray((n_pages, kv, page, hd), np.float32 if storage == "f32" else np.uint16) for _ in range(2)]
    small = Cache(storage, kv, hd, page, [n], seed=50)
    ids = [n_pages - 1, n_pages - 40, n_pages - 2]
    for j, a in enumerate(ids):
        for dev, src in zip(big, (small.k, small.v)):
            one = np.ascontiguousarray(src[small.pages[0, j]])
            br.lib.mi355_buf_write(dev.handle, a * one.nbytes, one.ctypes.data, one.nbytes)
    table, pos = br.DevArray.from_numpy(np.array([ids], np.int32)), br.DevArray.from_numpy(np.array([n - 1], np.int32))
    c = br.KvCache(big[0].ptr, big[1].ptr, table.ptr, n_pages, page, 1, 3, kv, hd)
    rng = np.random.default_rng(51)
    q, k, v = (stored(storage, rng.standard_normal((1, h * hd, 1))) for h in (16, kv, kv))
    D = br.DevArray.from_numpy
    qd, kd, vd, o = D(q), D(k), D(v), D(np.zeros_like(q))
    br.check(fn(br, "attn_paged", storage)(C.byref(c), o.ptr, None, qd.ptr, None, pos.ptr, 16, 1, 1, 0.09))
    want = expected(small, q, None, [n - 1], 16, 0.09)
    assert np.all(np.abs(f64(o.numpy()) - want[0]) <= want[1])
    # one more position, appended there
    pos2 = D(np.array([n], np.int32))
    br.check(fn(br, "kv_append", storage)(C.byref(c), None, None, kd.ptr, vd.ptr, None, None, None, pos2.ptr, 0, 1, 1, None, None, 0, 0.0))
    for dev, new in zip(big, (k, v)):
        got = np.empty((kv, page, hd), new.dtype)
        br.lib.mi355_buf_read(dev.handle, ids[2] * got.nbytes, got.ctypes.data, got.nbytes)
        assert np.array_equal(got[:, n % page], new.reshape(kv, hd))
    for a in big:
        a.free()


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_a_table_of_a_billion_positions(br, storage):
    """Columns go in several launches where their tiles could be more than 32 bits count: 20 of them, 16 heads, 2^30 positions to a row of the table."""
    kv, hd, page = 16, 8, 1 << 16
    lengths = [300, 66000, 1, 131073]
    small = Cache(storage, kv, hd, 16, lengths, seed=55)                # the oracle's own
    ids, table = iter(range(100)), np.full((4, 1 << 14), -1, np.int32)
    shape = (8, kv, page, hd)
    k, v = np.zeros(shape, small.k.dtype), np.zeros(shape, small.k.dtype)
    for i, n in enumerate(lengths):
        for j in range(-(-n // page)):
            table[i, j] = next(ids)
        at = np.arange(n)
        old = small.pages[i, at // 16]
        for new, src in ((k, small.k), (v, small.v)):
            new[table[i, at // page], :, at % page] = src[old, :, at % 16]
    seq = np.array([0, 1, 2, 3] * 5, np.int32)
    pos = np.array([n - 1 for n in lengths] * 5, np.int32)
    pos[4:8], pos[-1] = [150, 65535, 0, 65536], 17
    q = stored(storage, np.random.default_rng(56).standard_normal((1, kv * hd, 20)))
    D = br.DevArray.from_numpy
    kd, vd, td, qd, sd, pd, o, l = D(k), D(v), D(table), D(q), D(seq), D(pos), D(np.zeros_like(q)), br.DevArray((1, kv, 20))
    c = br.KvCache(kd.ptr, vd.ptr, td.ptr, 8, page, 4, 1 << 14, kv, hd)
    br.check(fn(br, "attn_paged", storage)(C.byref(c), o.ptr, l.ptr, qd.ptr, sd.ptr, pd.ptr, kv, 20, 1, 0.35))
    check((o.numpy(), l.numpy()), expected(small, q, seq, pos, kv, 0.35))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("S", [5, 333])
def test_a_prompt_through_the_cache(br, storage, S):
    """A prompt appended, and each of its positions attending over the cache, gives what mi355_qknorm_rope_fwd_dev and mi355_attn_fwd_dev give: the
    same values but for the order of sums and their rounding (twice, where a rounded k is multiplied again)."""
    heads, kv, hd, end = 8, 4, 64, "_dev" if storage == "f32" else "_bf16_dev"
    rng = np.random.default_rng(57)
    q, k, v = (stored(storage, rng.standard_normal((1, h * hd, S))) for h in (heads, kv, kv))
    wq, wk = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    D = br.DevArray.from_numpy
    cos, sin = br.rope_tables_dev(S, hd, 10000.0)
    qd, kd, vd, wqd, wkd = D(q), D(k), D(v), D(wq), D(wk)
    qr, kr, o, l = D(np.zeros_like(q)), D(np.zeros_like(k)), D(np.zeros_like(q)), br.DevArray((1, heads, S))
    br.check(getattr(br.lib, "mi355_qknorm_rope_fwd" + end)(qr.ptr, kr.ptr, qd.ptr, kd.ptr, wqd.ptr, wkd.ptr, heads, kv, hd, S, 1, cos, sin, 1e-5))
    br.check(getattr(br.lib, "mi355_attn_fwd" + end)(o.ptr, l.ptr, qr.ptr, kr.ptr, vd.ptr, None, heads, kv, hd, S, 1, 0.125))
    cache = Cache(storage, kv, hd, 16, [S], seed=58, values=False)
    c, seq, pos = cache.to(br), D(np.zeros((1, S), np.int32)), D(np.arange(S, dtype=np.int32)[None])
    q2, o2, l2 = D(np.zeros_like(q)), D(np.zeros_like(q)), br.DevArray((1, heads, S))
    br.check(fn(br, "kv_append", storage)(C.byref(c), q2.ptr, qd.ptr, kd.ptr, vd.ptr, wqd.ptr, wkd.ptr, seq.ptr, pos.ptr, heads, S, 1, cos, sin, S, 1e-5))
    br.check(fn(br, "attn_paged", storage)(C.byref(c), o2.ptr, l2.ptr, q2.ptr, seq.ptr, pos.ptr, heads, S, 1, 0.125))
    cache.k, cache.v = cache.kd.numpy(), cache.vd.numpy()
    step = STEP[storage]
    a, b = f64(qr.numpy()), f64(q2.numpy())
    off = 2.1 * step * np.abs(a) + E32 * (hd + 16) * 8          # (values are below 8)
    assert np.all(np.abs(a - b) <= off)
    want = expected(cache, q2.numpy(), np.zeros(S, int), np.arange(S), heads, 0.125)
    check((o2.numpy(), l2.numpy()), want)
    # against the other path: scores differ by what their rounded q and k do, 2 * 2.1 steps of the sum of magnitudes
    K = np.abs(f64(kr.numpy()).reshape(kv, hd, S))
    for h in range(heads):
        A = np.abs(a[0, h * hd:(h + 1) * hd])
        dz = 0.125 * (A.T @ K[h // 2]).max(1) * 4.3 * (step + E32 * hd)
        V = np.abs(f64(v).reshape(kv, hd, S)[h // 2]).max()
        assert np.all(np.abs(f64(o.numpy())[0, h * hd:(h + 1) * hd] - f64(o2.numpy())[0, h * hd:(h + 1) * hd]).max(0) <= V * (2.2 * dz + 3 * step + E32 * S))
        assert np.all(np.abs(l.numpy()[0, h] - l2.numpy()[0, h]) <= dz + E32 * (S + 64))


# ---- appending -------------------------------------------------------------------------------------------------------------------

def append(br, cache, q, k, v, wq, wk, seq, pos, heads, cos, sin, eps, fill=5.0, inplace=False):
    B, _, S = k.shape
    D = br.DevArray.from_numpy
    at = lambda a: None if a is None else D(a)          # noqa: E731
    c = cache.to(br)
    qd, kd, vd, wqd, wkd, cd, sd, seqd, posd = (at(a) for a in (q, k, v, wq, wk, cos, sin, seq, pos))
    out = None if q is None else qd if inplace else D(stored(cache.storage, np.full(q.shape, fill)))
    ptr = lambda d: None if d is None else d.ptr        # noqa: E731
    br.check(fn(br, "kv_append", cache.storage)(C.byref(c), ptr(out), ptr(qd), kd.ptr, vd.ptr, ptr(wqd), ptr(wkd), ptr(seqd), posd.ptr,
                                                heads, S, B, ptr(cd), ptr(sd), 0 if cos is None else cos.shape[1], eps))
    return (None if out is None else out.numpy()), cache.kd.numpy(), cache.vd.numpy()


def turned(x, heads, w, cos, sin, pos, eps, storage):
    """Values and bounds of rotate(norm(x), pos), [batch][heads*hd][S]."""
    B, Ch, S = x.shape
    hd = Ch // heads
    y = f64(x).reshape(B, heads, hd, S)
    rel = 0.0
    if w is not None:
        y = y / np.sqrt((y * y).mean(2, keepdims=True) + eps) * w.astype(np.float64)[:, None]
        rel = E32 * (hd / 2 + 8)            # the sum of squares halves under the root; root, reciprocal, mean, two products
    if cos is None:
        val, mag = y, np.abs(y) * rel
    else:
        p = np.clip(pos, 0, cos.shape[1] - 1)
        c, s = (t.astype(np.float64)[:, p].transpose(1, 0, 2)[:, None] for t in (cos, sin))      # [B][1][hd/2][S]
        a, b = y[:, :, 0::2], y[:, :, 1::2]
        val, mag = np.empty_like(y), np.empty_like(y)
        val[:, :, 0::2], val[:, :, 1::2] = a * c - b * s, a * s + b * c
        mag[:, :, 0::2] = np.abs(a * c) + np.abs(b * s)
        mag[:, :, 1::2] = np.abs(a * s) + np.abs(b * c)
        mag *= rel + 3 * E32
    bound = 1.01 * mag + (1.01 * STEP[storage] * np.abs(val) if storage == "bf16" else E32 * np.abs(val)) + 1e-40
    return val.reshape(x.shape), bound.reshape(x.shape)


APPENDS = [
    # heads, kv, hd, page, batch, S, lengths (of prompts, padded to S; None: one new token of each column's sequence), norm, rotation
    (1, 1, 8, 16, 1, 1, None, False, True), (12, 12, 64, 16, 1, 1, None, False, True), (16, 8, 128, 16, 1, 64, None, True, True),
    (4, 2, 128, 16, 37, 1, None, True, True), (6, 1, 96, 48, 3, 5, None, True, True), (5, 5, 72, 64, 1, 7, None, False, False),
    (16, 8, 128, 16, 2, 256, [256, 100], True, True), (2, 1, 64, 32, 1, 197, [197], True, True), (3, 3, 40, 16, 3, 33, [33, 1, 0], False, True),
    (12, 12, 64, 16, 1, 1030, [1030], False, True), (8, 2, 120, 16, 2, 65, [64, 65], True, False), (0, 2, 128, 16, 2, 40, [40, 17], True, True),
    (40, 2, 128, 256, 1, 300, [300], True, True), (4, 4, 16, 16, 5, 15, [15, 3, 16 - 1, 8, 2], True, True), (2, 2, 88, 16, 1, 130, [129], True, True),
    # enough columns for tiles: rows of odd lengths, sizes of heads that fill no tile, the last columns of a row short, columns of different sequences
    (8, 2, 120, 16, 2, 345, [345, 65], True, True), (3, 3, 40, 32, 5, 211, [211, 0, 64, 65, 128], False, True), (6, 1, 88, 48, 3, 449, [449, 448, 3], True, False),
    (16, 8, 8, 16, 1, 515, [515], True, True), (5, 5, 72, 16, 40, 19, None, True, True), (16, 8, 128, 16, 1, 300, None, True, True),
    (0, 4, 64, 64, 4, 260, [260, 100, 259, 1], True, True), (16, 8, 24, 16, 16, 16, [16] * 15 + [7], True, True),
]


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(br, i, storage):
    heads, kv, hd, page, B, S, lengths, norm, rotate = APPENDS[i]
    rng = np.random.default_rng(60 + i)
    if lengths is None:
        have = rng.integers(1, 200, B * S)
        seq, pos = None, (have - 1).reshape(B, S).astype(np.int32)
    else:
        have = lengths
        pos = np.where(np.arange(S)[None] < np.array(lengths)[:, None], np.arange(S)[None], -1).astype(np.int32)
        seq = np.where(pos >= 0, np.arange(B)[:, None], -1).astype(np.int32)
    cache = Cache(storage, kv, hd, page, have, seed=i, values=False)
    table = int(max(have)) + 3
    cos = sin = None
    if rotate:
        angle = np.arange(table)[None] / 10000.0 ** (2 * np.arange(hd // 2) / hd)[:, None]
        cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    q, k, v = (stored(storage, rng.standard_normal((B, h * hd, S))) for h in (max(heads, 1), kv, kv))
    q = q if heads else None
    wq, wk = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    got_q, got_k, got_v = append(br, cache, q, k, v, wq, wk, seq, pos, heads, cos, sin, 1e-5)
    token = np.broadcast_to((pos >= 0)[:, None], (B, max(heads, 1) * hd, S))
    if heads:
        val, bound = turned(q, heads, wq, cos, sin, pos, 1e-5, storage)
        assert np.all(f64(got_q)[~token] == 5.0)
        assert np.all((np.abs(f64(got_q) - val) <= bound)[token])
        again = append(br, cache, q, k, v, wq, wk, seq, pos, heads, cos, sin, 1e-5, inplace=True)
        assert np.array_equal(again[0][token], got_q[token]) and np.array_equal(again[0][~token], q[~token])
        assert np.array_equal(again[1], got_k) and np.array_equal(again[2], got_v)
    val, bound = turned(k, kv, wk, cos, sin, pos, 1e-5, storage)
    want_k, off_k, want_v = f64(cache.k), np.zeros(cache.k.shape), cache.v.copy()
    for b in range(B):
        for s in range(S):
            if pos[b, s] < 0:
                continue
            page_id, slot = cache.row(b * S + s if seq is None else seq[b, s], pos[b, s])
            want_k[page_id, :, slot] = val[b, :, s].reshape(kv, hd)
            off_k[page_id, :, slot] = bound[b, :, s].reshape(kv, hd)
            want_v[page_id, :, slot] = v[b, :, s].reshape(kv, hd)
    assert np.all(np.abs(f64(got_k) - want_k) <= off_k)         # (nothing else is written: a bound of zero)
    assert np.array_equal(got_v, want_v)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("S", [4, 70, 403])
def test_append_of_columns_that_are_no_token(br, storage, S):
    """Sequences, positions, pages and angles that are none: nothing is written for them, everything for the others."""
    cache = Cache(storage, 2, 64, 16, [200, 200, 90], seed=80, values=False)
    cache.pages[1, 2], cache.pages[1, 4] = -1, cache.n_pages
    rng = np.random.default_rng(81)
    q, k, v = (stored(storage, rng.standard_normal((3, h * 64, S))) for h in (4, 2, 2))
    seq = np.array([0, 1, 1, 5, -1, 2, 0, 2 ** 31 - 1, -2 ** 31, 1], np.int64)
    pos = np.array([199, 37, 70, 0, 3, 13 * 16, 2 ** 31 - 1, 5, 5, -2 ** 31], np.int64)
    places = [(0, 100 + j) for j in range(60)] + [(2, j) for j in range(50)] + [(1, 80 + j) for j in range(90)] + [(0, j) for j in range(99)]     # of the others, each its own
    seqs, poss = np.empty(3 * S, np.int32), np.empty(3 * S, np.int32)
    good = np.zeros(3 * S, bool)
    for n in range(3 * S):
        if n % 3 == 0 and places:
            (seqs[n], poss[n]), good[n] = places.pop(0), True
        else:
            seqs[n], poss[n] = seq[1 + n % 9], pos[1 + n % 9]
    good &= poss < 150                                          # the angles end there
    cos, sin = rng.standard_normal((2, 32, 150)).astype(np.float32)
    seqs, poss, good = (a.reshape(3, S) for a in (seqs, poss, good))
    got_q, got_k, got_v = append(br, cache, q, k, v, None, None, seqs, poss, 4, cos, sin, 0.0)
    val, bound = turned(q, 4, None, cos, sin, poss, 0.0, storage)
    mask = np.broadcast_to(good[:, None], q.shape)
    assert np.all(f64(got_q)[~mask] == 5.0) and np.all((np.abs(f64(got_q) - val) <= bound)[mask])
    val, bound = turned(k, 2, None, cos, sin, poss, 0.0, storage)
    want_k, off_k, want_v = f64(cache.k), np.zeros(cache.k.shape), cache.v.copy()
    for b, s in np.argwhere(good):
        page, slot = cache.row(seqs[b, s], poss[b, s])
        want_k[page, :, slot], off_k[page, :, slot] = val[b, :, s].reshape(2, 64), bound[b, :, s].reshape(2, 64)
        want_v[page, :, slot] = v[b, :, s].reshape(2, 64)
    assert good.sum() > min(S // 2, 100) and np.all(np.abs(f64(got_k) - want_k) <= off_k) and np.array_equal(got_v, want_v)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_rows_of_any_alignment(br, storage):
    """q, k, v and the results at any element, and an odd number of columns."""
    cache = Cache(storage, 2, 64, 16, [77] * 5, seed=82)
    rng = np.random.default_rng(83)
    q, k, v = (stored(storage, rng.standard_normal((1, h * 64, 5))) for h in (4, 2, 2))
    pos = np.full(5, 76, np.int32)
    want = append(br, cache, q, k, v, None, None, None, pos, 4, None, None, 0.0)
    D, size = br.DevArray.from_numpy, q.dtype.itemsize
    for shift in (1, 3):
        off = [D(np.concatenate([np.zeros(shift, a.dtype), a.ravel()])) for a in (q, k, v, np.zeros_like(q), np.zeros_like(q))]
        p = [a.ptr + shift * size for a in off]
        c, posd = cache.to(br), D(pos)
        br.check(fn(br, "kv_append", storage)(C.byref(c), p[3], p[0], p[1], p[2], None, None, None, posd.ptr, 4, 5, 1, None, None, 0, 0.0))
        assert np.array_equal(off[3].numpy()[shift:].reshape(q.shape), want[0]) and np.array_equal(cache.kd.numpy(), want[1])
        br.check(fn(br, "attn_paged", storage)(C.byref(c), p[4], None, p[3], None, posd.ptr, 4, 5, 1, 0.125))
        once = [D(want[0]), D(np.zeros_like(q))]
        br.check(fn(br, "attn_paged", storage)(C.byref(c), once[1].ptr, None, once[0].ptr, None, posd.ptr, 4, 5, 1, 0.125))
        assert np.array_equal(off[4].numpy()[shift:].reshape(q.shape), once[1].numpy())


# ---- streams and graphs ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_graphs_that_share_the_workspace(br, storage):
    """Two recorded steps (append, then attention whose sequences several workgroups share), replayed in turn with eager work between."""
    D = br.DevArray.from_numpy
    steps = []
    for seed, lengths in ((90, [3000, 10, 700]), (91, [1, 5000, 64])):
        cache = Cache(storage, 2, 128, 16, lengths, seed=seed)
        rng = np.random.default_rng(seed)
        q, k, v = (stored(storage, rng.standard_normal((1, h * 128, 3))) for h in (4, 2, 2))
        pos = np.array(lengths, np.int32) - 1
        eager_q, eager_k, eager_v = append(br, cache, q, k, v, None, None, None, pos, 4, None, None, 0.0)
        cache.k, cache.v = eager_k, eager_v
        want = attend(br, cache, eager_q, None, pos, 4, 0.09, fill=0.0)
        c = cache.to(br)
        d = [D(a) for a in (q, k, v, pos)] + [D(np.zeros_like(q)), D(np.zeros_like(q)), br.DevArray((1, 4, 3))]
        br.check(br.lib.mi355_graph_begin())
        br.check(fn(br, "kv_append", storage)(C.byref(c), d[4].ptr, d[0].ptr, d[1].ptr, d[2].ptr, None, None, None, d[3].ptr, 4, 3, 1, None, None, 0, 0.0))
        br.check(fn(br, "attn_paged", storage)(C.byref(c), d[5].ptr, d[6].ptr, d[4].ptr, None, d[3].ptr, 4, 3, 1, 0.09))
        graph = br.lib.mi355_graph_end()
        assert graph, br.last_error()
        steps.append((cache, d, graph, want))
    for _ in range(3):
        for cache, d, graph, want in steps:
            d[5].zero(), d[6].zero()
            br.check(br.lib.mi355_graph_launch(graph))
        for cache, d, graph, want in steps:
            assert np.array_equal(d[5].numpy(), want[0]) and np.array_equal(d[6].numpy(), want[1])
        other = Cache(storage, 1, 64, 16, [2500], seed=92)
        attend(br, other, stored(storage, np.ones((1, 64, 1))), None, [2499], 1, 0.125)
    for s in steps:
        br.lib.mi355_graph_free(s[2])


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_another_stream(br, storage):
    """Append, attention, a beam's step and the rows that follow, on a stream of the caller's."""
    hip, stream = br.lib, C.c_void_p()          # (the runtime that the library itself has loaded)
    cache = Cache(storage, 2, 64, 16, [700, 9], seed=95)
    rng = np.random.default_rng(96)
    q, k, v = (stored(storage, rng.standard_normal((1, h * 64, 2))) for h in (4, 2, 2))
    pos = np.array([699, 8], np.int32)

    def all_four():
        new = append(br, cache, q, k, v, None, None, None, pos, 4, None, None, 0.0)
        out = attend(br, cache, new[0], None, pos, 4, 0.125)
        D = br.DevArray.from_numpy
        x, s = D(q.reshape(1, 256, 2)), D(np.zeros(2, np.float32))
        o = [br.DevArray(2)] + [br.DevArray(2, np.int32) for _ in range(3)]
        br.check(fn(br, "beam_step", storage)(*[a.ptr for a in o], x.ptr, s.ptr, None, 256, 2, 1, 2, 3, 0))
        c, par, po, sp, t = cache.to(br), D(np.array([1, 1], np.int32)), D(np.array([8, 8], np.int32)), D(np.array([0, 1], np.int32)), [D(np.zeros((2, cache.max_pages), np.int32)), D(np.zeros(2, np.int32)), D(np.zeros(2, np.int32))]
        br.check(fn(br, "kv_reorder", storage)(C.byref(c), 1, t[0].ptr, t[1].ptr, t[2].ptr, par.ptr, po.ptr, sp.ptr, 1))
        return list(new) + list(out) + [a.numpy() for a in o + t] + [cache.kd.numpy()]

    want = all_four()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    br.check(br.lib.mi355_set_stream(stream))
    try:
        got = all_four()
    finally:
        br.check(br.lib.mi355_set_stream(None))         # (waits for the other one)
        assert hip.hipStreamDestroy(stream) == 0
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
