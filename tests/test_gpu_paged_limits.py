"""A paged cache at the ends of what its entry points take."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_attention import E32, STEP
from test_gpu_paged import Cache, append, attend, f64, fn, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage,kv,max_pages", [("f32", 32, 67108848), ("bf16", 64, 67108824)])
def test_as_many_tiles_as_a_launch_counts(br, storage, kv, max_pages):
    """One column at the last position of a table of nearly 2^30 whose tiles and heads are 2^31 - 256 (2^31 - 768) places; all but four entries of the
    table are no page.  The bounds are those of the other tests of attention: n * 2^-24 of the magnitudes for the sums, the weights' 2^-15, one rounding."""
    hd, page, scale = 8, 16, 0.35
    rng = np.random.default_rng(kv)
    k, v = (stored(storage, rng.standard_normal((5, kv, page, hd))) for _ in range(2))
    q = stored(storage, rng.standard_normal((1, kv * hd, 1)))
    table = np.full((1, max_pages), -1, np.int32)
    places = {0: 2, 4242424: 0, 40000001: 4, max_pages - 1: 3}
    for at, page_id in places.items():
        table[0, at] = page_id
    D = br.DevArray.from_numpy
    kd, vd, td, qd, pd = D(k), D(v), D(table), D(q), D(np.array([max_pages * page - 1], np.int32))
    o, lse = D(stored(storage, np.full(q.shape, 7.0))), D(np.full((1, kv, 1), 7.0, np.float32))
    c = br.KvCache(kd.ptr, vd.ptr, td.ptr, 5, page, 1, max_pages, kv, hd)
    br.check(fn(br, "attn_paged", storage)(C.byref(c), o.ptr, lse.ptr, qd.ptr, None, pd.ptr, kv, 1, 1, scale))
    ids = list(places.values())
    K, V = (f64(a)[ids].transpose(1, 0, 2, 3).reshape(kv, -1, hd) for a in (k, v))
    Q = f64(q).reshape(kv, hd)
    z = scale * np.einsum("gtc,gc->gt", K, Q)
    dz = E32 * (hd + 6) * scale * np.einsum("gtc,gc->gt", np.abs(K), np.abs(Q)).max(1)
    e = np.exp(z - z.max(1, keepdims=True))
    w, n = e / e.sum(1, keepdims=True), K.shape[1]
    row = 2 * dz + E32 * (n + 32 + 2 * np.abs(z).max(1))
    want, mag = np.einsum("gt,gtc->gc", w, V), np.einsum("gt,gtc->gc", w, np.abs(V))
    bound = 1.01 * mag * (2 * row[:, None] + E32 * (n + 16) + (2.0 ** -15 if storage == "bf16" else 0.0)) + 1.01 * STEP[storage] * np.abs(want)
    assert np.all(np.abs(f64(o.numpy()).reshape(kv, hd) - want) <= bound)
    want_lse = z.max(1) + np.log(e.sum(1))
    assert np.all(np.abs(lse.numpy().reshape(kv) - want_lse) <= row + 4 * E32 * (1 + np.abs(want_lse)))


def definition(K, V, Q, scale, storage):
    """(o, bound of o, lse, bound of lse) of one head: K, V [n][hd], Q [hd]; bounds as in test_gpu_paged."""
    n, hd = K.shape
    z = scale * (K @ Q)
    w = np.exp(z - z.max())
    lse = z.max() + np.log(w.sum())
    w /= w.sum()
    row = 2 * E32 * (hd + 6) * scale * (np.abs(K) @ np.abs(Q)).max() + E32 * (n + 32 + 2 * np.abs(z).max())
    o = w @ V
    extra = 2.0 ** -15 if storage == "bf16" else 0.0
    return o, 1.01 * (w @ np.abs(V)) * (2 * row + E32 * (n + 16) + extra) + 1.01 * STEP[storage] * np.abs(o), lse, row + 4 * E32 * (1 + abs(lse))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 40, 700, 9000])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_a_key_of_infinity(br, storage, n, value):
    """A score of +inf leaves NaN in all of its head, one of -inf takes its position out and no more, one of 0 * inf is NaN."""
    hd, heads, at = 64, 4, n // 2
    cache = Cache(storage, 1, hd, 16, [n], seed=70)
    q = stored(storage, np.random.default_rng(71).standard_normal((1, heads * hd, 1)))
    sign = np.array([1.0, -1.0, 0.0, -0.25])                    # of each head's query in that channel, 5
    q[0, 5::hd, 0] = stored(storage, sign)
    page, slot = cache.row(0, at)
    cache.k[page, 0, slot, 5] = stored(storage, np.full(1, value))[0]
    o, lse = attend(br, cache, q, None, [n - 1], heads, 0.125)
    o, lse = f64(o)[0, :, 0].reshape(heads, hd), lse[0, :, 0].astype(np.float64)
    K, V = cache.rows(cache.k, 0, n)[0], cache.rows(cache.v, 0, n)[0]
    others = np.arange(n) != at
    for h in range(heads):
        if sign[h] == 0 or sign[h] * value > 0:
            assert np.all(np.isnan(o[h])) and not np.isfinite(lse[h]), h
        elif n == 1:
            assert np.all(np.isnan(o[h])) and lse[h] == -np.inf, h      # nothing is left: 0 / 0
        else:
            want, bound, want_lse, bound_lse = definition(K[others], V[others], f64(q)[0, h * hd:(h + 1) * hd, 0], 0.125, storage)
            assert np.all(np.abs(o[h] - want) <= bound) and abs(lse[h] - want_lse) <= bound_lse, h


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("S", [6, 40, 700])
def test_two_columns_at_one_place(br, storage, S):
    """Every value of a row is that of a column that names it, also where two do; rows that none names, and all columns' queries, are as they should be."""
    heads, kv, hd = 8, 4, 64
    cache = Cache(storage, kv, hd, 16, [S], seed=72, values=False)
    rng = np.random.default_rng(73)
    q, k, v = (stored(storage, rng.standard_normal((1, h * hd, S))) for h in (heads, kv, kv))
    pos = np.arange(S, dtype=np.int32)[None]
    twice = [(0, 1), (2, S - 1), (S // 2, S // 2 - 1)]          # side by side, far apart
    for a, b in twice:
        pos[0, b] = pos[0, a]
    got_q, got_k, got_v = append(br, cache, q, k, v, None, None, np.zeros((1, S), np.int32), pos, heads, None, None, 0.0)
    assert np.array_equal(got_q, q)
    for got, new, old in ((got_k, k, cache.k), (got_v, v, cache.v)):
        new = new.reshape(kv, hd, S)
        want = old.copy()
        for place in np.unique(pos):
            page, slot = cache.row(0, place)
            row = got[page, :, slot]
            assert np.all((row[:, :, None] == new[:, :, pos[0] == place]).any(2)), place
            want[page, :, slot] = row
        assert np.array_equal(got, want)
