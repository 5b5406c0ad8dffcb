"""Attention over a paged cache at the ends of what its entry point takes."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_attention import E32, STEP
from test_gpu_paged import f64, fn, stored

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
