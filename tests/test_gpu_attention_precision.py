"""Attention on bfloat16 storage is as exact as its results' type: weights and score gradients are multiplied again as pairs of bfloat16
values, so what is left beside the rounding of a result is 2^-15 of the magnitudes that enter it, and the error of fp32 sums.

The bound of an element: the fp32 chain's (test_gpu_attention.reference on the same values held as fp32), 2^-15 of the sum of magnitudes
of its last product, and half a step of bfloat16 at the result, which is 2^-8 of the power of two at or below it."""
import numpy as np
import pytest

import test_gpu_attention as A

pytestmark = pytest.mark.gpu

PAIR = 2.0 ** -15


def as_fp32(c):
    """The same case with its values held as fp32."""
    w = A.Case("f32", c.heads, c.kv, c.hd, c.S, c.batch, c.cu)
    w.q, w.k, w.v, w.do, w.scale = *(A.from_bf16(a) for a in (c.q, c.k, c.v, c.do)), c.scale
    return w


def magnitudes(w, o=None, lse=None):
    """Sums of magnitudes of the last products: of o, or, given o and lse, of dq, dk and dv."""
    G, hd, S = w.heads // w.kv, w.hd, w.S
    out = {n: np.zeros((w.batch, (w.kv if n in ("dk", "dv") else w.heads) * hd, S)) for n in (("o",) if o is None else ("dq", "dk", "dv"))}
    for b in range(w.batch):
        ok = w.allowed(b)
        used = ok.any(1)
        for h in range(w.heads):
            rq, rk = slice(h * hd, (h + 1) * hd), slice(h // G * hd, (h // G + 1) * hd)
            Q, K, V, dO = (a.astype(np.float64) for a in (w.q[b, rq], w.k[b, rk], w.v[b, rk], w.do[b, rq]))
            z = np.where(ok, w.scale * (Q.T @ K), -np.inf)
            if o is None:
                e = np.exp(z - np.where(used, np.max(z, axis=1, initial=-1e300), 0.0)[:, None])
                p = e / np.where(used, e.sum(1), 1.0)[:, None]
                out["o"][b, rq] = np.abs(V) @ p.T
                continue
            p = np.where(ok, np.exp(np.where(ok, z, 0.0) - np.where(used, lse[b, h], 0.0)[:, None]), 0.0)
            dO, O = np.where(used, dO, 0.0), np.where(used, o[b, rq].astype(np.float64), 0.0)
            ds = np.abs(p * (dO.T @ V - (dO * O).sum(0)[:, None]))
            out["dq"][b, rq] = w.scale * (np.abs(K) @ ds.T)
            out["dk"][b, rk] += w.scale * (np.abs(Q) @ ds)
            out["dv"][b, rk] += np.abs(dO) @ p
    return out


def check(c, got, want, mags):
    _, end = c.plan()
    for name, mag in mags.items():
        val, bound = want[name]
        bound = bound + 1.01 * PAIR * mag
        top = np.abs(val) + bound
        half = np.exp2(np.floor(np.log2(np.maximum(top, 2.0 ** -126))) - 8)
        used = np.broadcast_to((end > 0)[:, None, :], val.shape)
        over = np.where(used, np.abs(A.from_bf16(got[name]).astype(np.float64) - val) / (bound + half), 0.0)
        assert np.all(over <= 1.0), (name, float(over.max()), float((over > 1.0).mean()))


CASES = [
    # heads, kv, hd, S, batch, offsets: one, two and four position blocks side by side
    (4, 2, 64, 200, 2, [[0, 2, 5, 40, 200]] * 2), (2, 1, 128, 130, 1, None), (3, 1, 96, 300, 1, [[0, 3, 300]]),
    (12, 12, 64, 256, 8, None), (24, 8, 128, 197, 4, None), (24, 24, 72, 140, 6, [[0, 60, 62, 139]] * 6),
    (64, 32, 64, 300, 3, [[0, 4, 50, 300]] * 3), (64, 64, 128, 270, 3, None), (48, 24, 96, 150, 6, None),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_as_exact_as_the_type(br, i):
    c = A.Case("bf16", *CASES[i], seed=20 + i)
    w = as_fp32(c)
    o, lse = A.forward(br, c)
    check(c, dict(o=o), A.reference(w), magnitudes(w))
    g = A.backward(br, c, o, lse)
    O = A.from_bf16(o)
    check(c, g, A.reference(w, O, lse), magnitudes(w, O, lse))


@pytest.mark.parametrize("hd,S,heads", [(64, 200, 2), (128, 197, 24), (96, 300, 64)])
def test_own_infinities_are_what_they_were(br, hd, S, heads):
    """An infinity among a sequence's own values: o is infinite with its sign in that channel from there on, as the formula gives; where
    two of both signs meet it is NaN.  dv of an infinite do likewise, for the keys that its query sees."""
    c = A.Case("bf16", heads, heads, hd, S, 1, seed=3)
    o, lse = A.forward(br, c)
    for channel, at, value in ((5, 10, np.inf), (6, 70, -np.inf), (7, 5, np.inf), (7, 80, -np.inf)):
        c.v[0, channel, at] = c.stored(np.full(1, value))[0]
    got = A.from_bf16(A.forward(br, c)[0])[0, :hd]
    assert np.all(got[5, 10:] == np.inf) and np.all(got[6, 70:] == -np.inf)
    assert np.all(got[7, 5:80] == np.inf) and np.all(np.isnan(got[7, 80:]))
    clean = A.from_bf16(o)[0, :hd]
    rest = [r for r in range(hd) if r not in (5, 6, 7)]
    assert np.array_equal(got[rest], clean[rest]) and np.array_equal(got[5, :10], clean[5, :10])

    c = A.Case("bf16", heads, heads, hd, S, 1, seed=3)
    base = A.backward(br, c, o, lse)
    c.do[0, 9, 100] = c.stored(np.full(1, np.inf))[0]
    dv = A.from_bf16(A.backward(br, c, o, lse)["dv"])[0, :hd]
    assert np.all(dv[9, :101] == np.inf)
    want = A.from_bf16(base["dv"])[0, :hd]
    rest = [r for r in range(hd) if r != 9]
    assert np.array_equal(dv[rest], want[rest]) and np.array_equal(dv[9, 101:], want[9, 101:])


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e4, 3e6, 1e12])
@pytest.mark.parametrize("shape", [(2, 1, 64, 150, 1, None), (24, 8, 96, 200, 4, [[0, 50, 200]] * 4), (64, 64, 128, 270, 3, None)])
def test_scores_beyond_what_an_exponential_holds(br, storage, size, shape):
    """Scores of 1e8 to 1e25: all of a row's weight goes to its largest score, one key or several equal ones.  A row is held to that where
    its second largest score is behind by 100 and by more than both sums' errors (E32 * (hd + 6) of the sums of
    magnitudes, twice for each); lse has a rounding each of two constants, of scale times one of them, of two products and of a sum."""
    c = A.Case(storage, *shape, seed=31)
    f = lambda a: (a if storage == "f32" else A.from_bf16(a))       # noqa: E731
    c.q, c.k = c.stored(f(c.q) * np.float32(size)), c.stored(f(c.k) * np.float32(size))
    o, lse = A.forward(br, c)
    start, end = c.plan()
    held = 0
    for b in range(c.batch):
        ok, used = c.allowed(b), end[b] > 0
        for h in range(0, c.heads, 5):
            rq, rk = slice(h * c.hd, (h + 1) * c.hd), slice(h // (c.heads // c.kv) * c.hd, (h // (c.heads // c.kv) + 1) * c.hd)
            Q, K, V = c.f64(c.q)[b, rq], c.f64(c.k)[b, rk], c.f64(c.v)[b, rk]
            z = np.where(ok, c.scale * (Q.T @ K), -np.inf)
            err = A.E32 * (c.hd + 6) * c.scale * (np.abs(Q).T @ np.abs(K))
            order = np.sort(z, axis=1)
            gap = order[:, -1] - np.where(np.isfinite(order[:, -2]), order[:, -2], -1e30)
            clear = used & (gap > 100 + 4 * np.where(ok, err, 0).max(1))
            got = c.f64(o)[b, rq]
            assert np.all(np.isfinite(got[:, used])) and np.all(np.isfinite(lse[b, h, used]))
            best = V[:, z.argmax(1)]
            assert np.all(np.abs(got - best)[:, clear] <= 8 * A.E32 * np.abs(best)[:, clear])
            assert np.all(np.abs(lse[b, h] - order[:, -1])[clear] <= (err.max(1) + 7 * A.E32 * np.abs(order[:, -1]))[clear])
            held += clear.sum()
    assert held > 100


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_the_largest_scale(br, storage):
    """A scale whose product with log2(e) is beyond fp32 is refused; the largest below it gives what the formula does (scores of equal
    keys: the mean of the values, as good as its sum of 40 terms and a product)."""
    c = A.Case(storage, 1, 1, 8, 40, 1, seed=33)
    p, fn = br.DevArray((4096,)).ptr, br.lib.mi355_attn_fwd_dev if storage == "f32" else br.lib.mi355_attn_fwd_bf16_dev
    bwd = br.lib.mi355_attn_bwd_dev if storage == "f32" else br.lib.mi355_attn_bwd_bf16_dev
    for scale in (2.5e38, 3.4e38):
        assert fn(p, p, p, p, p, None, 1, 1, 8, 40, 1, scale) == -1 and "scale" in br.last_error()
        assert bwd(*[p] * 9, None, 1, 1, 8, 40, 1, scale) == -1
    c.scale, c.q = 2.3e38, np.zeros_like(c.q)
    o, _ = A.forward(br, c)
    v = c.f64(c.v)[0]
    n = np.arange(1, 41)
    want, off = v.cumsum(1) / n, 48 * A.E32 * np.abs(v).cumsum(1) / n
    assert np.all(np.abs(c.f64(o)[0] - want) <= off + A.STEP[storage] * (np.abs(want) + off))
