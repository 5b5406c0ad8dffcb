"""Causal attention over packed rows, both directions, against the formulas in 64 bits.

Tolerances are bounds, element by element, from the magnitudes that enter a value: a sum of n products in fp32 is off by at most
n * 2^-24 of the sum of their magnitudes, exp by its argument's error, and each rounding to bfloat16 by 2^-8 of what is rounded
(scores' weights and score gradients once, results once)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
STEP = {"f32": E32, "bf16": 2.0 ** -8}


def to_bf16(a):
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


class Case:
    def __init__(self, storage, heads, kv, hd, S, batch, cu=None, seed=0, spread=1.0):
        self.storage, self.heads, self.kv, self.hd, self.S, self.batch = storage, heads, kv, hd, S, batch
        self.cu = None if cu is None else np.asarray(cu, np.int32).reshape(batch, -1)
        self.scale = float(np.float32(1.0 / np.sqrt(hd)))
        rng = np.random.default_rng(seed)
        self.q, self.do = (self.stored(spread * rng.standard_normal((batch, heads * hd, S))) for _ in range(2))
        self.k, self.v = (self.stored(spread * rng.standard_normal((batch, kv * hd, S))) for _ in range(2))

    def stored(self, a):
        return np.asarray(a, np.float32) if self.storage == "f32" else to_bf16(a)

    def f64(self, a):
        return (a if a.dtype == np.float32 else from_bf16(a)).astype(np.float64)

    def plan(self):
        """(start, end) [batch][S] by definition."""
        start = np.zeros((self.batch, self.S), np.int64)
        end = np.full((self.batch, self.S), self.S, np.int64)
        if self.cu is not None:
            start[:], end[:] = self.S, 0
            for b in range(self.batch):
                for lo, hi in zip(self.cu[b, :-1], self.cu[b, 1:]):
                    start[b, lo:hi], end[b, lo:hi] = lo, hi
        return start, end

    def allowed(self, b):
        start, _ = self.plan()
        s = np.arange(self.S)
        return (s[None, :] <= s[:, None]) & (s[None, :] >= start[b][:, None])


def reference(c, o=None, lse=None):
    """Forward (o, lse) or, given them, the gradients, with their bounds: dicts of [value, bound]."""
    G, hd, S, eps = c.heads // c.kv, c.hd, c.S, STEP[c.storage]
    q, k, v, do = (c.f64(a) for a in (c.q, c.k, c.v, c.do))
    out = {}

    def put(name, b, rows, value, bound):
        val, bnd = out.setdefault(name, (np.zeros((c.batch, {"lse": c.heads}.get(name, 0) or (c.kv if name in ("dk", "dv") else c.heads) * hd, S)),
                                         np.zeros((c.batch, {"lse": c.heads}.get(name, 0) or (c.kv if name in ("dk", "dv") else c.heads) * hd, S))))
        val[b, rows] += value
        bnd[b, rows] += bound

    for b in range(c.batch):
        ok = c.allowed(b)
        n = S + 16
        for h in range(c.heads):
            rq, rk = slice(h * hd, (h + 1) * hd), slice(h // G * hd, (h // G + 1) * hd)
            Q, K, V, dO = q[b, rq], k[b, rk], v[b, rk], do[b, rq]
            z = np.where(ok, c.scale * (Q.T @ K), -np.inf)
            dz = E32 * (hd + 6) * c.scale * (np.abs(Q).T @ np.abs(K))       # error of a score, and of the exponent made of it
            if o is None:
                m = np.max(z, axis=1, keepdims=True)
                m = np.where(np.isfinite(m), m, 0.0)
                e = np.exp(z - m)
                tot = e.sum(1, keepdims=True)
                p = e / np.where(tot == 0, 1.0, tot)
                row = (np.where(ok, dz, 0.0).max(1) * 2 + E32 * (n + 2 * np.abs(np.where(ok, z, 0.0)).max(1)))      # relative, of a row's weights
                pv = p @ np.abs(V).T
                val = (p @ V.T).T
                put("o", b, rq, val, (pv * (2 * row[:, None] + E32 * n + (eps if c.storage == "bf16" else 0.0))).T * 1.01 + 1.01 * eps * np.abs(val))
                with np.errstate(divide="ignore"):
                    le = (m + np.log(tot))[:, 0]
                put("lse", b, h, np.where(np.isfinite(le), le, 0.0), row + 4 * E32 * (1 + np.abs(np.where(np.isfinite(le), le, 0.0))))
                continue
            used = ok.any(1)
            L = np.where(used, lse[b, h].astype(np.float64), 0.0)
            O = np.where(used[None], c.f64(o)[b, rq], 0.0)
            dO = np.where(used[None], dO, 0.0)
            p = np.where(ok, np.exp(np.where(ok, z, 0.0) - L[:, None]), 0.0)
            rel = dz + 4 * E32 * (np.abs(np.where(ok, z, 0.0)) + np.abs(L)[:, None] + 4)
            delta = (dO * O).sum(0)
            g = dO.T @ V - delta[:, None]
            g_off = E32 * (hd + 4) * (np.abs(dO).T @ np.abs(V) + (np.abs(dO) * np.abs(O)).sum(0)[:, None] * 2)
            ds = p * g
            extra = eps if c.storage == "bf16" else 0.0
            ds_off = np.abs(ds) * (rel + extra + E32 * n) + p * g_off * 1.01
            p_off = p * (rel + extra + E32 * n)
            put("dq", b, rq, c.scale * (ds @ K.T).T, c.scale * (ds_off @ np.abs(K).T).T * 1.02)
            put("dk", b, rk, c.scale * (ds.T @ Q.T).T, c.scale * (ds_off.T @ np.abs(Q).T).T * 1.02)
            put("dv", b, rk, (p.T @ dO.T).T, (p_off.T @ np.abs(dO).T).T * 1.02)
    if o is not None:
        for name, (val, bnd) in out.items():
            bnd += 1.01 * eps * np.abs(val) + 2.0 ** -126 * (2.0 ** 16 if c.storage == "bf16" else 1)
    return out


def plan_dev(br, c):
    if c.cu is None:
        return None
    cu, bounds = br.DevArray.from_numpy(c.cu), br.DevArray((c.batch, 2, c.S), np.int32)
    br.check(br.lib.mi355_attn_plan_dev(bounds.ptr, cu.ptr, c.cu.shape[1] - 1, c.S, c.batch))
    bounds.cu = cu
    return bounds


def forward(br, c, fill=7.0, bounds=None, want_lse=True):
    D = br.DevArray.from_numpy
    q, k, v = D(c.q), D(c.k), D(c.v)
    o = D(c.stored(np.full(c.q.shape, fill)))
    lse = D(np.full((c.batch, c.heads, c.S), fill, np.float32)) if want_lse else None
    bounds = bounds or plan_dev(br, c)
    fn = br.lib.mi355_attn_fwd_dev if c.storage == "f32" else br.lib.mi355_attn_fwd_bf16_dev
    br.check(fn(o.ptr, lse.ptr if lse else None, q.ptr, k.ptr, v.ptr, bounds.ptr if bounds else None, c.heads, c.kv, c.hd, c.S, c.batch, c.scale))
    return o.numpy(), lse.numpy() if lse else None


def backward(br, c, o, lse, fill=7.0):
    D = br.DevArray.from_numpy
    args = [D(c.stored(np.full(a.shape, fill))) for a in (c.q, c.k, c.v)] + [D(a) for a in (c.do, c.q, c.k, c.v, o, lse)]
    bounds = plan_dev(br, c)
    fn = br.lib.mi355_attn_bwd_dev if c.storage == "f32" else br.lib.mi355_attn_bwd_bf16_dev
    br.check(fn(*[a.ptr for a in args], bounds.ptr if bounds else None, c.heads, c.kv, c.hd, c.S, c.batch, c.scale))
    return {n: a.numpy() for n, a in zip(("dq", "dk", "dv"), args)}


def check(c, got, want, fill=7.0):
    _, end = c.plan()
    for name, (val, bound) in want.items():
        a = got[name]
        a = a.astype(np.float64) if a.dtype == np.float32 else from_bf16(a).astype(np.float64)
        used = np.broadcast_to((end > 0)[:, None, :], a.shape)
        assert np.all(a[~used] == fill), name + ": a column of no sequence was written"
        off = np.abs(a - val) - bound
        assert not np.any(~(off[used] <= 0)), (name, float(np.nanmax(np.where(used, off, -np.inf))), np.argwhere(used & ~(off <= 0))[:3])


CASES = [
    # heads, kv, hd, S, batch, offsets
    (1, 1, 64, 1, 1, None), (2, 1, 64, 2, 3, None), (1, 1, 1, 5, 1, None), (3, 3, 7, 33, 2, None), (12, 12, 64, 256, 1, None),
    (4, 2, 128, 256, 2, None), (2, 2, 72, 197, 2, None), (6, 1, 96, 130, 1, None), (4, 2, 128, 129, 1, None), (2, 1, 100, 64, 2, None),
    (2, 1, 128, 511, 1, [0, 1, 2, 130, 130, 400]),                      # of one position, of none, the end unused
    (4, 4, 64, 320, 2, [[0, 64, 128, 192], [5, 100, 101, 320]]),        # on tile borders, and one that begins late
    (2, 2, 40, 100, 3, [[0, 100], [0, 37], [0, 0]]),                    # a padded batch, one row of it empty
    (64, 64, 64, 300, 4, [[0, 31, 32, 33, 290]] * 4),                   # enough workgroups for the widest tiles
    (64, 16, 128, 270, 5, None),
]


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward_and_gradients(br, i, storage):
    c = Case(storage, *CASES[i], seed=i)
    o, lse = forward(br, c)
    check(c, dict(o=o, lse=lse), reference(c))
    check(c, backward(br, c, o, lse), reference(c, o, lse))


def test_plan(br):
    cu = np.array([[0, 0, 3, 3, 10, 12], [2, 5, 5, 5, 9, 9], [0, 0, 0, 0, 0, 0]], np.int32)
    c = Case("f32", 1, 1, 4, 12, 3, cu)
    start, end = c.plan()
    assert np.array_equal(plan_dev(br, c).numpy(), np.stack([start, end], 1))


def test_plan_of_bad_offsets_stays_inside(br):
    """Offsets that descend or leave the row give some plan, and one that the kernels can be run with."""
    for cu in ([-5, 3, 900], [50, 10, 0], [7, 7, 2 ** 31 - 1], [-2 ** 31, -1, 5]):
        c = Case("bf16", 2, 1, 64, 100, 1, [cu])
        plan = plan_dev(br, c)
        p = plan.numpy()
        assert p.min() >= 0 and p.max() <= 100
        o, lse = forward(br, c, bounds=plan)
        backward(br, c, o, lse)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd,S,cu", [(64, 300, [[0, 70, 71, 200, 260]]), (128, 140, [[3, 40, 140]]), (96, 1030, [[0, 0, 1000]])])
def test_what_the_mask_hides_is_not_seen(br, storage, bad, hd, S, cu):
    """Infinities and NaNs in another sequence, behind the last one and in later positions leave a result as it is, to the bit."""
    c = Case(storage, 4, 2, hd, S, 1, cu, seed=3)
    lo, hi = cu[0][1], cu[0][2]         # the sequence that is looked at
    late = hi - 5                       # its positions from here on are spoilt too
    o, lse = forward(br, c)
    seen = np.arange(lo, late)
    spoilt = np.array([s for s in range(S) if s < lo or s >= late])
    names = ("q", "k", "v", "do")
    clean = {n: getattr(c, n).copy() for n in names}
    for n in names:
        a = clean[n].copy()
        a[:, :, spoilt] = c.stored(np.full(1, bad))[0]
        setattr(c, n, a)
    o2, lse2 = forward(br, c)
    assert np.array_equal(o2[:, :, seen], o[:, :, seen]) and np.array_equal(lse2[:, :, seen], lse[:, :, seen])
    # gradients: dq of a position sees earlier ones only; dk and dv see later ones, so there the others alone are spoilt
    for n in names:
        setattr(c, n, clean[n])
    g = backward(br, c, o, lse)
    for n in names:
        a = clean[n].copy()
        a[:, :, spoilt] = c.stored(np.full(1, bad))[0]
        setattr(c, n, a)
    o_s, lse_s = o.copy(), lse.copy()
    o_s[:, :, spoilt], lse_s[:, :, spoilt] = c.stored(np.full(1, bad))[0], bad
    g2 = backward(br, c, o_s, lse_s)
    assert np.array_equal(g2["dq"][:, :, seen], g["dq"][:, :, seen])
    others = np.array([s for s in range(S) if s < lo or s >= hi])
    for n in names:
        a = clean[n].copy()
        a[:, :, others] = c.stored(np.full(1, bad))[0]
        setattr(c, n, a)
    o_s, lse_s = o.copy(), lse.copy()
    o_s[:, :, others], lse_s[:, :, others] = c.stored(np.full(1, bad))[0], bad
    g3 = backward(br, c, o_s, lse_s)
    for n in ("dq", "dk", "dv"):
        assert np.array_equal(g3[n][:, :, lo:hi], g[n][:, :, lo:hi]), n


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_a_value_that_counts_is_seen(br, storage):
    """A NaN among a sequence's own values reaches every position from there on, and none before; nor one head another's."""
    c = Case(storage, 2, 2, 64, 100, 1, seed=4)
    o, _ = forward(br, c)
    c.v[0, 5, 60] = c.stored(np.full(1, np.nan))[0]
    o2, _ = forward(br, c)
    v2 = o2 if storage == "f32" else from_bf16(o2)
    assert np.all(np.isnan(v2[0, 5, 60:])) and np.array_equal(o2[0, 5, :60], o[0, 5, :60])
    rest = [r for r in range(128) if r != 5]
    assert np.array_equal(o2[0, rest], o[0, rest])


def test_scores_of_any_size(br):
    """Scores whose exponentials overflow, and rows of equal ones."""
    c = Case("f32", 1, 1, 64, 80, 1, seed=5, spread=12.0)       # scores in the hundreds
    c.q[:, :, 10] = 0.0                                         # equal scores: the mean of the values
    o, lse = forward(br, c)
    assert np.all(np.isfinite(o)) and np.all(np.isfinite(lse))
    assert np.allclose(o[0, :, 10], c.v[0, :, :11].mean(1), atol=1e-4 * 12)
    want = reference(c)
    check(c, dict(o=o, lse=lse), want)


def test_gradients_match_differences(br):
    """dq, dk, dv along random directions against differences of the loss <do, o> in 64 bits."""
    c = Case("f32", 2, 1, 16, 40, 1, [[0, 25, 40]], seed=6)
    o, lse = forward(br, c)
    g = backward(br, c, o, lse)
    rng = np.random.default_rng(7)

    def loss(dq, dk, dv):
        q, k, v = c.q.astype(np.float64) + dq, c.k.astype(np.float64) + dk, c.v.astype(np.float64) + dv
        total, ok = 0.0, c.allowed(0)
        for h in range(2):
            rq = slice(16 * h, 16 * h + 16)
            z = np.where(ok, c.scale * (q[0, rq].T @ k[0]), -np.inf)
            e = np.exp(z - z.max(1, keepdims=True))
            total += np.sum((e / e.sum(1, keepdims=True) @ v[0].T).T * c.do[0, rq])
        return total

    for n, shape in (("dq", c.q.shape), ("dk", c.k.shape), ("dv", c.v.shape)):
        d = rng.standard_normal(shape)
        arg = {m: d * (m == n) if m == n else 0.0 for m in ("dq", "dk", "dv")}
        h = 1e-5
        num = (loss(**{m: h * a for m, a in arg.items()}) - loss(**{m: -h * a for m, a in arg.items()})) / (2 * h)
        # fp32 sums of the gradient against differences that are good to about h^2
        assert abs(np.sum(g[n].astype(np.float64) * d) - num) < 2e-5 * np.sum(np.abs(g[n] * d)) + 1e-6, n


def test_rows_that_begin_anywhere(br):
    """Tensors at any element and rows of any length give what aligned ones do."""
    for storage, shift in (("bf16", 1), ("bf16", 3), ("f32", 1)):
        c = Case(storage, 2, 1, 64, 136, 1, seed=8)
        o, lse = forward(br, c)
        D, size = br.DevArray.from_numpy, c.q.dtype.itemsize
        off = [D(np.concatenate([np.zeros(shift, a.dtype), a.ravel()])) for a in (c.q, c.k, c.v, np.zeros_like(c.q))]
        fn = br.lib.mi355_attn_fwd_dev if storage == "f32" else br.lib.mi355_attn_fwd_bf16_dev
        br.check(fn(off[3].ptr + shift * size, None, off[0].ptr + shift * size, off[1].ptr + shift * size, off[2].ptr + shift * size, None, 2, 1, 64, 136, 1, c.scale))
        assert np.array_equal(off[3].numpy()[shift:].reshape(o.shape), o)


def test_refusals(br):
    D = br.DevArray((4096,))
    p, lib = D.ptr, br.lib
    ok = [p, p, p, p, p, None, 2, 1, 8, 4, 1, 1.0]
    for i, v in ((0, None), (2, None), (3, None), (4, None), (6, 0), (7, 0), (7, 3), (8, 0), (8, 129), (9, 0), (9, -1), (9, 2 ** 23), (10, 0), (11, 0.0),
                 (11, -1.0), (11, float("nan")), (11, float("inf")), (10, 2 ** 30)):
        for fn in (lib.mi355_attn_fwd_dev, lib.mi355_attn_fwd_bf16_dev):
            a = list(ok)
            a[i] = v
            assert fn(*a) == -1, (i, v)
            assert br.last_error()
    bwd = [p] * 9 + [None, 2, 1, 8, 4, 1, 1.0]
    for i, v in [(j, None) for j in range(9)] + [(10, 0), (11, 3), (12, 200), (13, 0), (14, 0), (15, 0.0)]:
        for fn in (lib.mi355_attn_bwd_dev, lib.mi355_attn_bwd_bf16_dev):
            a = list(bwd)
            a[i] = v
            assert fn(*a) == -1, (i, v)
    for a in ((None, p, 1, 4, 1), (p, None, 1, 4, 1), (p, p, 0, 4, 1), (p, p, 1, 0, 1), (p, p, 1, 4, 0), (p, p, 1, 4, 70000)):
        assert lib.mi355_attn_plan_dev(*a) == -1


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_replayed_graph(br, storage):
    """Forward and backward recorded into a graph, with other work between the replays."""
    c = Case(storage, 4, 2, 64, 200, 2, [[0, 90, 200]] * 2, seed=9)
    o, lse = forward(br, c)
    g = backward(br, c, o, lse)
    D = br.DevArray.from_numpy
    q, k, v, do = (D(a) for a in (c.q, c.k, c.v, c.do))
    bounds = plan_dev(br, c)
    od, ld = D(np.zeros_like(o)), br.DevArray(lse.shape)
    outs = [D(np.zeros_like(a)) for a in (c.q, c.k, c.v)]
    end = "_dev" if storage == "f32" else "_bf16_dev"
    shape = (c.heads, c.kv, c.hd, c.S, c.batch, c.scale)
    br.check(br.lib.mi355_graph_begin())
    br.check(getattr(br.lib, "mi355_attn_fwd" + end)(od.ptr, ld.ptr, q.ptr, k.ptr, v.ptr, bounds.ptr, *shape))
    br.check(getattr(br.lib, "mi355_attn_bwd" + end)(*[a.ptr for a in outs], do.ptr, q.ptr, k.ptr, v.ptr, od.ptr, ld.ptr, bounds.ptr, *shape))
    graph = br.lib.mi355_graph_end()
    assert graph
    for _ in range(3):
        for a in outs + [od]:
            a.zero()
        br.check(br.lib.mi355_graph_launch(graph))
        assert np.array_equal(od.numpy(), o) and np.array_equal(ld.numpy(), lse)
        for a, n in zip(outs, ("dq", "dk", "dv")):
            assert np.array_equal(a.numpy(), g[n])
        other = Case(storage, 4, 2, 64, 200, 2, [[0, 90, 200]] * 2, seed=10)
        forward(br, other)
    br.lib.mi355_graph_free(graph)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(4, 2, 64, 1, 5, None), (2, 2, 128, 70, 1, list(range(71))), (3, 1, 96, 40, 2, [[0, 1, 2, 2, 40], [7, 8, 39, 40, 40]]),
                                   (128, 128, 72, 3, 8, [[0, 1, 2, 3]] * 8)])
def test_a_single_key(br, storage, shape):
    """A query with one key has a weight of 1 whatever its score: exactly no gradient for it, nor for a key that no other query has; dv is do
    times exp of what the score's and lse's rounding leave (a few units of 2^-24 of a score below 2^6, so 2^-14), rounded."""
    heads, kv, hd, S, batch, cu = shape
    c = Case(storage, heads, kv, hd, S, batch, cu, seed=11)
    o, lse = forward(br, c)
    g = backward(br, c, o, lse)
    start, end = c.plan()
    for b in range(batch):
        s = np.arange(S)
        first, alone = start[b] == s, (start[b] == s) & (end[b] == s + 1)
        assert alone.any()
        assert not np.any(c.f64(g["dq"])[b][:, first]) and not np.any(c.f64(g["dk"])[b][:, alone])
        # o = (p v) * (1 / p): three roundings of fp32 (each 2^-24 of the value), and 2^-22 in all is lost again when v itself has eight bits
        v = c.f64(np.repeat(c.v[b].reshape(kv, hd, S), heads // kv, 0).reshape(heads * hd, S)[:, first])
        assert np.all(np.abs(c.f64(o)[b][:, first] - v) <= (4 * E32 * np.abs(v) if storage == "f32" else 0.0))
        do = c.f64(c.do)[b].reshape(kv, heads // kv, hd, S)
        off = np.abs(c.f64(g["dv"])[b].reshape(kv, hd, S) - do.sum(1))[..., alone]
        assert np.all(off <= ((2.0 ** -14 + 2 * STEP[storage]) * np.abs(do).sum(1))[..., alone])


def test_more_than_a_launch_numbers_is_refused(br):
    p = br.DevArray((4096,)).ptr
    for fn in (br.lib.mi355_attn_fwd_dev, br.lib.mi355_attn_fwd_bf16_dev):
        for heads, S, batch in ((1, 1, 1 << 24), (1 << 12, 64, 1 << 12), (64, 1 << 22, 4)):
            assert fn(p, p, p, p, p, None, heads, 1, 1, S, batch, 1.0) == -1 and br.last_error()
    for fn in (br.lib.mi355_attn_bwd_dev, br.lib.mi355_attn_bwd_bf16_dev):
        assert fn(*[p] * 9, None, 1, 1, 1, 1, 1 << 24, 1.0) == -1 and br.last_error()
    assert br.lib.mi355_act_bwd_bf16_dev(p, p, p, 1.0, 0, 1 << 35) == -1 and br.last_error()
