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
