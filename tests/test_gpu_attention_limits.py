"""Attention at the ends of what it takes: the longest rows, the most workgroups, the same tensor for several inputs, another stream, and
recorded graphs that share the workspace.  Bounds: test_gpu_attention.py's."""
import ctypes

import numpy as np
import pytest

import test_gpu_attention as A

pytestmark = pytest.mark.gpu


class Rows:
    """[rows][S] on the device, zeros but for some columns."""

    def __init__(self, br, rows, S, dtype):
        self.br, self.rows, self.S = br, rows, S
        self.dev = br.DevArray((rows, S), dtype)
        self.ptr = self.dev.ptr

    def put(self, lo, a):
        for r in range(self.rows):
            row = np.ascontiguousarray(a[r])
            self.br.lib.mi355_buf_write(self.dev.handle, (r * self.S + lo) * row.itemsize, row.ctypes.data, row.nbytes)

    def get(self, lo, n):
        out = np.empty((self.rows, n), self.dev.dtype)
        for r in range(self.rows):
            self.br.lib.mi355_buf_read(self.dev.handle, (r * self.S + lo) * out.itemsize, out[r].ctypes.data, out[r].nbytes)
        return out


@pytest.mark.parametrize("storage,S", [("f32", 1 << 22), ("bf16", 1 << 22), ("bf16", (1 << 22) - 3)])
def test_rows_of_four_million(br, storage, S):
    """128 channels of 2^22 positions (2 GiB a tensor in fp32), packed from sequences of a hundred: the first, one in the middle and the last."""
    hd, dtype = 128, np.float32 if storage == "f32" else np.uint16
    cu = np.append(np.arange(0, S - 150, 100), S).astype(np.int32)
    seqs = [0, len(cu) // 2, len(cu) - 2]
    cases = [A.Case(storage, 1, 1, hd, int(cu[s + 1] - cu[s]), 1, seed=90 + s) for s in seqs]
    q, k, v, do, o, dq, dk, dv = (Rows(br, hd, S, dtype) for _ in range(8))
    lse = Rows(br, 1, S, np.float32)
    for s, c in zip(seqs, cases):
        for t, a in ((q, c.q), (k, c.k), (v, c.v), (do, c.do)):
            t.put(cu[s], a[0])
    cud, bounds = br.DevArray.from_numpy(cu), br.DevArray((2, S), np.int32)
    br.check(br.lib.mi355_attn_plan_dev(bounds.ptr, cud.ptr, len(cu) - 1, S, 1))
    end = "_dev" if storage == "f32" else "_bf16_dev"
    shape = (1, 1, hd, S, 1, cases[0].scale)
    br.check(getattr(br.lib, "mi355_attn_fwd" + end)(o.ptr, lse.ptr, q.ptr, k.ptr, v.ptr, bounds.ptr, *shape))
    br.check(getattr(br.lib, "mi355_attn_bwd" + end)(dq.ptr, dk.ptr, dv.ptr, do.ptr, q.ptr, k.ptr, v.ptr, o.ptr, lse.ptr, bounds.ptr, *shape))
    for s, c in zip(seqs, cases):
        lo, n = int(cu[s]), c.S
        got_o, got_l = o.get(lo, n)[None], lse.get(lo, n)[None]
        A.check(c, dict(o=got_o, lse=got_l), A.reference(c))
        A.check(c, {m: t.get(lo, n)[None] for m, t in (("dq", dq), ("dk", dk), ("dv", dv))}, A.reference(c, got_o, got_l))
    for t in (o, dq, dk, dv):                   # sequences of zeros
        assert not t.get(int(cu[7]), 300).any() and not t.get(int(cu[-5]), 300).any()


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_as_many_workgroups_as_a_launch_numbers(br, storage):
    """2^24 - 1 rows of one position: o is v, dv is do, dq and dk are zero (test_a_single_key has the bounds)."""
    n = (1 << 24) - 1
    c = A.Case(storage, 1, 1, 1, 1, 1)
    rng = np.random.default_rng(95)
    draw = lambda: c.stored(rng.standard_normal(n, np.float32))         # noqa: E731
    D = br.DevArray.from_numpy
    qh, kh, vh, gh = draw(), draw(), draw(), draw()
    q, k, v, g = D(qh), D(kh), D(vh), D(gh)
    o, lse, dq, dk, dv = br.DevArray(n, c.q.dtype), br.DevArray(n), D(vh), D(vh), br.DevArray(n, c.q.dtype)
    end = "_dev" if storage == "f32" else "_bf16_dev"
    br.check(getattr(br.lib, "mi355_attn_fwd" + end)(o.ptr, lse.ptr, q.ptr, k.ptr, v.ptr, None, 1, 1, 1, 1, n, 1.0))
    br.check(getattr(br.lib, "mi355_attn_bwd" + end)(dq.ptr, dk.ptr, dv.ptr, g.ptr, q.ptr, k.ptr, v.ptr, o.ptr, lse.ptr, None, 1, 1, 1, 1, n, 1.0))
    V, G = c.f64(vh), c.f64(gh)
    assert np.all(np.abs(c.f64(o.numpy()) - V) <= (4 * A.E32 * np.abs(V) if storage == "f32" else 0.0))
    z = c.f64(qh) * c.f64(kh)
    assert np.all(np.abs(lse.numpy() - z) <= 8 * A.E32 * np.abs(z) + 2.0 ** -126)
    assert not c.f64(dq.numpy()).any() and not c.f64(dk.numpy()).any()
    assert np.all(np.abs(c.f64(dv.numpy()) - G) <= (2.0 ** -14 + 2 * A.STEP[storage]) * np.abs(G))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("S", [130, 136])
def test_one_tensor_for_q_k_and_v(br, storage, S):
    """Inputs may be the same memory: the same bits as from copies."""
    c = A.Case(storage, 2, 2, 64, S, 2, [[0, 60, 125]] * 2, seed=96)
    c.k = c.v = c.q
    o, lse = A.forward(br, c)
    g = A.backward(br, c, o, lse)
    D = br.DevArray.from_numpy
    x, do, bounds = D(c.q), D(c.do), A.plan_dev(br, c)
    od, ld = D(c.stored(np.full(c.q.shape, 7.0))), D(np.full(lse.shape, 7.0, np.float32))
    outs = [D(c.stored(np.full(c.q.shape, 7.0))) for _ in range(3)]
    end, shape = "_dev" if storage == "f32" else "_bf16_dev", (2, 2, 64, S, 2, c.scale)
    br.check(getattr(br.lib, "mi355_attn_fwd" + end)(od.ptr, ld.ptr, x.ptr, x.ptr, x.ptr, bounds.ptr, *shape))
    br.check(getattr(br.lib, "mi355_attn_bwd" + end)(*[t.ptr for t in outs], do.ptr, x.ptr, x.ptr, x.ptr, od.ptr, ld.ptr, bounds.ptr, *shape))
    assert np.array_equal(od.numpy(), o) and np.array_equal(ld.numpy(), lse)
    assert all(np.array_equal(t.numpy(), g[n]) for t, n in zip(outs, ("dq", "dk", "dv")))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_another_stream(br, storage):
    c = A.Case(storage, 4, 2, 96, 205, 2, [[0, 90, 200]] * 2, seed=97)
    o, lse = A.forward(br, c)
    g = A.backward(br, c, o, lse)
    hip = br.lib                # (the runtime that the library itself has loaded, whatever else the process has)
    stream = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    br.check(br.lib.mi355_set_stream(stream))
    try:
        o2, lse2 = A.forward(br, c)
        g2 = A.backward(br, c, o, lse)
    finally:
        br.check(br.lib.mi355_set_stream(None))         # (waits for the other one)
        assert hip.hipStreamDestroy(stream) == 0
    assert np.array_equal(o, o2) and np.array_equal(lse, lse2) and all(np.array_equal(g[n], g2[n]) for n in g)


def test_graphs_that_share_the_workspace(br):
    """Two recorded graphs whose copies and sums lie in the same workspace, replayed in turn, with eager calls between."""
    from test_gpu_linear import SILU
    c = A.Case("bf16", 4, 2, 64, 197, 2, [[0, 90, 190]] * 2, seed=98)
    o, lse = A.forward(br, c)
    g = A.backward(br, c, o, lse)
    rng = np.random.default_rng(99)
    M, K, S, B = 100, 150, 33, 40
    D = br.DevArray.from_numpy
    x, w, dy = (D(A.to_bf16(rng.standard_normal(s))) for s in ((B, K, S), (M, K), (B, M, S)))
    y, dx, dw, db = br.DevArray((B, M, S), np.uint16), br.DevArray((B, K, S), np.uint16), br.DevArray((M, K)), br.DevArray(M)
    q, k, v, do, bounds = D(c.q), D(c.k), D(c.v), D(c.do), A.plan_dev(br, c)
    od, ld, outs = D(c.stored(np.full(c.q.shape, 7.0))), D(np.full(lse.shape, 7.0, np.float32)), [D(c.stored(np.full(a.shape, 7.0))) for a in (c.q, c.k, c.v)]
    shape = (c.heads, c.kv, c.hd, c.S, c.batch, c.scale)

    def attention():
        br.check(br.lib.mi355_attn_fwd_bf16_dev(od.ptr, ld.ptr, q.ptr, k.ptr, v.ptr, bounds.ptr, *shape))
        br.check(br.lib.mi355_attn_bwd_bf16_dev(*[t.ptr for t in outs], do.ptr, q.ptr, k.ptr, v.ptr, od.ptr, ld.ptr, bounds.ptr, *shape))

    def linear():
        br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, None, x.ptr, w.ptr, None, SILU, None, 1.0, M, K, S, B))
        br.check(br.lib.mi355_linear_bwd_bf16_dev(dx.ptr, dw.ptr, db.ptr, dy.ptr, x.ptr, w.ptr, 1.0, 0, None, 0, M, K, S, B))

    linear()
    want = [t.numpy() for t in (y, dx, dw, db)]
    graphs = []
    for calls in (attention, linear):
        br.check(br.lib.mi355_graph_begin())
        calls()
        graphs.append(br.lib.mi355_graph_end())
        assert graphs[-1]
    for turn in range(4):
        for t in (y, dx, dw, db):
            t.zero()
        for i in ((0, 1), (1, 0), (0, 0, 1, 1), (1, 0, 1))[turn]:
            br.check(br.lib.mi355_graph_launch(graphs[i]))
        assert all(np.array_equal(t.numpy(), a) for t, a in zip((y, dx, dw, db), want))
        assert np.array_equal(od.numpy(), o) and np.array_equal(ld.numpy(), lse) and all(np.array_equal(t.numpy(), g[n]) for t, n in zip(outs, ("dq", "dk", "dv")))
        linear() if turn % 2 else attention()
    for h in graphs:
        br.lib.mi355_graph_free(h)
