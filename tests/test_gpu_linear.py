"""The products of a layer with their epilogues, both directions, against the formulas in 64 bits.

Tolerances are bounds, element by element: a sum of n products in fp32 is off by at most n * 2^-24 of the sum of their magnitudes, an
activation by its slope (at most 1.13) times its argument's error and 2^-19 of its argument's size, a bfloat16 result by 2^-8 of itself."""
import numpy as np
import pytest

from test_gpu_attention import E32, from_bf16, to_bf16

pytestmark = pytest.mark.gpu

NONE, RELU, SILU, GELU = range(4)
TINY = 2.0 ** -110      # below it a bfloat16 has lost bits


def act(a, z):
    with np.errstate(over="ignore"):
        if a == RELU:
            return np.maximum(z, 0.0)
        if a == SILU:
            return z / (1.0 + np.exp(-z))
        if a == GELU:
            return 0.5 * z * (1.0 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(a, z):
    if a == RELU:
        return (z > 0).astype(np.float64)
    if a == SILU:
        g = 1.0 / (1.0 + np.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    if a == GELU:
        c = np.sqrt(2 / np.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return np.ones_like(z)


def close(got, want, bound):
    got = from_bf16(got) if got.dtype == np.uint16 else got
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], float(np.nanmax(np.abs(got - want) - bound)))


def run_forward(br, x, w, bias, a, res, alpha, pre=True):
    (B, K, S), M = x.shape, w.shape[0]
    D = br.DevArray.from_numpy
    y = br.DevArray((B, M, S), np.uint16)
    z = br.DevArray((B, M, S), np.uint16) if pre else None
    xd, wd, bd, rd = D(x), D(w), D(bias) if bias is not None else None, D(res) if res is not None else None
    br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, z.ptr if z else None, xd.ptr, wd.ptr, bd.ptr if bd else None, a, rd.ptr if rd else None, alpha, M, K, S, B))
    return y.numpy(), z.numpy() if z else None


def check_forward(br, M, K, S, B, a, with_bias, with_res, seed):
    rng = np.random.default_rng(seed)
    x, w = to_bf16(rng.standard_normal((B, K, S))), to_bf16(rng.standard_normal((M, K)) / np.sqrt(K))
    bias = rng.standard_normal(M).astype(np.float32) if with_bias else None
    res = to_bf16(rng.standard_normal((B, M, S))) if with_res else None
    alpha = float(np.float32(0.3)) if with_res else 1.0
    X, W = from_bf16(x).astype(np.float64), from_bf16(w).astype(np.float64)
    b = 0.0 if bias is None else bias.astype(np.float64)[:, None]
    z = W @ X + b
    dz = E32 * (K + 4) * (np.abs(W) @ np.abs(X) + np.abs(b))
    y = alpha * act(a, z) + (0.0 if res is None else from_bf16(res).astype(np.float64))
    got, pre = run_forward(br, x, w, bias, a, res, alpha)
    close(pre, z, dz + 2.0 ** -8 * (np.abs(z) + dz) + TINY)
    off = alpha * (1.13 * dz + 2.0 ** -19 * np.abs(z) * (a != NONE)) + 2 * E32 * (np.abs(y) + alpha * np.abs(z))
    close(got, y, off + 2.0 ** -8 * (np.abs(y) + off) + TINY)


def check_backward(br, M, K, S, B, a, accumulate, seed, parts=("dx", "dw", "dbias")):
    rng = np.random.default_rng(seed)
    x, w, dy = to_bf16(rng.standard_normal((B, K, S))), to_bf16(rng.standard_normal((M, K)) / np.sqrt(K)), to_bf16(rng.standard_normal((B, M, S)))
    pre = to_bf16(2 * rng.standard_normal((B, K, S)))
    alpha = float(np.float32(0.7))
    dw0, db0 = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal(M).astype(np.float32)
    D = br.DevArray.from_numpy
    dx, dw, db = br.DevArray((B, K, S), np.uint16), D(dw0), D(db0)
    keep = [D(t) for t in (dy, x, w, pre)]
    br.check(br.lib.mi355_linear_bwd_bf16_dev(dx.ptr if "dx" in parts else None, dw.ptr if "dw" in parts else None, db.ptr if "dbias" in parts else None,
                                              keep[0].ptr, keep[1].ptr, keep[2].ptr, alpha, a, keep[3].ptr if a else None, accumulate, M, K, S, B))
    X, W, G, P = (from_bf16(t).astype(np.float64) for t in (x, w, dy, pre))
    if "dx" in parts:
        want = alpha * (W.T @ G) * slope(a, P)
        off = alpha * (E32 * (M + 6) * 1.13 + 2.0 ** -19 * (a != NONE)) * (np.abs(W).T @ np.abs(G)) * (1 + np.abs(P) * (a != NONE))
        close(dx.numpy(), want, off + 2.0 ** -8 * (np.abs(want) + off) + TINY)
    n = B * S
    if "dw" in parts:
        want = alpha * np.einsum("bms,bks->mk", G, X) + (dw0 if accumulate else 0.0)
        off = E32 * (n + 6) * np.einsum("bms,bks->mk", np.abs(G), np.abs(X)) + 2 * E32 * (np.abs(want) + np.abs(dw0))
        close(dw.numpy(), want, off)
    else:
        assert np.array_equal(dw.numpy(), dw0)
    if "dbias" in parts:
        want = alpha * G.sum((0, 2)) + (db0 if accumulate else 0.0)
        close(db.numpy(), want, E32 * (n + 6) * np.abs(G).sum((0, 2)) + 2 * E32 * (np.abs(want) + np.abs(db0)))
    else:
        assert np.array_equal(db.numpy(), db0)


SHAPES = [  # M, K, S, batch
    (1, 1, 1, 1), (5, 3, 2, 1), (64, 64, 64, 1), (65, 63, 7, 3), (128, 200, 1, 1), (300, 520, 1, 1), (96, 1024, 3, 2), (256, 136, 1, 9),
    (130, 72, 197, 2), (768, 768, 256, 1), (200, 129, 33, 5), (2048, 96, 256, 8), (1100, 320, 197, 11), (77, 4096, 40, 1), (520, 264, 8, 2),
    (1, 512, 300, 1), (512, 1, 65, 1),
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_forward(br, i):
    for j in (i, i + 5):
        check_forward(br, *SHAPES[i], j % 4, j % 2 == 0, j % 3 == 0, seed=10 * i + j)


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_gradients(br, i):
    check_backward(br, *SHAPES[i], i % 4, i % 2, seed=i)


@pytest.mark.parametrize("parts", [("dx",), ("dw",), ("dbias",), ("dx", "dbias")])
def test_gradients_one_at_a_time(br, parts):
    check_backward(br, 70, 66, 50, 2, SILU, 1, 3, parts)


@pytest.mark.parametrize("a", [NONE, RELU, SILU, GELU])
def test_activation_gradient(br, a):
    rng = np.random.default_rng(a)
    n = 100003
    pre, dy = to_bf16(4 * rng.standard_normal(n)), to_bf16(rng.standard_normal(n))
    pre[:8] = to_bf16([0.0, -0.0, 88.0, -88.0, 3e38, -3e38, 1e-30, -1e-30])
    D = br.DevArray.from_numpy
    out, g, p = br.DevArray(n, np.uint16), D(dy), D(pre)
    br.check(br.lib.mi355_act_bwd_bf16_dev(out.ptr, g.ptr, p.ptr, 0.5, a, n))
    P, G = from_bf16(pre).astype(np.float64), from_bf16(dy).astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(np.abs(P) > 40, (P > 0) if a else 1.0, slope(a, np.clip(P, -40, 40)))
    want = 0.5 * G * s
    off = 0.5 * np.abs(G) * 2.0 ** -19 * (1 + np.minimum(np.abs(P), 40)) * (a != NONE)
    close(out.numpy(), want, off + 2.0 ** -8 * (np.abs(want) + off) + TINY)
    br.check(br.lib.mi355_act_bwd_bf16_dev(g.ptr, g.ptr, p.ptr, 0.5, a, n))       # in place
    assert np.array_equal(g.numpy(), out.numpy())


def test_residual_in_place(br):
    rng = np.random.default_rng(1)
    x, w, res = to_bf16(rng.standard_normal((3, 96, 75))), to_bf16(rng.standard_normal((130, 96)) / 10), to_bf16(rng.standard_normal((3, 130, 75)))
    want, _ = run_forward(br, x, w, None, NONE, res, 0.25)
    D = br.DevArray.from_numpy
    y, xd, wd = D(res), D(x), D(w)
    br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, None, xd.ptr, wd.ptr, None, NONE, y.ptr, 0.25, 130, 96, 75, 3))
    assert np.array_equal(y.numpy(), want)


@pytest.mark.parametrize("M,K,S,B", [(64, 128, 64, 2), (40, 72, 8, 1), (16, 256, 1, 1)])
def test_tensors_at_any_element(br, M, K, S, B):
    rng = np.random.default_rng(2)
    x, w = to_bf16(rng.standard_normal((B, K, S))), to_bf16(rng.standard_normal((M, K)))
    want, _ = run_forward(br, x, w, None, NONE, None, 1.0)
    D = br.DevArray.from_numpy
    for sx, sw, sy in ((1, 0, 0), (0, 3, 0), (0, 0, 5), (1, 1, 1)):
        xd, wd = D(np.concatenate([np.zeros(sx, np.uint16), x.ravel()])), D(np.concatenate([np.zeros(sw, np.uint16), w.ravel()]))
        yd = D(np.full(sy + B * M * S + 8, 7, np.uint16))
        br.check(br.lib.mi355_linear_fwd_bf16_dev(yd.ptr + 2 * sy, None, xd.ptr + 2 * sx, wd.ptr + 2 * sw, None, NONE, None, 1.0, M, K, S, B))
        got = yd.numpy()
        assert np.array_equal(got[sy:sy + B * M * S].reshape(want.shape), want)
        assert np.all(got[:sy] == 7) and np.all(got[sy + B * M * S:] == 7)


def test_what_is_outside_is_not_seen(br):
    """Infinities right behind every tensor: sums end where they should, whatever the sizes leave of the last steps."""
    for M, K, S, B in ((70, 72, 40, 3), (33, 65, 19, 2), (130, 130, 256, 1), (9, 520, 8, 1)):
        rng = np.random.default_rng(M)
        x, w, dy = to_bf16(rng.standard_normal((B, K, S))), to_bf16(rng.standard_normal((M, K))), to_bf16(rng.standard_normal((B, M, S)))
        D, inf = br.DevArray.from_numpy, np.full(4096, 0x7F80, np.uint16)
        xd, wd, gd = (D(np.concatenate([t.ravel(), inf])) for t in (x, w, dy))
        y, dx, dw, db = br.DevArray((B, M, S), np.uint16), br.DevArray((B, K, S), np.uint16), br.DevArray((M, K)), br.DevArray(M)
        br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, None, xd.ptr, wd.ptr, None, NONE, None, 1.0, M, K, S, B))
        br.check(br.lib.mi355_linear_bwd_bf16_dev(dx.ptr, dw.ptr, db.ptr, gd.ptr, xd.ptr, wd.ptr, 1.0, NONE, None, 0, M, K, S, B))
        for t in (from_bf16(y.numpy()), from_bf16(dx.numpy()), dw.numpy(), db.numpy()):
            assert np.all(np.isfinite(t)), (M, K, S, B)


def test_a_nan_stays_in_its_column(br):
    rng = np.random.default_rng(3)
    x, w = to_bf16(rng.standard_normal((2, 64, 50))), to_bf16(rng.standard_normal((70, 64)))
    want, _ = run_forward(br, x, w, None, GELU, None, 1.0)
    x[1, 7, 20] = to_bf16([np.nan])[0]
    got, _ = run_forward(br, x, w, None, GELU, None, 1.0)
    bad = np.isnan(from_bf16(got))
    assert bad[1, :, 20].all() and bad.sum() == 70
    got[1, :, 20] = want[1, :, 20]
    assert np.array_equal(got, want)


def test_refusals(br):
    d = br.DevArray((4096,))
    p, lib = d.ptr, br.lib
    fwd = [p, None, p, p, None, 0, None, 1.0, 4, 4, 4, 1]
    for i, v in ((0, None), (2, None), (3, None), (5, -1), (5, 4), (8, 0), (9, 0), (10, 0), (11, 0), (8, -3), (8, 2 ** 23), (10, 2 ** 23), (11, 2 ** 22)):
        a = list(fwd)
        a[i] = v
        assert lib.mi355_linear_fwd_bf16_dev(*a) == -1, (i, v)
        assert br.last_error()
    bwd = [p, p, p, p, p, p, 1.0, 0, None, 0, 4, 4, 4, 1]
    for change in ({3: None}, {4: None}, {5: None}, {0: None, 1: None, 2: None}, {7: 2}, {7: 9}, {10: 0}, {11: 0}, {12: 0}, {13: 0}, {13: 2 ** 22}):
        a = list(bwd)
        for i, v in change.items():
            a[i] = v
        assert lib.mi355_linear_bwd_bf16_dev(*a) == -1, change
    for a in ((None, p, p, 1.0, 0, 4), (p, None, p, 1.0, 0, 4), (p, p, None, 1.0, 0, 4), (p, p, p, 1.0, 7, 4)):
        assert lib.mi355_act_bwd_bf16_dev(*a) == -1
    assert lib.mi355_act_bwd_bf16_dev(p, p, p, 1.0, 0, 0) == 0


@pytest.mark.parametrize("M,K,S,B", [(128, 192, 64, 2), (96, 100, 33, 3)])
def test_replayed_graph(br, M, K, S, B):
    """Recorded and replayed, other calls that use the same workspace in between."""
    rng = np.random.default_rng(4)
    x, w, dy = to_bf16(rng.standard_normal((B, K, S))), to_bf16(rng.standard_normal((M, K))), to_bf16(rng.standard_normal((B, M, S)))
    D = br.DevArray.from_numpy
    xd, wd, gd = D(x), D(w), D(dy)
    y, dx, dw, db = br.DevArray((B, M, S), np.uint16), br.DevArray((B, K, S), np.uint16), br.DevArray((M, K)), br.DevArray(M)

    def calls():
        br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, None, xd.ptr, wd.ptr, None, SILU, None, 1.0, M, K, S, B))
        br.check(br.lib.mi355_linear_bwd_bf16_dev(dx.ptr, dw.ptr, db.ptr, gd.ptr, xd.ptr, wd.ptr, 1.0, NONE, None, 0, M, K, S, B))

    calls()
    want = [t.numpy() for t in (y, dx, dw, db)]
    br.check(br.lib.mi355_graph_begin())
    calls()
    graph = br.lib.mi355_graph_end()
    assert graph
    for _ in range(3):
        for t in (y, dx, dw, db):
            t.zero()
        br.check(br.lib.mi355_graph_launch(graph))
        for t, r in zip((y, dx, dw, db), want):
            assert np.array_equal(t.numpy(), r)
        run_forward(br, to_bf16(rng.standard_normal((1, 96, 31))), to_bf16(rng.standard_normal((64, 96))), None, NONE, None, 1.0)
    br.lib.mi355_graph_free(graph)


def test_attention_block_in_one_run(br):
    """A layer's attention as a step runs it, bfloat16 storage: norm, q/k/v products, rotation, attention, output product with the scaled
    residual; back through all of it.  Every stage against the formulas in 64 bits on the stage's own stored inputs."""
    import test_gpu_attention as A
    C, heads, kv, hd, S, B = 96, 4, 2, 32, 75, 2
    rng = np.random.default_rng(5)
    D, lib, n = br.DevArray.from_numpy, br.lib, S
    new = lambda c: br.DevArray((B, c, S), np.uint16)       # noqa: E731
    x, dy = to_bf16(rng.standard_normal((B, C, S))), to_bf16(rng.standard_normal((B, C, S)))
    wn = np.ones(C, np.float32)
    w = {k: to_bf16(rng.standard_normal(s) / np.sqrt(s[1])) for k, s in dict(q=(heads * hd, C), k=(kv * hd, C), v=(kv * hd, C), o=(C, heads * hd)).items()}
    wd = {k: D(v) for k, v in w.items()}
    xd, wnd, xn, y = D(x), D(wn), new(C), new(C)
    q, k, v, qr, kr, o = new(heads * hd), new(kv * hd), new(kv * hd), new(heads * hd), new(kv * hd), new(heads * hd)
    lse = br.DevArray((B, heads, S))
    cos, sin = br.rope_tables_dev(S, hd, 1e4)
    alpha, scale = 0.25, float(np.float32(hd ** -0.5))
    br.check(lib.mi355_rmsnorm_fwd_bf16_dev(xn.ptr, xd.ptr, wnd.ptr, C, S, B, 1e-5))
    for t, out in (("q", q), ("k", k), ("v", v)):
        br.check(lib.mi355_linear_fwd_bf16_dev(out.ptr, None, xn.ptr, wd[t].ptr, None, NONE, None, 1.0, w[t].shape[0], C, S, B))
    br.check(lib.mi355_rope_bf16_dev(qr.ptr, kr.ptr, q.ptr, k.ptr, heads, kv, hd, S, B, cos, sin, 1))
    br.check(lib.mi355_attn_fwd_bf16_dev(o.ptr, lse.ptr, qr.ptr, kr.ptr, v.ptr, None, heads, kv, hd, S, B, scale))
    br.check(lib.mi355_linear_fwd_bf16_dev(y.ptr, None, o.ptr, wd["o"].ptr, None, NONE, xd.ptr, alpha, C, heads * hd, S, B))
    f = lambda t: from_bf16(t.numpy()).astype(np.float64)   # noqa: E731
    W = {t: from_bf16(a).astype(np.float64) for t, a in w.items()}
    for t, out in (("q", q), ("k", k), ("v", v)):
        z, off = W[t] @ f(xn), E32 * (C + 4) * (np.abs(W[t]) @ np.abs(f(xn)))
        close(out.numpy(), z, off + 2.0 ** -8 * (np.abs(z) + off))
    c = A.Case("bf16", heads, kv, hd, S, B)
    c.q, c.k, c.v, c.scale = qr.numpy(), kr.numpy(), v.numpy(), scale
    A.check(c, dict(o=o.numpy(), lse=lse.numpy()), A.reference(c))
    z, off = from_bf16(x) + alpha * (W["o"] @ f(o)), alpha * E32 * (heads * hd + 8) * (np.abs(W["o"]) @ np.abs(f(o)))
    close(y.numpy(), z, off + 2.0 ** -8 * (np.abs(z) + off) + E32 * 4)
    # back: dy -> d_o, dw_o; attention; rotation; dw_q, dw_k, dw_v
    dyd, d_o, dqr, dkr, dv, dq, dk = D(dy), new(heads * hd), new(heads * hd), new(kv * hd), new(kv * hd), new(heads * hd), new(kv * hd)
    dwo = br.DevArray(w["o"].shape)
    br.check(lib.mi355_linear_bwd_bf16_dev(d_o.ptr, dwo.ptr, None, dyd.ptr, o.ptr, wd["o"].ptr, alpha, NONE, None, 0, C, heads * hd, S, B))
    br.check(lib.mi355_attn_bwd_bf16_dev(dqr.ptr, dkr.ptr, dv.ptr, d_o.ptr, qr.ptr, kr.ptr, v.ptr, o.ptr, lse.ptr, None, heads, kv, hd, S, B, scale))
    br.check(lib.mi355_rope_bf16_dev(dq.ptr, dk.ptr, dqr.ptr, dkr.ptr, heads, kv, hd, S, B, cos, sin, -1))
    c.do = d_o.numpy()
    A.check(c, dict(dq=dqr.numpy(), dk=dkr.numpy(), dv=dv.numpy()), A.reference(c, o.numpy(), lse.numpy()))
    G, O = from_bf16(dy).astype(np.float64), f(o)
    want = alpha * np.einsum("bms,bks->mk", G, O)
    close(dwo.numpy(), want, E32 * (B * n + 6) * np.einsum("bms,bks->mk", np.abs(G), np.abs(O)))
    for t, g in (("q", dq), ("k", dk), ("v", dv)):
        dw = br.DevArray(w[t].shape)
        br.check(lib.mi355_linear_bwd_bf16_dev(None, dw.ptr, None, g.ptr, xn.ptr, None, 1.0, NONE, None, 0, w[t].shape[0], C, S, B))
        want = np.einsum("bms,bks->mk", f(g), f(xn))
        close(dw.numpy(), want, E32 * (B * n + 6) * np.einsum("bms,bks->mk", np.abs(f(g)), np.abs(f(xn))) + TINY)


@pytest.mark.parametrize("M,K,S,B", [(5003, 72, 1, 1), (5003, 70, 3, 1), (4200, 8, 1, 4),           # more rows than a round of the grid
                                     (2100, 2050, 4, 1), (4104, 1024, 1, 4), (300, 96, 5, 1)])      # the same columns in tiles
def test_few_columns(br, M, K, S, B):
    check_forward(br, M, K, S, B, SILU, True, True, seed=M)


@pytest.mark.parametrize("M,K,S,B", [(24, 8190, 2565, 1), (16, 8192, 1280, 2),         # one product's many tiles decide for both
                                     (20, 1600, 1901, 1), (1600, 24, 66, 2), (33, 40, 5000, 1)])
def test_gradients_of_unequal_products(br, M, K, S, B):
    check_backward(br, M, K, S, B, NONE, 1, seed=K)


def test_offsets_beyond_32_bits(br):
    """A tensor of 1100 rows of 2^21 values (4.6 GB) as x, as dy of dx and as dy of dw: what its few rows that are not zero hold arrives,
    those behind 2^32 bytes included."""
    N, R, C, rows = 1 << 21, 1100, 8, (3, 511, 1030, 1097)
    rng = np.random.default_rng(8)
    big = br.DevArray((R, N), np.uint16).zero()
    held = to_bf16(rng.standard_normal((len(rows), N)))
    for r, a in zip(rows, held):
        br.lib.mi355_buf_write(big.handle, r * N * 2, a.ctypes.data, a.nbytes)
    w = to_bf16(rng.standard_normal((C, R)))
    D, out = br.DevArray.from_numpy, br.DevArray((C, N), np.uint16)
    X, W = from_bf16(held).astype(np.float64), from_bf16(w).astype(np.float64)[:, rows]
    off = E32 * (len(rows) + 4) * (np.abs(W) @ np.abs(X))           # (sums of zeros but for four terms)
    wd, wtd = D(w), D(np.ascontiguousarray(w.T))
    br.check(br.lib.mi355_linear_fwd_bf16_dev(out.ptr, None, big.ptr, wd.ptr, None, NONE, None, 1.0, C, R, N, 1))
    close(out.numpy(), W @ X, off + 2.0 ** -8 * (np.abs(W @ X) + off) + TINY)
    out.zero()
    br.check(br.lib.mi355_linear_bwd_bf16_dev(out.ptr, None, None, big.ptr, None, wtd.ptr, 1.0, NONE, None, 0, R, C, N, 1))
    got = out.numpy()
    close(got, W @ X, off + 2.0 ** -8 * (np.abs(W @ X) + off) + TINY)
    dw, db, Y = br.DevArray((R, C)), br.DevArray(R), from_bf16(got).astype(np.float64)
    br.check(br.lib.mi355_linear_bwd_bf16_dev(None, dw.ptr, db.ptr, big.ptr, out.ptr, None, 1.0, NONE, None, 0, R, C, N, 1))
    want, bound = np.zeros((R, C)), np.zeros((R, C))
    want[rows, :], bound[rows, :] = X @ Y.T, E32 * (N + 6) * (np.abs(X) @ np.abs(Y).T)
    close(dw.numpy(), want, bound)
    assert not np.any(np.delete(dw.numpy(), rows, 0)) and not np.any(np.delete(db.numpy(), rows))
