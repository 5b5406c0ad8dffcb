"""Linear layers beside test_gpu_linear.py: calls in place, and every size of tile with every epilogue at sizes that are no multiple of it."""
import numpy as np
import pytest

from test_gpu_attention import E32, from_bf16, to_bf16
from test_gpu_linear import GELU, NONE, RELU, SILU, TINY, act, close, run_forward, slope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2049, 70001])
@pytest.mark.parametrize("a", [NONE, RELU, SILU, GELU])
def test_activation_gradient_in_place(br, a, n):
    """dpre may be dy: the same bits as into another tensor, at whole and broken groups of eight."""
    rng = np.random.default_rng(n)
    pre, dy = to_bf16(3 * rng.standard_normal(n)), to_bf16(rng.standard_normal(n))
    D = br.DevArray.from_numpy
    out, g, p = br.DevArray(n, np.uint16), D(dy), D(pre)
    br.check(br.lib.mi355_act_bwd_bf16_dev(out.ptr, g.ptr, p.ptr, 0.25, a, n))
    br.check(br.lib.mi355_act_bwd_bf16_dev(g.ptr, g.ptr, p.ptr, 0.25, a, n))
    assert np.array_equal(g.numpy(), out.numpy()) and np.all(np.isfinite(from_bf16(out.numpy())))


def columns(a):
    """[batch][rows][S] as [rows][batch * S], 64 bits."""
    return from_bf16(a).astype(np.float64).transpose(1, 0, 2).reshape(a.shape[1], -1)


def tile_of(products, quarters, cu):
    """The tile that a call takes by the rule that its source states: (256 or 128 or 64, tiles of that size)."""
    count = lambda t: sum(-(-m // t) * -(-n // t) for m, n in products)         # noqa: E731
    for t, q in zip((256, 128), quarters):
        if 4 * count(t) >= q * cu:
            return t, count(t)
    return 64, count(64)


FORWARD = [  # M, K, S, batch, activation; the tile, whether there are more than a compute unit each
    (1500, 72, 197, 17, GELU, 128, True), (1500, 136, 200, 17, SILU, 128, True), (1500, 65, 197, 11, RELU, 128, False), (1510, 192, 192, 11, GELU, 128, False),
    (4300, 72, 197, 39, GELU, 256, True), (4290, 264, 200, 39, SILU, 256, True), (5000, 40, 6605, 1, NONE, 256, True), (130, 2056, 75, 5, GELU, 64, False),
]


@pytest.mark.parametrize("i", range(len(FORWARD)))
def test_forward_in_every_tile(br, i):
    """Bias, activation, residual and pre, in rows that end inside a tile and columns of sequences that do.  Bounds: test_gpu_linear.py's."""
    M, K, S, B, a, tile, many = FORWARD[i]
    if br.device_info()[2] == 256:
        t, n = tile_of([(M, B * S)], (8, 2 if K >= 2048 else 3), 256)
        assert t == tile and (n > 256) == many
    rng = np.random.default_rng(i)
    x, w = to_bf16(rng.standard_normal((B, K, S), np.float32)), to_bf16(rng.standard_normal((M, K), np.float32) / np.float32(np.sqrt(K)))
    bias, res, alpha = rng.standard_normal(M).astype(np.float32), to_bf16(rng.standard_normal((B, M, S), np.float32)), float(np.float32(0.3))
    got, pre = run_forward(br, x, w, bias, a, res, alpha)
    W, X, R = from_bf16(w).astype(np.float64), columns(x), columns(res)
    Y, Z = columns(got), columns(pre)
    for rows, cols in ((np.arange(M), rng.choice(B * S, 250, False)), (np.unique(np.r_[rng.choice(M, 60), M - 1]), np.arange(B * S))):
        at = np.ix_(rows, cols)
        b = bias.astype(np.float64)[rows, None]
        z, dz = W[rows] @ X[:, cols] + b, E32 * (K + 4) * (np.abs(W[rows]) @ np.abs(X[:, cols]) + np.abs(b))
        y = alpha * act(a, z) + R[at]
        close(Z[at], z, dz + 2.0 ** -8 * (np.abs(z) + dz) + TINY)
        off = alpha * (1.13 * dz + 2.0 ** -19 * np.abs(z) * (a != NONE)) + 2 * E32 * (np.abs(y) + alpha * np.abs(z))
        close(Y[at], y, off + 2.0 ** -8 * (np.abs(y) + off) + TINY)


BACKWARD = [  # M, K, S, batch, activation, accumulate, parts; the tile
    (200, 1500, 197, 11, SILU, 0, "dx dw db", 128), (200, 1500, 197, 11, GELU, 0, "dx", 128), (1500, 2100, 200, 3, NONE, 0, "dw", 128),
    (100, 8200, 40, 5, SILU, 0, "dx dw db", 128),           # several sequences of 40 columns, as many units as compute units or fewer
    (90, 8200, 56, 4, GELU, 1, "dx dw db", 128), (300, 4300, 197, 27, GELU, 0, "dx dw db", 256), (304, 4312, 200, 27, RELU, 0, "dx dw db", 256),
    (4200, 4300, 40, 7, NONE, 0, "dw db", 128), (5000, 5100, 24, 3, NONE, 1, "dw", 256), (66, 70, 50, 3, SILU, 0, "dx dw db", 64),
]


@pytest.mark.parametrize("i", range(len(BACKWARD)))
def test_gradients_in_every_tile(br, i):
    M, K, S, B, a, accumulate, parts, tile = BACKWARD[i]
    if br.device_info()[2] == 256:
        t, n = tile_of([(K, B * S)] * ("dx" in parts) + [(M, K)] * ("dw" in parts), (6, 3), 256)
        assert t == tile, (t, n)
    rng = np.random.default_rng(100 + i)
    normal = lambda *s: to_bf16(rng.standard_normal(s, np.float32))         # noqa: E731
    x, w, dy, pre = normal(B, K, S), to_bf16(rng.standard_normal((M, K), np.float32) / np.float32(np.sqrt(K))), normal(B, M, S), normal(B, K, S)
    alpha, n = float(np.float32(0.7)), B * S
    dw0, db0 = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal(M).astype(np.float32)
    D = br.DevArray.from_numpy
    dx, dw, db = br.DevArray((B, K, S), np.uint16), D(dw0), D(db0)
    g, xd, wd, p = D(dy), D(x), D(w), D(pre)
    br.check(br.lib.mi355_linear_bwd_bf16_dev(dx.ptr if "dx" in parts else None, dw.ptr if "dw" in parts else None, db.ptr if "db" in parts else None,
                                              g.ptr, xd.ptr, wd.ptr, alpha, a, p.ptr if a else None, accumulate, M, K, S, B))
    G, X, W, P = columns(dy), columns(x), from_bf16(w).astype(np.float64), columns(pre)
    if "dx" in parts:
        got = columns(dx.numpy())
        for rows, cols in ((np.arange(K), rng.choice(n, min(n, 250), False)), (np.unique(np.r_[rng.choice(K, 60), K - 1]), np.arange(n))):
            at = np.ix_(rows, cols)
            want = alpha * (W[:, rows].T @ G[:, cols]) * slope(a, P[at])
            off = alpha * (E32 * (M + 6) * 1.13 + 2.0 ** -19 * (a != NONE)) * (np.abs(W[:, rows]).T @ np.abs(G[:, cols])) * (1 + np.abs(P[at]) * (a != NONE))
            close(got[at], want, off + 2.0 ** -8 * (np.abs(want) + off) + TINY)
    got = dw.numpy()
    if "dw" in parts:
        for rows, cols in ((np.arange(M), rng.choice(K, min(K, 250), False)), (np.unique(np.r_[rng.choice(M, 60), M - 1]), np.arange(K))):
            at = np.ix_(rows, cols)
            want = alpha * (G[rows] @ X[cols].T) + (dw0[at] if accumulate else 0.0)
            close(got[at], want, E32 * (n + 6) * (np.abs(G[rows]) @ np.abs(X[cols]).T) + 2 * E32 * (np.abs(want) + np.abs(dw0[at])))
    else:
        assert np.array_equal(got, dw0)
    if "db" in parts:
        want = alpha * G.sum(1) + (db0 if accumulate else 0.0)
        close(db.numpy(), want, E32 * (n + 6) * np.abs(G).sum(1) + 2 * E32 * (np.abs(want) + np.abs(db0)))
    else:
        assert np.array_equal(db.numpy(), db0)


@pytest.mark.parametrize("M,K,S,B", [(300, 200, 1, 2), (130, 96, 75, 3), (1500, 72, 197, 11), (1500, 136, 200, 17), (4300, 24, 197, 39), (77, 4096, 40, 1), (2050, 2048, 1, 4)])
def test_residual_in_place_in_every_tile(br, M, K, S, B):
    """y may be res: the same bits as into another tensor, by rows, in every tile and by way of slices; pre beside it."""
    rng = np.random.default_rng(M)
    x, w = to_bf16(rng.standard_normal((B, K, S), np.float32)), to_bf16(rng.standard_normal((M, K), np.float32) / np.float32(np.sqrt(K)))
    res = to_bf16(rng.standard_normal((B, M, S), np.float32))
    want, wpre = run_forward(br, x, w, None, SILU, res, -0.25)
    D = br.DevArray.from_numpy
    y, xd, wd, pre = D(res), D(x), D(w), br.DevArray((B, M, S), np.uint16)
    br.check(br.lib.mi355_linear_fwd_bf16_dev(y.ptr, pre.ptr, xd.ptr, wd.ptr, None, SILU, y.ptr, -0.25, M, K, S, B))
    assert np.array_equal(y.numpy(), want) and np.array_equal(pre.numpy(), wpre)
