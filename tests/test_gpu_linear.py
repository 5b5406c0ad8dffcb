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
