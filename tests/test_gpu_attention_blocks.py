"""Attention with one, two and four position blocks side by side in a workgroup, in the forward pass with dq and in dk/dv, at every size of head:
packed and odd rows of several tiles, and what the mask hides.  Bounds: test_gpu_attention.py's."""
import numpy as np
import pytest

import test_gpu_attention as A

pytestmark = pytest.mark.gpu


def side_by_side(heads, S, two_from):
    """The rule that the source states, on 256 compute units."""
    if -(-S // 128) * heads >= 2 * 256:
        return 4
    return 2 if 2 * -(-S // 64) * heads >= two_from * 256 else 1


def blocks(storage, heads, kv, hd, S, batch, cu):
    return side_by_side(heads * batch, S, 2 if storage == "bf16" else 3), side_by_side(kv * batch, S, 3)


CASES = [
    # heads, kv, hd, S, batch, offsets; blocks side by side of queries, of keys
    ((12, 12, 64, 197, 8, [[0, 1, 66, 150, 190]] * 8), 2, 2), ((12, 12, 64, 256, 8, None), 2, 2), ((10, 10, 96, 300, 8, [[0, 130, 131, 300]] * 8), 2, 2),
    ((10, 10, 72, 299, 8, None), 2, 2), ((16, 8, 128, 270, 12, [[5, 70, 200, 269]] * 12), 4, 2), ((8, 4, 128, 310, 12, [[0, 300, 305]] * 12), 2, 1),
    ((32, 16, 72, 210, 8, [[0, 64, 129, 210]] * 8), 4, 2), ((32, 32, 96, 150, 8, None), 4, 4), ((32, 32, 96, 200, 8, [[0, 40, 190]] * 8), 4, 4),
    ((64, 64, 128, 140, 4, [[0, 3, 140]] * 4), 4, 4), ((64, 32, 64, 257, 9, [[0, 100, 257]] * 9), 4, 4), ((3, 1, 96, 400, 1, [[0, 150, 399]]), 1, 1),
]


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward_and_gradients(br, i, storage):
    shape, queries, keys = CASES[i]
    if br.device_info()[2] == 256:
        assert blocks(storage, *shape) == (queries, keys)
    c = A.Case(storage, *shape, seed=40 + i)
    o, lse = A.forward(br, c)
    A.check(c, dict(o=o, lse=lse), A.reference(c))
    A.check(c, A.backward(br, c, o, lse), A.reference(c, o, lse))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("i", [0, 2, 4, 5, 6, 8, 9, 10])
def test_what_the_mask_hides_is_not_seen(br, i, bad, storage):
    """Infinities and NaNs in other sequences, outside of all and in later positions leave a result as it is, to the bit."""
    shape, _, _ = CASES[i]
    c = A.Case(storage, *shape, seed=60 + i)
    cu = shape[5][0]
    n = int(np.argmax(np.diff(cu)))
    lo, hi = cu[n], cu[n + 1]
    late = hi - 5
    names = ("q", "k", "v", "do")
    clean = {m: getattr(c, m).copy() for m in names}
    mark = c.stored(np.full(1, bad))[0]

    def spoil(where):
        for m in names:
            a = clean[m].copy()
            a[:, :, where] = mark
            setattr(c, m, a)

    o, lse = A.forward(br, c)
    g = A.backward(br, c, o, lse)
    positions = np.arange(c.S)
    spoilt, others = (positions < lo) | (positions >= late), (positions < lo) | (positions >= hi)
    seen = ~spoilt
    spoil(spoilt)
    o2, lse2 = A.forward(br, c)
    assert np.array_equal(o2[:, :, seen], o[:, :, seen]) and np.array_equal(lse2[:, :, seen], lse[:, :, seen])
    # dq of a position sees earlier ones only; dk and dv see later ones, so there the other sequences alone are spoilt
    for where, columns, results in ((spoilt, seen, ("dq",)), (others, ~others, ("dq", "dk", "dv"))):
        spoil(where)
        o_s, lse_s = o.copy(), lse.copy()
        o_s[:, :, where], lse_s[:, :, where] = mark, bad
        g2 = A.backward(br, c, o_s, lse_s)
        for m in results:
            assert np.array_equal(g2[m][:, :, columns], g[m][:, :, columns]), m


@pytest.mark.parametrize("i", [0, 3, 6, 9])
def test_the_same_bits_again(br, i):
    """Teams and blocks are added up in a fixed order."""
    shape, _, _ = CASES[i]
    for storage in ("f32", "bf16"):
        c = A.Case(storage, *shape, seed=80 + i)
        o, lse = A.forward(br, c)
        g = A.backward(br, c, o, lse)
        for _ in range(3):
            o2, lse2 = A.forward(br, c)
            g2 = A.backward(br, c, o, lse)
            assert np.array_equal(o, o2) and np.array_equal(lse, lse2) and all(np.array_equal(g[n], g2[n]) for n in g)
