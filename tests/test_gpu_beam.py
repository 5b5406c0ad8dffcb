"""Beam search: its step against the definition in 64 bits, the cache's rows following the beams, and a search written with both.

A candidate is score + (logit - lse) in fp64 from an lse whose sum of exponentials has fp32 terms: each is off by at most 2^-22 of itself
(the hardware exponential, the difference's rounding and its product), and so is the sum; 4 * 2^-22 covers the blocks' fp32 sums as well, and
2^-24 of the value the rounding of the score.  Candidates that differ are further apart than that in these tests, which is looked at first."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_paged import Cache, append, attend, expected, f64, fn, stored

pytestmark = pytest.mark.gpu

OFF = 2.0 ** -20


def step(br, storage, logits, score, done, beams, eos=-1, pad=0):
    """logits [batch][V][S]"""
    B, V, S = logits.shape
    D = br.DevArray.from_numpy
    ld, sd = D(logits), D(np.asarray(score, np.float32))
    dd = None if done is None else D(np.asarray(done, np.int32))
    out = [br.DevArray(B * S)] + [br.DevArray(B * S, np.int32) for _ in range(3)]
    br.check(fn(br, "beam_step", storage)(out[0].ptr, out[1].ptr, out[2].ptr, out[3].ptr, ld.ptr, sd.ptr, dd.ptr if dd else None, V, S, B, beams, eos, pad))
    return [a.numpy() for a in out]


def definition(logits, score, done, beams, eos, pad):
    B, V, S = logits.shape
    N = B * S
    x = f64(logits).transpose(0, 2, 1).reshape(N, V)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        lse = m + np.log(np.exp(x - m).sum(1, keepdims=True))
        cand = np.asarray(score, np.float32).astype(np.float64)[:, None] + (x - lse)
    for n in range(N):
        if done is not None and done[n]:
            cand[n] = -np.inf
            cand[n, pad] = np.float32(score[n])
    cand = np.where(np.isnan(cand), -np.inf, cand)
    out = [np.zeros(N), np.zeros(N, int), np.zeros(N, int), np.zeros(N, int)]
    for g in range(N // beams):
        flat = cand[g * beams:(g + 1) * beams].reshape(-1)
        for i, j in enumerate(np.argsort(-flat, kind="stable")[:beams]):
            n, v = g * beams + j // V, j % V
            for a, val in zip(out, (flat[j], v, n, int(bool(done is not None and done[n]) or v == eos))):
                a[g * beams + i] = val
    return out


def check(got, want):
    assert np.array_equal(got[2], want[2]), (got[2], want[2])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    assert np.array_equal(got[3], want[3])
    finite = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(got[0]), finite) and np.all(got[0][~finite] == want[0][~finite])
    assert np.all(np.abs(got[0][finite] - want[0][finite]) <= OFF + 2.0 ** -23 * np.abs(want[0][finite]))


def apart(rng, storage, B, V, S):
    """Logits that are whole numbers of steps of 1/64 (bfloat16: 1/8), so that equal ones are frequent in a column, and scores."""
    steps = 64 if storage == "f32" else 8
    x = np.round(np.clip(3.0 * rng.standard_normal((B, V, S)), -15.9, 15.9) * steps) / steps
    return stored(storage, x), (-20.0 - 6.0 * rng.random(B * S)).astype(np.float32)


STEPS = [
    # batch, V, S, beams
    (1, 1, 1, 1), (1, 5, 4, 4), (3, 4, 1, 1), (1, 64, 64, 64), (1, 1000, 4, 4), (4, 999, 1, 4), (5, 1023, 3, 3), (1, 4096, 16, 8), (6, 257, 5, 5),
    (1, 32000, 4, 4), (8, 32000, 1, 8), (2, 50001, 5, 5), (1, 20000, 100, 5), (1, 151936, 16, 8), (10, 8193, 1, 2), (1, 777, 130, 13), (1, 3000, 640, 16),
    (3, 2, 2, 2), (64, 300, 1, 16), (7, 70, 32, 32),
]


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(STEPS)))
def test_step(br, i, storage):
    B, V, S, beams = STEPS[i]
    rng = np.random.default_rng(i)
    logits, score = apart(rng, storage, B, V, S)
    N = B * S
    done = (rng.random(N) < 0.2).astype(np.int32) * rng.integers(-2, 3, N).astype(np.int32)
    eos, pad = min(3, V - 1), V // 2
    want = definition(logits, score, done, beams, eos, pad)
    for d, p in ((done, pad), (None, 0)):
        assert gap(logits, score, d, beams, p) > 4 * OFF
    check(step(br, storage, logits, score, done, beams, eos, pad), want)
    check(step(br, storage, logits, score, None, beams, -1, 0), definition(logits, score, None, beams, -1, 0))


def gap(logits, score, done, beams, pad):
    """The smallest difference of neighbouring candidates among the first beams + 1 of each group that are not equal."""
    B, V, S = logits.shape
    x = f64(logits).transpose(0, 2, 1).reshape(B * S, V)
    m = x.max(1, keepdims=True)
    cand = np.asarray(score, np.float64)[:, None] + (x - (m + np.log(np.exp(x - m).sum(1, keepdims=True))))
    for n in range(B * S):
        if done is not None and done[n]:
            cand[n] = -np.inf
            cand[n, pad] = score[n]
    least = np.inf
    for part in cand.reshape(-1, beams * V):
        top = np.sort(part)[::-1][:beams + 1]
        d = -np.diff(top[np.isfinite(top)])
        least = min(least, d[d > 1e-12].min(initial=np.inf))
    return least


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 40, 8), (1, 5000, 8), (8, 5000, 1), (2, 5000, 4)])
def test_first_step_of_equal_beams(br, storage, shape):
    """Scores 0, -inf, ...: every new beam comes from the first, in the order of its tokens; and rows of equal logits give the lowest tokens."""
    B, V, S = shape
    rng = np.random.default_rng(100 + V)
    logits, _ = apart(rng, storage, B, V, S)
    score = np.where(np.arange(B * S) % 4 == 0, 0.0, -np.inf)
    got = step(br, storage, logits, score, None, 4)
    check(got, definition(logits, score, None, 4, -1, 0))
    assert np.all(got[2] % 4 == 0)
    same = stored(storage, np.full(shape, 1.5))
    got = step(br, storage, same, score, None, 4)
    check(got, definition(same, score, None, 4, -1, 0))
    assert np.array_equal(got[1], np.arange(B * S) % 4)
    got = step(br, storage, same, np.zeros(B * S), None, 4)             # all candidates of a group are equal
    assert np.array_equal(got[1], np.arange(B * S) % 4) and np.array_equal(got[2], np.arange(B * S) // 4 * 4)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["first", "first of equal", "equal", "three allowed", "one allowed", "rising", "falling"])
@pytest.mark.parametrize("shape", [(1, 70, 64, 64), (1, 1000, 64, 64), (64, 1000, 1, 64), (2, 9000, 48, 48), (1, 9000, 63, 63), (16, 2000, 1, 16)])
def test_many_candidates_at_the_border(br, storage, kind, shape):
    """Many beams of which one counts, masked vocabularies, equal logits: more candidates at the last new beam's than a short list holds."""
    B, V, S, beams = shape
    N = B * S
    rng = np.random.default_rng(140 + V + beams)
    logits, score = apart(rng, storage, B, V, S)
    if not kind.endswith("allowed"):
        score = np.repeat(score[:N // beams], beams)
    if kind.startswith("first"):
        score = np.where(np.arange(N) % beams == 0, 0.0, -np.inf)
    if kind.endswith("equal"):
        logits = stored(storage, np.full((B, V, S), -0.5))
    elif kind.endswith("allowed"):
        keep = rng.choice(V, 3 if kind[0] == "t" else 1, replace=False)
        masked = stored(storage, np.full((B, V, S), -np.inf))
        masked[:, keep] = logits[:, keep]
        logits = masked
    elif kind in ("rising", "falling"):
        rows = np.sort(np.round(rng.uniform(-15.9, 15.9, V) * 8) / 8)
        logits = stored(storage, np.tile((rows if kind == "rising" else rows[::-1])[None, :, None], (B, 1, S)))
    assert gap(logits, score, None, beams, 0) > 4 * OFF
    check(step(br, storage, logits, score, None, beams), definition(logits, score, None, beams, -1, 0))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 3000, 8), (8, 3000, 1), (2, 30, 4)])
def test_logits_that_are_no_numbers(br, storage, shape):
    """Masked vocabularies, by -inf and by the type's lowest value, columns of nothing else, infinities and NaNs."""
    B, V, S = shape
    rng = np.random.default_rng(110)
    logits, score = apart(rng, storage, B, V, S)
    cols = logits.transpose(0, 2, 1).reshape(B * S, V).copy()
    low = stored(storage, np.array([np.finfo(np.float32).min if storage == "f32" else -3.3895313892515355e38]))[0]
    val = lambda a: stored(storage, np.array([a]))[0]           # noqa: E731
    cols[0, ::2] = val(-np.inf)
    cols[1, 2:] = low                           # two tokens are left
    cols[2] = val(-np.inf)                      # none
    cols[3, 7] = val(np.nan)
    cols[4, 9] = val(np.inf)
    cols[5] = low                               # equal ones
    cols[6, 3:] = val(-np.inf)
    logits = np.ascontiguousarray(cols.reshape(B, S, V).transpose(0, 2, 1))
    check(step(br, storage, logits, score, None, 4), definition(logits, score, None, 4, -1, 0))
    alone = np.full(B * S, -np.inf, np.float32)                 # only beams that give nothing are left: the lowest tokens
    got = step(br, storage, logits, alone, None, 4)
    assert np.all(got[0] == -np.inf) and np.array_equal(got[1], np.arange(8) % 4) and np.array_equal(got[2], np.arange(8) // 4 * 4)


def test_step_in_a_graph(br):
    rng = np.random.default_rng(120)
    D = br.DevArray.from_numpy
    graphs = []
    for storage, (B, V, S, beams) in (("f32", (1, 32000, 8, 4)), ("bf16", (6, 9000, 1, 3))):
        logits, score = apart(rng, storage, B, V, S)
        want = step(br, storage, logits, score, None, beams, 5)
        ld, sd = D(logits), D(score)
        out = [br.DevArray(B * S)] + [br.DevArray(B * S, np.int32) for _ in range(3)]
        br.check(br.lib.mi355_graph_begin())
        br.check(fn(br, "beam_step", storage)(*[a.ptr for a in out], ld.ptr, sd.ptr, None, V, S, B, beams, 5, 0))
        g = br.lib.mi355_graph_end()
        assert g, br.last_error()
        graphs.append((g, out, want, ld, sd))
    for _ in range(3):
        for g, out, want, _, _ in graphs:
            for a in out:
                a.zero()
            br.check(br.lib.mi355_graph_launch(g))
        for g, out, want, _, _ in graphs:
            assert all(np.array_equal(a.numpy(), w) for a, w in zip(out, want))
        step(br, "f32", np.zeros((1, 700, 12), np.float32), np.zeros(12), None, 3)
    for g in graphs:
        br.lib.mi355_graph_free(g[0])


# ---- the cache's rows ------------------------------------------------------------------------------------------------------------

def reorder(br, caches, parent, pos, spare, advance=1, positions=True):
    D = br.DevArray.from_numpy
    cs = [c.to(br) for c in caches]
    for c in cs:
        c.pages = cs[0].pages
    arr = (br.KvCache * len(cs))(*cs)
    par, po, sp = (D(np.asarray(a, np.int32)) for a in (parent, pos, spare))
    pages_out, pos_out, spare_out = D(np.full(caches[0].pages.shape, 99, np.int32)), D(np.full(len(pos), 99, np.int32)), D(np.full(len(pos), 99, np.int32))
    br.check(fn(br, "kv_reorder", caches[0].storage)(arr, len(cs), pages_out.ptr, pos_out.ptr if positions else None, spare_out.ptr, par.ptr, po.ptr,
                                                     sp.ptr, advance))
    return pages_out.numpy(), pos_out.numpy(), spare_out.numpy(), [(c.kd.numpy(), c.vd.numpy()) for c in caches]


def follow(caches, parent, pos, spare, advance=1):
    """The definition."""
    c0 = caches[0]
    page, n = c0.page, len(pos)
    pages, spare_out = c0.pages.copy(), np.array(spare).copy()
    pos_out = np.array([p if p < 0 else p + advance for p in pos])
    after = [(c.k.copy(), c.v.copy()) for c in caches]
    for i in range(n):
        p = parent[i]
        if not 0 <= p < n or pos[p] != pos[i]:
            p = i
        if pos[i] < 0:
            continue
        tail, filled = pos[i] // page, pos[i] % page + 1
        pages[i, :tail + 1] = c0.pages[p, :tail + 1]
        if p != i and filled < page and tail < c0.max_pages and 0 <= c0.pages[p, tail] < c0.n_pages:
            pages[i, tail], spare_out[i] = spare[i], c0.pages[i, tail]
            if 0 <= spare[i] < c0.n_pages:
                for c, (k, v) in zip(caches, after):
                    k[spare[i], :, :filled] = c.k[c0.pages[p, tail], :, :filled]
                    v[spare[i], :, :filled] = c.v[c0.pages[p, tail], :, :filled]
    return pages, pos_out, spare_out, after


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(7))
def test_rows_follow_their_parents(br, storage, i):
    kv, hd, page, lengths, layers = [(2, 64, 16, [37] * 4, 1), (8, 128, 16, [33] * 8 + [48] * 8 + [1] * 8, 3), (1, 72, 48, [95] * 5 + [96] * 5 + [97] * 5, 2),
                                     (12, 64, 64, [200] * 4, 12), (2, 8, 16, [5] * 3, 2), (1, 120, 256, [250, 250, 7, 7], 70), (3, 96, 32, [90] * 130, 1)][i]
    rng = np.random.default_rng(130 + i)
    n = len(lengths)
    caches = [Cache(storage, kv, hd, page, [m + page for m in lengths] + [1] * n, seed=l) for l in range(layers)]
    spare = caches[0].pages[n:, 0].copy()
    for c in caches:
        c.pages = np.ascontiguousarray(caches[0].pages[:n])
    pos = np.array(lengths) - 1
    same = [np.flatnonzero(pos == p) for p in pos]
    parent = np.array([rng.choice(s) for s in same])
    got, want = reorder(br, caches, parent, pos, spare), follow(caches, parent, pos, spare)
    for a, b in zip(got[:3], want[:3]):
        assert np.array_equal(a, b)
    for (k, v), (wk, wv) in zip(got[3], want[3]):
        assert np.array_equal(k, wk) and np.array_equal(v, wv)
    # swapped in pairs, all from one, everybody its own; positions not asked for
    for parent in (np.arange(n) ^ 1, np.zeros(n, int), np.arange(n)):
        parent = np.minimum(parent, n - 1)
        got, want = reorder(br, caches, parent, pos, spare, 0, False), follow(caches, parent, pos, spare, 0)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[2], want[2]) and np.all(got[1] == 99)
        assert all(np.array_equal(a, b) for x, y in zip(got[3], want[3]) for a, b in zip(x, y))


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_rows_without_a_place(br, storage):
    """Parents that are none or at another position, rows that hold nothing, spare pages and tails that are none, positions behind the table."""
    cache = Cache(storage, 2, 64, 16, [40] * 10, seed=140)
    pos = np.array([35, 35, 35, 35, -1, -1, 20, 35, 700, 700])
    parent = np.array([-1, 10, 2 ** 31 - 1, 6, 0, 5, 3, 1, 9, 8])
    spare = np.array([int(cache.n_pages) - 1, -1, 3, 4, 5, 6, 7, -5, 8, 9])
    cache.pages[7, 2], parent[1], pos[1] = -3, 7, 35               # a tail that is no page
    got, want = reorder(br, [cache], parent, pos, spare), follow([cache], parent, pos, spare)
    for a, b in zip(got[:3], want[:3]):
        assert np.array_equal(a, b)
    assert got[0][1, 2] == -3 and got[2][1] == -1
    assert np.array_equal(got[3][0][0], want[3][0][0]) and np.array_equal(got[3][0][1], want[3][0][1])


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_a_search(br, storage):
    """Twelve steps of two prompts and three beams, in two layers, as a program runs them: append, attention, a classifier, the step, the rows that follow.
    Each step's attention equals the one over the beam's own history, kept apart on the host, and pages never have two writers."""
    rng = np.random.default_rng(150)
    heads, kv, hd, page, beams, groups, V, layers, start = 4, 2, 64, 16, 3, 2, 500, 2, 27
    N, scale = beams * groups, 0.125
    room = -(-(start + 14) // page)
    caches = [Cache(storage, kv, hd, page, [room * page] * N + [1] * N, seed=151) for _ in range(layers)]
    spare = caches[0].pages[N:, 0].copy()
    for c in caches:
        c.pages = np.ascontiguousarray(caches[0].pages[:N])
    history = [[([], []) for _ in range(layers)] for _ in range(N)]         # of each beam and layer: rows of k and of v
    for layer, c in enumerate(caches):                                      # the prompt: the same in all beams of a group
        for g in range(groups):
            for p in range(start):
                kr, vr = (stored(storage, rng.standard_normal((kv, hd))) for _ in range(2))
                for n in range(g * beams, (g + 1) * beams):
                    a, b = c.row(n, p)
                    c.k[a, :, b], c.v[a, :, b] = kr, vr
                    history[n][layer][0].append(kr), history[n][layer][1].append(vr)
    w = rng.standard_normal((V, heads * hd)) * 0.3
    pos, score, done = np.full(N, start), np.zeros(N, np.float32), np.zeros(N, np.int32)
    score[np.arange(N) % beams > 0] = -np.inf
    for t in range(12):
        assert len(set(spare) | {c for c in caches[0].pages[np.arange(N), pos // page]}) == 2 * N
        logits = np.zeros((1, V, N))
        for layer, c in enumerate(caches):
            q, k, v = (stored(storage, rng.standard_normal((1, h * hd, N))) for h in (heads, kv, kv))
            _, c.k, c.v = append(br, c, q, k, v, None, None, None, pos.astype(np.int32), heads, None, None, 0.0)
            for n in range(N):
                history[n][layer][0].append(k[0, :, n].reshape(kv, hd)), history[n][layer][1].append(v[0, :, n].reshape(kv, hd))
            got = attend(br, c, q, None, pos, heads, scale)
            own = Cache(storage, kv, hd, page, [int(pos[0]) + 1] * N, seed=152)
            for n in range(N):
                for p in range(int(pos[0]) + 1):
                    a, b = own.row(n, p)
                    own.k[a, :, b], own.v[a, :, b] = history[n][layer][0][p], history[n][layer][1][p]
            same = attend(br, own, q, None, pos, heads, scale)
            assert np.array_equal(got[0], same[0]) and np.array_equal(got[1], same[1])
            want = expected(own, q, None, pos, heads, scale)
            assert np.all(np.abs(f64(got[0]) - want[0]) <= want[1])
            logits += w @ f64(got[0])[0]
        x = np.round(logits * 64) / 64 + np.arange(N) / 512             # (beams' candidates further apart than a step's error)
        new = step(br, "f32", x.astype(np.float32), score, done, beams, 7, 0)
        check(new, definition(x.astype(np.float32), score, done, beams, 7, 0))
        score, _, parent, done = new
        pages, pos, spare, after = reorder(br, caches, parent, pos, spare)
        for c, (k, v) in zip(caches, after):
            c.pages, c.k, c.v = pages, k, v
        history = [[(list(history[p][l][0]), list(history[p][l][1])) for l in range(layers)] for p in parent]
    assert np.all(pos == start + 12)
