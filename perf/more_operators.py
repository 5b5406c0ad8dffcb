"""The steps of a program that generates text with a model of this library: new keys and values go into a paged cache, one new token of
each sequence attends over it, beam search picks the next tokens, and the rows of the cache follow the beams.

Four operators.  Activations are in the library's channel-first layout (``[batch][channels][S]``); column ``n = b * S + s`` is one token.
The cache of a layer is ``k, v [n_pages][kv_heads][page][hd]`` with a table ``pages [n_seqs][max_pages]``:

* ``append``: q, k and v of new tokens through the per-head norm and the rotation at each token's position, k and v into the cache;
* ``attend``: attention of one new token over positions 0 .. pos of its sequence, grouped KV heads;
* ``beam``: the best ``beams`` of all continuations of a group of beams, from logits over the vocabulary;
* ``reorder``: table rows follow the parents, the pages that are being filled are copied, in all layers at once.

The plain forms use products, sums, exponentials, comparisons and indexing in 32 bits, rounded once at the end; the beams' scores, which are
compared with one another, in 64.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One sequence of the 110 M parameter model's shape being continued: latency counts.
        dict(name="attend_one_sequence_f32", kind="attend", storage="f32", heads=12, kv=12, hd=64, page=16, batch=1, S=1, longest=256),
        # A batch of conversations of very different lengths, one layer of the 0.6 B model.
        dict(name="attend_batch_bf16", kind="attend", storage="bf16", heads=16, kv=8, hd=128, page=16, batch=1, S=64, longest=4096),
        # One document of 131 071 positions: the cache's length is the only thing that there is to share out.
        dict(name="attend_long_bf16", kind="attend", storage="bf16", heads=16, kv=8, hd=128, page=64, batch=1, S=1, longest=131071),
        # All query heads on one KV head, fp32, an odd number of sequences and pages of no power of two.
        dict(name="attend_shared_head_f32", kind="attend", storage="f32", heads=6, kv=1, hd=96, page=48, batch=91, S=1, longest=3001),
        # One new token of each of 64 sequences, with the per-head norm of the 0.6 B model: latency counts.
        dict(name="append_tokens_bf16", kind="append", storage="bf16", heads=16, kv=8, hd=128, page=16, batch=1, S=64, prompt=False, norm=True,
             longest=1024),
        # A batch of prompts of 256 positions, padded, as the model reads them before it answers.
        dict(name="append_prompts_bf16", kind="append", storage="bf16", heads=16, kv=8, hd=128, page=16, batch=16, S=256, prompt=True, norm=True,
             longest=256),
        # One long prompt of an odd length in fp32, no norm.
        dict(name="append_long_prompt_f32", kind="append", storage="f32", heads=12, kv=12, hd=64, page=32, batch=1, S=8191, prompt=True,
             norm=False, longest=8191),
        # Four beams of one prompt over a vocabulary of 32000: latency counts.
        dict(name="beam_one_prompt_f32", kind="beam", storage="f32", V=32000, batch=1, S=4, beams=4),
        # 64 prompts of eight beams over the 0.6 B model's vocabulary, logits as the classifier's product leaves them.
        dict(name="beam_batch_bf16", kind="beam", storage="bf16", V=151936, batch=1, S=512, beams=8),
        # Five beams of eleven prompts, a row of logits to a beam, a vocabulary of an odd size.
        dict(name="beam_rows_f32", kind="beam", storage="f32", V=50001, batch=55, S=1, beams=5),
        # The caches of twelve layers following four beams: latency counts.
        dict(name="reorder_one_prompt_f32", kind="reorder", storage="f32", layers=12, kv=12, hd=64, page=16, beams=4, groups=1, longest=251),
        # The caches of 28 layers following 256 beams.
        dict(name="reorder_batch_bf16", kind="reorder", storage="bf16", layers=28, kv=8, hd=128, page=32, beams=8, groups=32, longest=160),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["attend", "append", "beam", "reorder"])
    case = dict(kind=kind, storage=rng.choice(["f32", "bf16"]))
    size = 4 if case["storage"] == "f32" else 2
    heads, kv, hd = rng.choice([(12, 12, 64), (16, 8, 128), (8, 2, 64), (6, 1, 96), (5, 5, 72), (40, 2, 128)])
    page = rng.choice([16, 16, 32, 48, 64, 256])
    if kind == "attend":
        longest = _spread(rng, 1, 65536)
        n = _spread(rng, 1, max(1, min(256, 131071 * 8 * 128 * 2 // (longest * kv * hd * size))))
        columns = rng.random() < 0.5
        case.update(heads=heads, kv=kv, hd=hd, page=page, batch=1 if columns else n, S=n if columns else 1, longest=longest)
    elif kind == "append":
        prompt = rng.random() < 0.5
        most = 8191 * 6 * 768 * 4 // ((2 * heads + 4 * kv) * hd * size)
        S = _spread(rng, 1, min(8191, most)) if prompt else _spread(rng, 1, 256)
        batch = _spread(rng, 1, max(1, min(32, most // S)))
        case.update(heads=heads, kv=kv, hd=hd, page=page, batch=batch, S=S, prompt=prompt, norm=rng.random() < 0.5,
                    longest=S if prompt else _spread(rng, 16, 1024))
    elif kind == "beam":
        V, beams = _spread(rng, 200, 151936), rng.choice([1, 2, 4, 5, 8, 16])
        groups = _spread(rng, 1, max(1, min(64, 151936 * 512 * 2 // (V * beams * size))))
        batch, S = rng.choice([(1, groups * beams), (groups * beams, 1), (groups, beams)])
        case.update(V=V, batch=batch, S=S, beams=beams)
    else:
        layers, beams, longest = rng.choice([1, 6, 12, 28]), rng.choice([2, 4, 5, 8]), _spread(rng, 1, 200)
        row = 2 * layers * kv * hd * size * page * (longest // page + 3)        # bytes of a row's pages
        groups = _spread(rng, 1, max(1, min(32, (4 << 30) // (row * beams))))
        case.update(layers=layers, kv=kv, hd=hd, page=page, beams=beams, groups=groups, longest=longest)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _lengths(case, count):
    """Lengths of `count` sequences, spread over their logarithm from a tenth of the longest on; one of them is the longest."""
    longest = case["longest"]
    rng = np.random.default_rng([longest, count, case["page"]])
    n = np.maximum(1, np.floor(longest * np.exp(rng.uniform(np.log(0.1), 0.0, count)))).astype(np.int64)
    n[0] = longest
    return n


def _columns(case):
    """(seq, pos) of the new tokens of an append, numpy [batch][S]; -1: a column that is no token.  And the number of sequences."""
    B, S = case["batch"], case["S"]
    if not case["prompt"]:          # one token behind the end of each of batch * S sequences
        pos = (_lengths(case, B * S) - 1).reshape(B, S)
        return np.arange(B * S).reshape(B, S), pos, B * S
    n = _lengths(case, B)           # prompts padded to S
    pos = np.broadcast_to(np.arange(S), (B, S)).copy()
    seq = np.broadcast_to(np.arange(B)[:, None], (B, S)).copy()
    pos[pos >= n[:, None]] = -1
    seq[pos < 0] = -1
    return seq, pos, B


def _table(gen, lengths, page, spares=0):
    """Pages of sequences of these lengths, [n][max_pages], in no order; -1 where a sequence has none.  Their number, and `spares` more."""
    need = -(-np.asarray(lengths) // page)
    total = int(need.sum()) + spares
    ids = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    at = torch.from_numpy(np.concatenate([[0], np.cumsum(need)[:-1]])).cuda()
    j = torch.arange(int(need.max()), device="cuda")
    has = j[None] < torch.from_numpy(need).cuda()[:, None]
    return torch.where(has, ids[(at[:, None] + j[None]).clamp(max=total - 1)], -1).to(torch.int32), total, ids[total - spares:]


def _tables(positions, hd):
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[None] * (10000.0 ** (-2.0 * i / hd))[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["storage"]]

    def normal(*shape, dtype=dtype, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    s = dict(case=case)
    kind = case["kind"]
    if kind in ("attend", "append"):
        B, S, H, KV, hd, page = (case[n] for n in ("batch", "S", "heads", "kv", "hd", "page"))
        if kind == "attend":
            lengths = _lengths(case, B * S)
            s["pos"], s["seq"] = ints(lengths - 1).reshape(B, S), None
        else:
            seq, pos, n = _columns(case)
            lengths = np.zeros(n, np.int64)
            np.maximum.at(lengths, seq[seq >= 0], pos[seq >= 0] + 1)
            s["pos"], s["seq"] = ints(pos), ints(seq) if case["prompt"] else None
        s["pages"], total, _ = _table(gen, lengths, page)
        s["q"] = normal(B, H * hd, S)
        if kind == "attend":
            s["kc"], s["vc"] = normal(total, KV, page, hd), normal(total, KV, page, hd)
            s["scale"] = float(np.float32(1.0 / math.sqrt(hd)))
            s["o"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros((B, H, S), device="cuda")
        else:
            s["k"], s["v"] = normal(B, KV * hd, S), normal(B, KV * hd, S)
            s["kc"] = torch.zeros((total, KV, page, hd), dtype=dtype, device="cuda")
            s["vc"], s["q_out"], s["eps"] = torch.zeros_like(s["kc"]), torch.zeros_like(s["q"]), 1e-6
            s["wq"], s["wk"] = (1.0 + normal(hd, dtype=torch.float32, std=0.1) for _ in range(2)) if case["norm"] else (None, None)
            s["cos"], s["sin"] = _tables(case["longest"], hd)
    elif kind == "beam":
        V, B, S, K = case["V"], case["batch"], case["S"], case["beams"]
        N = B * S
        s["logits"] = normal(B, V, S, std=3.0)
        s["score"] = -torch.rand(N, device="cuda", generator=gen) * 6.0 - 20.0
        s["done"] = (torch.rand(N, device="cuda", generator=gen) < 0.1).to(torch.int32)
        s["score_out"] = torch.zeros_like(s["score"])
        s["token"], s["parent"], s["done_out"] = (torch.zeros(N, dtype=torch.int32, device="cuda") for _ in range(3))
        s["eos"], s["pad"] = min(2, V - 1), 0
    else:
        N, page = case["beams"] * case["groups"], case["page"]
        n = np.repeat(_lengths(case, case["groups"]), case["beams"])
        s["pages"], total, s["spare"] = _table(gen, n + page, page, N)      # room to grow: the page after the last as well
        s["spare"] = s["spare"].contiguous()
        s["pos"] = ints(n - 1)
        first = torch.arange(N, device="cuda") // case["beams"] * case["beams"]
        s["parent"] = (first + torch.randint(0, case["beams"], (N,), device="cuda", generator=gen)).to(torch.int32)
        s["cache"] = normal(case["layers"], 2, total, case["kv"], page, case["hd"])
        s["pages_out"], s["pos_out"], s["spare_out"] = torch.zeros_like(s["pages"]), torch.zeros_like(s["pos"]), torch.zeros_like(s["spare"])
    if own:
        from ane_amd import bridge as br
        br.init()
        br.check(br.lib.mi355_set_stream(torch.cuda.current_stream().cuda_stream or None))
        if kind == "reorder":
            s["caches"] = (br.KvCache * case["layers"])(*[_cache(br, s, s["cache"][i, 0], s["cache"][i, 1]) for i in range(case["layers"])])
        elif kind != "beam":
            s["caches"] = _cache(br, s, s["kc"], s["vc"])
    return s


def _cache(br, s, k, v):
    total, kv, page, hd = k.shape
    return br.KvCache(k.data_ptr(), v.data_ptr(), s["pages"].data_ptr(), total, page, s["pages"].shape[0], s["pages"].shape[1], kv, hd)


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _heads(x, heads):
    """[batch][heads*hd][S] -> fp32 [batch*S][heads][hd]"""
    B, C, S = x.shape
    return x.float().reshape(B, heads, C // heads, S).permute(0, 3, 1, 2).reshape(B * S, heads, C // heads)


def _back(x, like):
    """[batch*S][heads][hd] -> [batch][heads*hd][S], rounded"""
    B, C, S = like.shape
    return x.reshape(B, S, C).transpose(1, 2).to(like.dtype).contiguous()


def _attend(s):
    c = s["case"]
    H, KV, hd = c["heads"], c["kv"], c["hd"]
    N, T = c["batch"] * c["S"], s["pages"].shape[1] * c["page"]
    ids = s["pages"].long().clamp(min=0)
    rows = lambda x: x[ids].permute(0, 2, 1, 3, 4).reshape(N, KV, T, hd).float()        # noqa: E731
    seen = torch.arange(T, device="cuda")[None] <= s["pos"].reshape(N, 1)
    q = _heads(s["q"], H).reshape(N, KV, H // KV, hd).transpose(2, 3).contiguous()
    z = torch.matmul(rows(s["kc"]), q).transpose(2, 3).mul(s["scale"])                  # [N][KV][group][T]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - m)
    n = p.sum(-1, keepdim=True)
    o = torch.matmul((p / n).contiguous(), rows(s["vc"]))
    lse = (m + torch.log(n)).reshape(c["batch"], c["S"], H).transpose(1, 2).contiguous()
    return [_back(o.reshape(N, H, hd), s["q"]), lse]


def _append(s):
    c = s["case"]
    H, KV, hd, page = c["heads"], c["kv"], c["hd"], c["page"]
    pos = s["pos"].reshape(-1).long()
    token = pos >= 0
    seq = torch.arange(pos.numel(), device="cuda") if s["seq"] is None else s["seq"].reshape(-1).long()
    at = pos.clamp(min=0)

    def turned(x, heads, w):
        y = _heads(x, heads)
        if w is not None:
            y = y * (1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + s["eps"])) * w
        cs, sn = s["cos"][:, at].t()[:, None], s["sin"][:, at].t()[:, None]
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack((a * cs - b * sn, a * sn + b * cs), -1).reshape(y.shape)

    B, S = c["batch"], c["S"]
    q = torch.where(token.reshape(B, 1, S), _back(turned(s["q"], H, s["wq"]), s["q"]), s["q_out"])
    keep = token.nonzero()[:, 0]
    ids = s["pages"][seq[keep], at[keep] // page].long()
    s["kc"][ids, :, at[keep] % page] = turned(s["k"], KV, s["wk"])[keep].to(s["kc"].dtype)
    s["vc"][ids, :, at[keep] % page] = _heads(s["v"], KV)[keep].to(s["vc"].dtype)
    return [q, s["kc"], s["vc"]]


def _beam(s):
    c = s["case"]
    V, N, K = c["V"], c["batch"] * c["S"], c["beams"]
    x = s["logits"].transpose(1, 2).reshape(N, V).double()
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    score, done = s["score"].double()[:, None], s["done"][:, None] != 0
    pad = torch.arange(V, device="cuda")[None] == s["pad"]
    cand = torch.where(done, torch.where(pad, score, torch.full_like(score, -math.inf)), score + (x - lse))
    # the K largest values of each group; of those that equal the last of them, the ones of the lowest index
    cand = cand.reshape(N // K, K * V)
    last = torch.topk(cand, K, dim=1).values[:, -1:]
    above, equal = cand > last, cand == last
    take = above | (equal & (torch.cumsum(equal, 1) <= K - above.sum(1, keepdim=True)))
    index = torch.arange(K * V, device="cuda")[None]
    at = torch.topk(torch.where(take, index, K * V), K, dim=1, largest=False).values.sort(1).values
    best, order = torch.sort(torch.gather(cand, 1, at), dim=1, descending=True, stable=True)
    at = torch.gather(at, 1, order)
    parent = (at // V + torch.arange(N // K, device="cuda")[:, None] * K).reshape(-1)
    token = (at % V).reshape(-1)
    ended = (s["done"][parent] != 0) | (token == s["eos"])
    return [best.reshape(-1).float(), token.to(torch.int32), parent.to(torch.int32), ended.to(torch.int32)]


def _reorder(s):
    c = s["case"]
    N, page = c["beams"] * c["groups"], c["page"]
    row, parent, pos = torch.arange(N, device="cuda"), s["parent"].long(), s["pos"].long()[s["parent"].long()]
    tail = pos // page
    j = torch.arange(s["pages"].shape[1], device="cuda")[None]
    moves = (parent != row) & (pos % page != page - 1)
    old = s["pages"][parent, tail].long()
    out = torch.where(j <= tail[:, None], s["pages"][parent], s["pages"])
    out = torch.where((j == tail[:, None]) & moves[:, None], s["spare"][:, None], out)
    mine = s["pages"][row, s["pos"].long() // page]
    spare = torch.where(moves, mine, s["spare"])
    filled = torch.arange(page, device="cuda")[None] <= (pos % page)[:, None]
    go = moves.nonzero()[:, 0]
    old, new = old[go], s["spare"][go].long()
    s["cache"][:, :, new] = torch.where(filled[go][None, None, :, None, :, None], s["cache"][:, :, old], s["cache"][:, :, new])
    return [out, (pos + 1).to(torch.int32), spare, s["cache"]]


# ---- what a user's program calls ------------------------------------------------------------------------------------

def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import ctypes

    from ane_amd import bridge as br
    c = s["case"]
    kind, end = c["kind"], "_bf16_dev" if c["storage"] == "bf16" else "_dev"
    if kind == "attend":
        rc = getattr(br.lib, "mi355_attn_paged" + end)(ctypes.byref(s["caches"]), _at(s["o"]), _at(s["lse"]), _at(s["q"]), _at(s["seq"]),
                                                       _at(s["pos"]), c["heads"], c["S"], c["batch"], s["scale"])
        out = [s["o"], s["lse"]]
    elif kind == "append":
        rc = getattr(br.lib, "mi355_kv_append" + end)(ctypes.byref(s["caches"]), _at(s["q_out"]), _at(s["q"]), _at(s["k"]), _at(s["v"]),
                                                      _at(s["wq"]), _at(s["wk"]), _at(s["seq"]), _at(s["pos"]), c["heads"], c["S"],
                                                      c["batch"], _at(s["cos"]), _at(s["sin"]), c["longest"], s["eps"])
        out = [s["q_out"], s["kc"], s["vc"]]
    elif kind == "beam":
        rc = getattr(br.lib, "mi355_beam_step" + end)(_at(s["score_out"]), _at(s["token"]), _at(s["parent"]), _at(s["done_out"]),
                                                      _at(s["logits"]), _at(s["score"]), _at(s["done"]), c["V"], c["S"], c["batch"],
                                                      c["beams"], s["eos"], s["pad"])
        out = [s["score_out"], s["token"], s["parent"], s["done_out"]]
    else:
        rc = getattr(br.lib, "mi355_kv_reorder" + end)(s["caches"], c["layers"], _at(s["pages_out"]), _at(s["pos_out"]), _at(s["spare_out"]),
                                                       _at(s["parent"]), _at(s["pos"]), _at(s["spare"]), 1)
        out = [s["pages_out"], s["pos_out"], s["spare_out"], s["cache"]]
    br.check(rc, kind)
    return out


def run(state):
    if own:
        return _own(state)
    return dict(attend=_attend, append=_append, beam=_beam, reorder=_reorder)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; of the caches, the rows that are used."""
    size = 4 if case["storage"] == "f32" else 2
    if case["kind"] == "attend":
        N, H, KV, hd = case["batch"] * case["S"], case["heads"], case["kv"], case["hd"]
        n = _lengths(case, N)
        pairs, pages = int(n.sum()), int((-(-n // case["page"])).sum())
        return dict(bytes=size * (2 * pairs * KV * hd + 2 * N * H * hd) + 4 * (N * H + pages + N), flops=4 * H * hd * pairs)
    if case["kind"] == "append":
        H, KV, hd = case["heads"], case["kv"], case["hd"]
        _, pos, _ = _columns(case)
        n, places = int((pos >= 0).sum()), len(np.unique(pos[pos >= 0]))
        per = (2 * H + 4 * KV) * hd
        return dict(bytes=size * n * per + 4 * (places * hd + 3 * n), flops=n * (H + KV) * hd * (7 if case["norm"] else 3))
    if case["kind"] == "beam":
        n = case["batch"] * case["S"]
        return dict(bytes=size * case["V"] * n + 4 * 6 * n, flops=4 * case["V"] * n)
    N, page = case["beams"] * case["groups"], case["page"]
    n = np.repeat(_lengths(case, case["groups"]), case["beams"])
    # parents are drawn evenly: all but one row of `beams` moves, where the page is not full
    rows = float(np.where(n % page, n % page, 0).sum()) * (1.0 - 1.0 / case["beams"])
    copied = 2 * case["layers"] * rows * case["kv"] * case["hd"] * size
    return dict(bytes=int(2 * copied) + 4 * (2 * int(N * (-(-n // page) + 1).max()) + 5 * N), flops=0)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        B, S, H, KV, hd = (case[n] for n in ("batch", "S", "heads", "kv", "hd"))
        o, lse = torch.zeros((B, H * hd, S), dtype=torch.float64, device="cuda"), torch.zeros((B, H, S), dtype=torch.float64, device="cuda")
        pos = s["pos"].cpu().numpy()
        for b in range(B):
            for t in range(S):
                n = int(pos[b, t]) + 1
                ids = s["pages"][b * S + t, :-(-n // case["page"])].long()
                for g in range(KV):
                    k, v = (s[c][ids, g].reshape(-1, hd)[:n].double() for c in ("kc", "vc"))
                    mine = slice(g * (H // KV), (g + 1) * (H // KV))
                    z = s["q"][b, :, t].double().reshape(H, hd)[mine] @ k.t() * s["scale"]
                    o[b, mine.start * hd:mine.stop * hd, t] = (torch.softmax(z, 1) @ v).reshape(-1)
                    lse[b, mine, t] = torch.logsumexp(z, 1)
        return [o, lse]
    if kind == "append":
        seq, pos, _ = _columns(case)
        B, S, hd, page = case["batch"], case["S"], case["hd"], case["page"]
        used = torch.from_numpy(pos >= 0).cuda()
        p = torch.from_numpy(np.maximum(pos, 0)).cuda()
        turn = torch.complex(s["cos"].double(), s["sin"].double()).t()[p]                       # [B][S][hd/2]

        def turned(x, w):
            y = x.double().reshape(B, -1, hd, S).permute(0, 3, 1, 2)
            if w is not None:
                y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + s["eps"]) * w.double()
            y = torch.view_as_complex(y.reshape(*y.shape[:-1], hd // 2, 2).contiguous()) * turn[:, :, None]
            return torch.view_as_real(y).reshape(B, S, -1, hd)

        q = turned(s["q"], s["wq"]).reshape(B, S, -1).transpose(1, 2) * used[:, None]
        kc, vc = s["kc"].double(), s["vc"].double()
        k, v = turned(s["k"], s["wk"]), s["v"].double().reshape(B, -1, hd, S).permute(0, 3, 1, 2)
        flat = lambda c: c.permute(0, 2, 1, 3).reshape(-1, *c.shape[1:2], hd)                   # noqa: E731
        place = s["pages"][torch.from_numpy(np.maximum(seq, 0)).cuda(), p // page].long() * page + p % page
        out = []
        for c, new in ((kc, k), (vc, v)):
            rows = flat(c)
            rows.index_copy_(0, place[used], new[used])
            out.append(rows.reshape(c.shape[0], page, c.shape[1], hd).permute(0, 2, 1, 3).contiguous())
        return [q] + out
    if kind == "beam":
        K, V = case["beams"], case["V"]
        N = case["batch"] * case["S"]
        best = torch.zeros(N, dtype=torch.float64, device="cuda")
        for g in range(N // K):
            found = []
            for n in range(g * K, (g + 1) * K):
                if int(s["done"][n]):
                    found.append(s["score"][n:n + 1].double())
                else:
                    row = s["logits"][n // case["S"], :, n % case["S"]].double()
                    found.append(s["score"][n].double() + torch.topk(torch.log_softmax(row, 0), min(K, V)).values)
            best[g * K:(g + 1) * K] = torch.topk(torch.cat(found), K).values
        return [best, None, None, None]
    # copies: the cache's values as they are
    N, page = case["beams"] * case["groups"], case["page"]
    pages, pos, parent, spare = (s[n].cpu().numpy() for n in ("pages", "pos", "parent", "spare"))
    for n in range(N):
        at = int(pos[parent[n]])
        if parent[n] != n and (at + 1) % page:
            s["cache"][:, :, int(spare[n]), :, :at % page + 1] = s["cache"][:, :, int(pages[parent[n], at // page]), :, :at % page + 1]
    return [None, None, None, s["cache"]]
