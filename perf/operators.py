"""The products and the attention of a layer, as a training program that keeps its activations on the GPU calls them.

Four operators, each in the library's channel-first layout (``[batch][channels][positions]``, positions contiguous):

* ``linear_fwd``: ``y = res + alpha * act(w x + bias)``, activations and weights stored as bfloat16;
* ``linear_bwd``: its gradients: ``dx = alpha * (w' dy) * act'(x_pre)`` (the activation of the layer below rides in the
  epilogue), ``dw = alpha * dy x'`` and ``dbias``, both fp32;
* ``attn_fwd``: causal attention over whole prompts, grouped KV heads, sequences of different lengths packed into a row;
* ``attn_bwd``: the gradients of q, k and v.

The plain forms below use products, sums, exponentials and comparisons in 32 bits, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # A layer's attention on one sequence, as the training loops of the 110 M parameter model call it: latency counts.
        dict(name="attn_fwd_one_sequence", kind="attn_fwd", storage="f32", heads=12, kv=12, hd=64, S=256, batch=1, seqs=0, pad=0),
        # The same layer position in a batched bfloat16 step of the 0.6 B model, two query heads to a KV head.
        dict(name="attn_fwd_batch_bf16", kind="attn_fwd", storage="bf16", heads=16, kv=8, hd=128, S=256, batch=16, seqs=0, pad=0),
        # Long prompts of very different lengths packed into one row, the row's end unused.
        dict(name="attn_fwd_packed_long_bf16", kind="attn_fwd", storage="bf16", heads=16, kv=8, hd=128, S=8191, batch=1, seqs=9, pad=61),
        # Gradients of a batch in fp32, the loops' own storage.
        dict(name="attn_bwd_batch_f32", kind="attn_bwd", storage="f32", heads=16, kv=8, hd=128, S=256, batch=8, seqs=0, pad=0),
        # Gradients of one long sequence in bfloat16.
        dict(name="attn_bwd_long_bf16", kind="attn_bwd", storage="bf16", heads=16, kv=8, hd=128, S=4096, batch=1, seqs=0, pad=0),
        # Gradients of short sequences of odd lengths packed into rows of an odd length.
        dict(name="attn_bwd_packed_odd_bf16", kind="attn_bwd", storage="bf16", heads=12, kv=4, hd=64, S=997, batch=4, seqs=7, pad=30),
        # One position through a projection: all of the weights are read for one column.
        dict(name="linear_fwd_one_token", kind="linear_fwd", M=2048, K=1024, S=1, batch=1, act="none", bias=False, pre=False, res=False),
        # The output projection of a batched step with the scaled residual.
        dict(name="linear_fwd_residual", kind="linear_fwd", M=1024, K=2048, S=256, batch=16, act="none", bias=False, pre=False, res=True),
        # The first product of a feed-forward block on sequences of an odd length: bias, activation, its input kept.
        dict(name="linear_fwd_act_odd", kind="linear_fwd", M=2048, K=768, S=197, batch=8, act="gelu", bias=True, pre=True, res=False),
        # The classifier's product over a vocabulary of 32000 for a batch of text.
        dict(name="linear_fwd_vocabulary", kind="linear_fwd", M=32000, K=768, S=256, batch=16, act="none", bias=False, pre=False, res=False),
        # Gradients of the second product of a feed-forward block, the activation before it in the epilogue.
        dict(name="linear_bwd_act", kind="linear_bwd", M=1024, K=2048, S=256, batch=16, act="silu", bias=True),
        # Gradients of a projection on one sequence.
        dict(name="linear_bwd_one_sequence", kind="linear_bwd", M=768, K=768, S=256, batch=1, act="none", bias=True),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["attn_fwd", "attn_bwd", "linear_fwd", "linear_bwd"])
    if kind.startswith("attn"):
        heads, kv, hd = rng.choice([(12, 12, 64), (16, 8, 128), (8, 2, 64), (6, 1, 96), (5, 5, 72)])
        S = _spread(rng, 1, 8191 if kind == "attn_fwd" else 4096)
        cells = 16 * (8191 if kind == "attn_fwd" else 4096) ** 2        # heads x batch x S x S of the largest listed case
        batch = _spread(rng, 1, max(1, min(32, cells // (heads * S * S))))
        seqs = _spread(rng, 1, min(S, 32)) if rng.random() < 0.6 else 0
        pad = rng.randint(0, S // 8) if seqs else 0
        return dict(kind=kind, storage=rng.choice(["f32", "bf16"]), heads=heads, kv=kv, hd=hd, S=S, batch=batch, seqs=seqs, pad=pad)
    M, K = _spread(rng, 64, 4096), _spread(rng, 64, 4096)
    if rng.random() < 0.6:
        M, K = max(64, M & -64), max(64, K & -64)
    S = rng.choice([256, 1, _spread(rng, 2, 2048)])
    batch = _spread(rng, 1, max(1, min(32, 8192 // S)))
    case = dict(kind=kind, M=M, K=K, S=S, batch=batch, act=rng.choice(["none", "relu", "silu", "gelu"]), bias=rng.random() < 0.5)
    if kind == "linear_fwd":
        case.update(pre=rng.random() < 0.3, res=rng.random() < 0.5)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _offsets(case):
    """[batch][seqs + 1]: where each row's sequences begin and end; lengths spread over their logarithm, the last `pad`
    positions in no sequence."""
    n, S, room = case["seqs"], case["S"], case["S"] - case["pad"]
    rng = np.random.default_rng([n, S, case["pad"], case["batch"], case["heads"]])
    cu = np.zeros((case["batch"], n + 1), np.int64)
    for b in range(case["batch"]):
        share = np.exp(rng.uniform(0.0, 3.0, n))
        cu[b, 1:] = np.floor(np.cumsum(share) / share.sum() * room + 1e-9)
        cu[b, n] = room
    return cu


def _starts(case):
    """[batch][S]: the first position of each position's sequence, S where it is in none."""
    S, B = case["S"], case["batch"]
    if not case["seqs"]:
        return torch.zeros((B, S), dtype=torch.int64, device="cuda")
    cu = torch.from_numpy(_offsets(case)).cuda()
    at = torch.arange(S, device="cuda").expand(B, S).contiguous()
    seq = torch.searchsorted(cu[:, 1:].contiguous(), at, right=True)
    start = torch.gather(cu, 1, seq.clamp(max=case["seqs"]))
    return torch.where(seq < case["seqs"], start, torch.full_like(start, S))


def _pairs(case):
    """(query, key) pairs of one head of the whole batch that the mask leaves."""
    if not case["seqs"]:
        return case["batch"] * case["S"] * (case["S"] + 1) // 2
    n = np.diff(_offsets(case), axis=1)
    return int(np.sum(n * (n + 1) // 2))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).to(dtype)

    B, S = case["batch"], case["S"]
    s = dict(case=case)
    if case["kind"].startswith("attn"):
        dtype, H, KV, hd = DTYPES[case["storage"]], case["heads"], case["kv"], case["hd"]
        s.update(q=normal(B, H * hd, S, dtype=dtype), k=normal(B, KV * hd, S, dtype=dtype), v=normal(B, KV * hd, S, dtype=dtype),
                 start=_starts(case), scale=float(np.float32(1.0 / math.sqrt(hd))), bounds=None)
        s["o"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros((B, H, S), device="cuda")
        if case["kind"] == "attn_bwd":
            s["do"] = normal(B, H * hd, S, dtype=dtype)
            s["dq"], s["dk"], s["dv"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
            s["o"], s["lse"] = _attn_fwd(s)         # what the forward pass left behind
    else:
        M, K = case["M"], case["K"]
        s.update(w=normal(M, K, std=1.0 / math.sqrt(K)), x=normal(B, K, S), alpha=1.0, pre=None, res=None, bias=None)
        if case["kind"] == "linear_fwd":
            s["y"] = torch.zeros((B, M, S), dtype=torch.bfloat16, device="cuda")
            if case["bias"]:
                s["bias"] = normal(M, dtype=torch.float32, std=0.5)
            if case["pre"]:
                s["pre"] = torch.zeros_like(s["y"])
            if case["res"]:
                s["res"], s["alpha"] = normal(B, M, S), float(np.float32(1.0 / math.sqrt(24.0)))
        else:
            s.update(dy=normal(B, M, S), alpha=float(np.float32(1.0 / math.sqrt(24.0))), dx=torch.zeros_like(s["x"]),
                     dw=torch.zeros((M, K), device="cuda"), dbias=torch.zeros(M, device="cuda") if case["bias"] else None)
            if case["act"] != "none":
                s["pre"] = normal(B, K, S)
    if own:
        from ane_amd import bridge as br
        br.init()
        br.check(br.lib.mi355_set_stream(torch.cuda.current_stream().cuda_stream or None))
        if case.get("seqs"):
            s["cu"] = torch.from_numpy(_offsets(case).astype(np.int32)).cuda()
            s["bounds"] = torch.empty((B, 2, S), dtype=torch.int32, device="cuda")
            br.check(br.lib.mi355_attn_plan_dev(_at(s["bounds"]), _at(s["cu"]), case["seqs"], S, B), "attn_plan")
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _act(a, x):
    if a == "relu":
        return torch.clamp(x, min=0.0)
    if a == "silu":
        return x / (1.0 + torch.exp(-x))
    if a == "gelu":
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


def _act_slope(a, x):
    if a == "relu":
        return (x > 0).to(x.dtype)
    if a == "silu":
        g = 1.0 / (1.0 + torch.exp(-x))
        return g * (1.0 + x * (1.0 - g))
    if a == "gelu":
        t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * x * x)
    return torch.ones_like(x)


def _linear_fwd(s):
    c = s["case"]
    z = torch.matmul(s["w"].float(), s["x"].float())
    if c["bias"]:
        z = z + s["bias"][:, None]
    y = s["alpha"] * _act(c["act"], z)
    if c["res"]:
        y = s["res"].float() + y
    return [y.to(torch.bfloat16)] + ([z.to(torch.bfloat16)] if c["pre"] else [])


def _linear_bwd(s):
    c = s["case"]
    dy = s["dy"].float()
    dx = s["alpha"] * torch.matmul(s["w"].float().t().contiguous(), dy)
    if c["act"] != "none":
        dx = dx * _act_slope(c["act"], s["pre"].float())
    columns = dy.transpose(0, 1).reshape(c["M"], -1)
    dw = s["alpha"] * torch.matmul(columns, s["x"].float().transpose(0, 1).reshape(c["K"], -1).t().contiguous())
    return [dx.to(torch.bfloat16), dw] + ([s["alpha"] * columns.sum(1)] if c["bias"] else [])


def _scores(s):
    """Masked and scaled scores [B][KV][group][query][key] of fp32 rows, and the rows [B][KV][...] of q, k and v."""
    c = s["case"]
    B, H, KV, hd, S = c["batch"], c["heads"], c["kv"], c["hd"], c["S"]
    q = s["q"].float().reshape(B, KV, H // KV, hd, S).transpose(3, 4).reshape(B, KV, H // KV * S, hd)
    k, v = (s[n].float().reshape(B, KV, hd, S) for n in ("k", "v"))
    at = torch.arange(S, device="cuda")
    allowed = (at[None, None, :] >= s["start"][:, :, None]) & (at[None, :] <= at[:, None])[None]
    z = torch.matmul(q, k).mul_(s["scale"]).reshape(B, KV, H // KV, S, S)
    return z.masked_fill_(~allowed[:, None, None], -math.inf), q, k, v


def _softmax(z):
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)         # rows that the mask leaves empty
    p = (z - m).exp_()
    n = p.sum(-1, keepdim=True)
    p.div_(torch.where(n == 0, torch.ones_like(n), n))
    return p, (m + torch.log(n))[..., 0]


def _attn_fwd(s):
    c = s["case"]
    B, H, KV, hd, S = c["batch"], c["heads"], c["kv"], c["hd"], c["S"]
    z, _, _, v = _scores(s)
    p, lse = _softmax(z)
    o = torch.matmul(p.reshape(B, KV, H // KV * S, S), v.transpose(2, 3).contiguous())
    o = o.reshape(B, H, S, hd).transpose(2, 3).reshape(B, H * hd, S)
    used = (s["start"] < S)[:, None, :]             # columns of no sequence stay as they were
    return [torch.where(used, o.to(s["o"].dtype), s["o"]), torch.where(used, lse.reshape(B, H, S), s["lse"])]


def _attn_bwd(s):
    c = s["case"]
    B, H, KV, hd, S = c["batch"], c["heads"], c["kv"], c["hd"], c["S"]
    G = H // KV
    z, q, k, v = _scores(s)
    p, _ = _softmax(z)
    del z
    p = p.reshape(B, KV, G * S, S)
    do = s["do"].float().reshape(B, KV, G, hd, S).transpose(3, 4).reshape(B, KV, G * S, hd)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dz = torch.matmul(do, v)
    dz = dz.sub_((dz * p).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    del p
    dq = torch.matmul(dz, k.transpose(2, 3).contiguous())
    dk = torch.matmul(dz.transpose(2, 3).contiguous(), q)
    used = (s["start"] < S)[:, None, :]
    return [torch.where(used, g.transpose(-2, -1).reshape(old.shape).to(old.dtype), old)
            for g, old in ((dq.reshape(B, H, S, hd), s["dq"]), (dk, s["dk"]), (dv, s["dv"]))]


# ---- what a user's program calls ------------------------------------------------------------------------------------

def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from ane_amd import bridge as br
    c = s["case"]
    end = "_bf16_dev" if c.get("storage") == "bf16" else "_dev"
    if c["kind"] == "linear_fwd":
        rc = br.lib.mi355_linear_fwd_bf16_dev(_at(s["y"]), _at(s["pre"]), _at(s["x"]), _at(s["w"]), _at(s["bias"]), ACTS[c["act"]],
                                              _at(s["res"]), s["alpha"], c["M"], c["K"], c["S"], c["batch"])
        out = [s["y"]] + ([s["pre"]] if c["pre"] else [])
    elif c["kind"] == "linear_bwd":
        rc = br.lib.mi355_linear_bwd_bf16_dev(_at(s["dx"]), _at(s["dw"]), _at(s["dbias"]), _at(s["dy"]), _at(s["x"]), _at(s["w"]),
                                              s["alpha"], ACTS[c["act"]], _at(s["pre"]), 0, c["M"], c["K"], c["S"], c["batch"])
        out = [s["dx"], s["dw"]] + ([s["dbias"]] if c["bias"] else [])
    elif c["kind"] == "attn_fwd":
        rc = getattr(br.lib, "mi355_attn_fwd" + end)(_at(s["o"]), _at(s["lse"]), _at(s["q"]), _at(s["k"]), _at(s["v"]), _at(s["bounds"]),
                                                     c["heads"], c["kv"], c["hd"], c["S"], c["batch"], s["scale"])
        out = [s["o"], s["lse"]]
    else:
        rc = getattr(br.lib, "mi355_attn_bwd" + end)(_at(s["dq"]), _at(s["dk"]), _at(s["dv"]), _at(s["do"]), _at(s["q"]), _at(s["k"]),
                                                     _at(s["v"]), _at(s["o"]), _at(s["lse"]), _at(s["bounds"]), c["heads"], c["kv"],
                                                     c["hd"], c["S"], c["batch"], s["scale"])
        out = [s["dq"], s["dk"], s["dv"]]
    br.check(rc, c["kind"])
    return out


def run(state):
    if own:
        return _own(state)
    return dict(linear_fwd=_linear_fwd, linear_bwd=_linear_bwd, attn_fwd=_attn_fwd, attn_bwd=_attn_bwd)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; the products of the pairs that the mask leaves (two forward, five
    backward), of every column for the linear ones."""
    B, S = case["batch"], case["S"]
    if case["kind"].startswith("attn"):
        size, q, kv = (4 if case["storage"] == "f32" else 2), case["heads"] * case["hd"], case["kv"] * case["hd"]
        n, pairs = B * S, _pairs(case)
        if case["kind"] == "attn_fwd":
            return dict(bytes=size * n * (2 * q + 2 * kv) + 4 * n * case["heads"], flops=4 * q * pairs)
        return dict(bytes=size * n * (4 * q + 4 * kv) + 4 * n * case["heads"], flops=10 * q * pairs)
    M, K, n = case["M"], case["K"], B * S
    if case["kind"] == "linear_fwd":
        return dict(bytes=2 * (M * K + K * n + M * n * (1 + case["pre"] + case["res"])), flops=2 * M * K * n)
    return dict(bytes=2 * (M * K + 2 * K * n + M * n + (K * n if case["act"] != "none" else 0)) + 4 * M * K, flops=4 * M * K * n)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    B, S = case["batch"], case["S"]
    if not case["kind"].startswith("attn"):
        act = dict(none=lambda t: t, relu=torch.relu, silu=lambda t: t * torch.sigmoid(t),
                   gelu=lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))[case["act"]]
        w, x = s["w"].double(), s["x"].double()
        if case["kind"] == "linear_fwd":
            y, z = [], []
            for b in range(B):
                z.append(w @ x[b] + (s["bias"].double()[:, None] if case["bias"] else 0.0))
                y.append(s["alpha"] * act(z[-1]) + (s["res"][b].double() if case["res"] else 0.0))
            return [torch.stack(y)] + ([torch.stack(z)] if case["pre"] else [])
        dx, dw, db = [], torch.zeros_like(w), torch.zeros(case["M"], dtype=torch.float64, device="cuda")
        for b in range(B):
            dy = s["dy"][b].double()
            g = w.t() @ dy * s["alpha"]
            if case["act"] != "none":
                at = s["pre"][b].double().requires_grad_()
                g = torch.autograd.grad(act(at).sum(), at)[0] * g
            dx.append(g)
            dw += s["alpha"] * (dy @ x[b].t())
            db += s["alpha"] * dy.sum(1)
        return [torch.stack(dx), dw] + ([db] if case["bias"] else [])
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    back = case["kind"] == "attn_bwd"
    if B * H * S * S * hd > 3e12:
        return None
    out = [s["o"].double(), s["lse"].double()] if not back else [s[n].double() for n in ("dq", "dk", "dv")]
    cu = _offsets(case) if case["seqs"] else np.array([[0, S]] * B)
    for b in range(B):
        for lo, hi in zip(cu[b, :-1].tolist(), cu[b, 1:].tolist()):
            if hi == lo:
                continue
            later = torch.ones((hi - lo, hi - lo), device="cuda").triu(1).bool()
            for g in range(KV):
                k, v = (s[n][b, g * hd:(g + 1) * hd, lo:hi].double().requires_grad_(back) for n in ("k", "v"))
                for h in range(g * (H // KV), (g + 1) * (H // KV)):
                    rows = slice(h * hd, (h + 1) * hd)
                    q = s["q"][b, rows, lo:hi].double().requires_grad_(back)
                    z = (q.t() @ k * s["scale"]).masked_fill(later, -math.inf)
                    o = v @ torch.softmax(z, 1).t()
                    if back:
                        o.backward(s["do"][b, rows, lo:hi].double())
                        out[0][b, rows, lo:hi] = q.grad
                    else:
                        out[0][b, rows, lo:hi], out[1][b, h, lo:hi] = o, torch.logsumexp(z, 1)
                if back:
                    out[1][b, g * hd:(g + 1) * hd, lo:hi], out[2][b, g * hd:(g + 1) * hd, lo:hi] = k.grad, v.grad
    return out
