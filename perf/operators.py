"""What is measured of the gated delta rule and of the root-mean-square norm.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``run()`` makes one pass: the
plain torch form, or (``own``) the calls that a program makes of the package.  ``exact()`` computes the
same from the definition, in 64 bits and token by token.

Operators
  prefill  ``gated_delta_rule``       o and final states of whole sequences, one batch or packed
  train    ``gated_delta_rule``       o, final states and the gradients of every input
  step     ``gated_delta_step``       one or a few tokens against a pool of states, updated in place
  norm     ``rms_norm``               residual addition and norm
  quant    ``rms_norm_fp8``           the same with an 8-bit output and its scales
  norm_train ``rms_norm``             norm, residual and the gradients of every input
"""
import math
import random

import torch

own = False

CHUNK = 64
FP8_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _delta(name, op, seqs, tokens, packed, kh, vh, dk, dv, dtype, gates, initial):
    return dict(name=name, op=op, seqs=seqs, tokens=tokens, packed=packed, kh=kh, vh=vh, dk=dk,
                dv=dv, dtype=dtype, gates=gates, initial=initial)


def _norm(name, op, rows, width, dtype, residual, group=0):
    return dict(name=name, op=op, rows=rows, width=width, dtype=dtype, residual=residual,
                group=group)


def listed():
    return [
        # one user's next token: every launch counts (16 heads of 128, the study's model width)
        _delta("step_b1", "step", 1, 1, False, 16, 16, 128, 128, "bf16", "fp32", True),
        # a full decoding batch with shared key heads, some rows of the batch empty
        _delta("step_b128", "step", 128, 1, False, 8, 16, 128, 128, "bf16", "bf16", True),
        # a short prompt of odd length
        _delta("prefill_t77", "prefill", 1, 77, False, 16, 16, 128, 128, "bf16", "fp32", False),
        # the study's 16K-token sequence through one layer
        _delta("prefill_16k", "prefill", 1, 16384, False, 16, 16, 128, 128, "bf16", "fp32", False),
        # prompts of different lengths packed one behind the other, continued from states
        _delta("prefill_packed", "prefill", 24, 12000, True, 8, 16, 128, 128, "bf16", "fp32", True),
        # a training step of one layer: four sequences of 4096
        _delta("train_4x4k", "train", 4, 4096, False, 16, 16, 128, 128, "bf16", "bf16", False),
        # the fp32 module, small heads of odd sizes, shared key heads, an odd length
        _delta("train_fp32", "train", 2, 333, False, 2, 4, 64, 96, "fp32", "fp32", True),
        # the norm between two layers, one token and a whole 16K sequence
        _norm("norm_r1", "norm", 1, 2048, "bf16", True),
        _norm("norm_16k", "norm", 16384, 2048, "bf16", True),
        # the norm in front of an 8-bit product, a scale for each row
        _norm("quant_16k", "quant", 16384, 2048, "bf16", True),
        # the norm in front of an 8-bit product, decoding, a scale for each 128 values
        _norm("quant_r128", "quant", 128, 2048, "bf16", True, 128),
        # the norm's training step
        _norm("norm_train_16k", "norm_train", 16384, 2048, "bf16", True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "train", "step", "norm", "quant", "norm_train"])
    if op in ("norm", "quant", "norm_train"):
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        width = _log(rng, 64, 8192)
        group = 0
        if op == "quant" and rng.random() < 0.5:
            group, width = 128, (width + 127) // 128 * 128
        elif rng.random() < 0.6:
            width = (width + 7) // 8 * 8
        rows = _log(rng, 1, min(16384, 2 ** 24 // width))
        return _norm("", op, rows, width, dtype, rng.random() < 0.7, group)
    kh = rng.choice([1, 2, 4, 8, 16])
    vh = kh * rng.choice([1, 1, 2, 4])
    dk, dv = rng.choice([32, 64, 96, 128, 128]), rng.choice([32, 64, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    gates = "fp32" if dtype == "fp32" or (op != "train" and rng.random() < 0.5) else "bf16"
    if op == "step":
        return _delta("", op, _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5]), False, kh,
                      min(vh, 32), dk, dv, dtype, gates, True)
    # tokens x value heads, at most those of the largest listed case of the kind (fp32: a 16th)
    most = 16384 * 16 // (16 if dtype == "fp32" else 1)
    packed = rng.random() < 0.5
    seqs = _log(rng, 2, 32) if packed else _log(rng, 1, 8)
    each = most // vh // (1 if packed else seqs)
    tokens = _log(rng, 1 if not packed else seqs, min(16384 if op == "prefill" else 8192, each))
    return _delta("", op, seqs, tokens, packed, kh, vh, dk, dv, dtype, gates, rng.random() < 0.5)


def _lengths(case):
    """Lengths of a packed case's sequences: ragged, an empty one and a single token among them."""
    n, total = case["seqs"], case["tokens"]
    r = random.Random(n * 100003 + total)
    w = [r.uniform(0.2, 1.0) for _ in range(n)]
    lens = [int(total * x / sum(w)) for x in w]
    if n >= 4:
        lens[1], lens[2] = 0, min(1, total)
    lens[-1] += total - sum(lens)
    return lens if lens[-1] >= 0 else [total] + [0] * (n - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] in ("norm", "quant", "norm_train"):
        shape = (case["rows"], case["width"])
        s["x"] = randn(*shape).to(dt)
        s["w"] = (1 + 0.1 * randn(case["width"])).to(dt)
        s["res"] = (2 * randn(*shape)).to(dt) if case["residual"] else None
        if case["op"] == "norm_train":
            s["dy"], s["dh"] = randn(*shape).to(dt), randn(*shape).to(dt)
        return s
    B, T = (1, case["tokens"]) if case["packed"] else (case["seqs"], case["tokens"])
    kh, vh, dk, dv = case["kh"], case["vh"], case["dk"], case["dv"]
    gt = TYPES[case["gates"]]
    # unit-length queries and keys, decays and write strengths as a gated delta layer makes them
    s["q"] = torch.nn.functional.normalize(randn(B, T, kh, dk), dim=-1).to(dt)
    s["k"] = torch.nn.functional.normalize(randn(B, T, kh, dk), dim=-1).to(dt)
    s["v"] = randn(B, T, vh, dv).to(dt)
    rate = torch.exp(torch.linspace(math.log(0.01), math.log(4.0), vh, device="cuda"))
    s["g"] = (-rate * torch.nn.functional.softplus(randn(B, T, vh) - 3)).to(gt)
    s["beta"] = torch.sigmoid(randn(B, T, vh)).to(gt)
    s["scale"] = dk ** -0.5
    n = case["seqs"]
    if case["op"] == "step":
        pool = n + n // 2 + 1
        s["state"] = 0.5 * randn(pool, vh, dk, dv)
        idx = torch.randperm(pool, generator=gen, device="cuda")[:n].to(torch.int32)
        if n >= 8:
            idx[n // 3::8] = -1  # empty rows of the batch
        s["idx"] = idx
        return s
    s["s0"] = 0.5 * randn(n, vh, dk, dv) if case["initial"] else None
    if case["packed"]:
        lens = _lengths(case)
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32,
                               device="cuda")
        s["longest"] = max(lens)
    if case["op"] == "train":
        s["do"] = randn(B, T, vh, dv).to(dt)
        s["ds"] = 0.1 * randn(n, vh, dk, dv)
    return s


# ------------------------------------------------------------------ the plain forms

def _plain_chunks(q, k, v, g, beta, scale, state):
    """The delta rule by chunks of CHUNK tokens, fp32: q, k [N, L, H, dk], v [N, L, H, dv],
    g, beta [N, L, H], state [N, H, dk, dv]."""
    N, L, H, dk = q.shape
    dv = v.shape[-1]
    nc = max(1, -(-L // CHUNK))

    def cut(x):
        x = torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, nc * CHUNK - L])
        return x.reshape(N, nc, CHUNK, H, -1).permute(0, 3, 1, 2, 4)  # [N, H, nc, C, *]

    q, k, v, beta = cut(q), cut(k), cut(v), cut(beta.unsqueeze(-1))
    cum = cut(g.unsqueeze(-1)).double().cumsum(3)  # [N, H, nc, C, 1]
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.where(low, cum - cum.transpose(-1, -2), -math.inf).exp().float()
    strict = (beta * decay * (k @ k.transpose(-1, -2))).tril(-1)
    inv = torch.eye(CHUNK, device=q.device) - strict  # (I + strict)^-1 by doubling
    power = strict @ strict
    for _ in range(5):
        inv = inv + power @ inv
        power = power @ power
    inner = decay * (q @ k.transpose(-1, -2))
    grown = cum.exp().float()
    left = (cum[..., -1:, :] - cum).exp().float()
    out = []
    for c in range(nc):
        qc, kc, gc = q[:, :, c], k[:, :, c], grown[:, :, c]
        new = inv[:, :, c] @ (beta[:, :, c] * (v[:, :, c] - gc * (kc @ state)))
        out.append(gc * (qc @ state) + inner[:, :, c] @ new)
        state = gc[..., -1:, :] * state + (left[:, :, c] * kc).transpose(-1, -2) @ new
    o = torch.stack(out, 2).permute(0, 2, 3, 1, 4).reshape(N, nc * CHUNK, H, dv)[:, :L]
    return scale * o, state


def _plain_delta(s, q, k, v, g, beta, s0):
    """(o, final state) in fp32 of fp32 inputs, packed sequences laid out side by side."""
    case = s["case"]
    rep = case["vh"] // case["kh"]
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    if s0 is None:
        s0 = torch.zeros(case["seqs"], case["vh"], case["dk"], case["dv"], device=q.device)
    if not case["packed"]:
        return _plain_chunks(q, k, v, g, beta, s["scale"], s0)
    cu = s["cu"].long()
    at = cu[:-1, None] + torch.arange(max(1, s["longest"]), device=q.device)
    real = at < cu[1:, None]
    at = at.clamp(max=max(0, case["tokens"] - 1))

    def side(x):
        x = x[0][at]
        return torch.where(real.reshape(real.shape + (1,) * (x.dim() - 2)), x, 0.0)

    o, state = _plain_chunks(side(q), side(k), side(v), side(g), side(beta), s["scale"], s0)
    row = torch.arange(case["tokens"], device=q.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return o[seq, row - cu[seq]].unsqueeze(0), state


def _plain_step(s):
    case, dt = s["case"], s["q"].dtype
    rep = case["vh"] // case["kh"]
    real = (s["idx"] >= 0).float()[:, None, None, None]
    at = s["idx"].long().clamp(min=0)
    old = s["state"][at]
    state, out = old, []
    for t in range(case["tokens"]):
        q, k = (s[n][:, t].float().repeat_interleave(rep, 1).unsqueeze(-1) for n in "qk")
        state = state * s["g"][:, t].float().exp()[..., None, None]
        kept = (k * state).sum(-2)
        new = s["beta"][:, t].float().unsqueeze(-1) * (s["v"][:, t].float() - kept)
        state = state + k * new.unsqueeze(-2)
        out.append(s["scale"] * (q * state).sum(-2))
    s["state"].index_add_(0, at, (state - old) * real)
    return {"o": (torch.stack(out, 1) * real).to(dt), "state": s["state"]}


def _plain_norm(x, w, res, eps=1e-6):
    """(y in fp32, h): h is rounded to the inputs' type, which is what the next layer adds to."""
    dt = x.dtype
    h = x if res is None else (x.float() + res.float()).to(dt)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * w.float()
    return y, h


def _plain_quant(y, group):
    rows, width = y.shape
    y = y.reshape(rows, -1, group or width)
    most = y.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    y8 = (y * (FP8_MAX / most)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return y8.reshape(rows, width), (most / FP8_MAX).squeeze(-1)


def _plain_norm_train(s):
    x, w, dt = s["x"], s["w"].float(), s["x"].dtype
    y, h = _plain_norm(x, s["w"], s["res"])
    f = h.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)
    dy = s["dy"].float()
    p = dy * w
    d = r * (p - f * r.square() * (p * f).mean(-1, keepdim=True))
    if s["res"] is not None:
        d = d + s["dh"].float()
    d = d.to(dt)
    dw = (dy * f * r).sum(0).to(s["w"].dtype)
    return {"y": y.to(dt), "h": h, "dx": d, "dres": d if s["res"] is not None else None, "dw": dw}


def _plain(s):
    case, dt = s["case"], s["x" if "x" in s else "q"].dtype
    if case["op"] == "step":
        return _plain_step(s)
    if case["op"] == "norm":
        y, h = _plain_norm(s["x"], s["w"], s["res"])
        return {"y": y.to(dt), "h": h}
    if case["op"] == "quant":
        y, h = _plain_norm(s["x"], s["w"], s["res"])
        y8, scale = _plain_quant(y, case["group"])
        return {"y": y8, "scale": scale, "h": h}
    if case["op"] == "norm_train":
        return _plain_norm_train(s)
    names = ["q", "k", "v", "g", "beta"] + (["s0"] if s["s0"] is not None else [])
    if case["op"] == "prefill":
        with torch.no_grad():
            o, state = _plain_delta(s, *(s[n].float() for n in names[:5]), s["s0"])
        return {"o": o.to(dt), "state": state}
    leaves = [s[n].float().requires_grad_() for n in names]
    o, state = _plain_delta(s, *leaves[:5], leaves[5] if len(leaves) > 5 else None)
    grads = torch.autograd.grad([o, state], leaves, [s["do"].float(), s["ds"]])
    out = {"d" + n: x.to(s[n].dtype) for n, x in zip(names, grads)}
    return {"o": o.detach().to(dt), "state": state.detach(), **out}


# ------------------------------------------------------------------ the package's calls

def _own(s):
    import gsa_gdn_benchmarkstudy_b200 as gsa
    case = s["case"]
    if case["op"] == "step":
        o = gsa.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                                 scale=s["scale"], state_indices=s["idx"])
        return {"o": o, "state": s["state"]}
    if case["op"] in ("norm", "quant"):
        with torch.no_grad():
            if case["op"] == "norm":
                got = gsa.rms_norm(s["x"], s["w"], residual=s["res"])
                y, h = got if s["res"] is not None else (got, s["x"])
                return {"y": y, "h": h}
            got = gsa.rms_norm_fp8(s["x"], s["w"], residual=s["res"],
                                   group_size=case["group"] or None)
        return {"y": got[0], "scale": got[1], "h": got[2] if s["res"] is not None else s["x"]}
    if case["op"] == "norm_train":
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        if s["res"] is None:
            y = gsa.rms_norm(x, w)
            dx, dw = torch.autograd.grad(y, [x, w], s["dy"])
            return {"y": y.detach(), "h": s["x"], "dx": dx, "dres": None, "dw": dw}
        res = s["res"].detach().requires_grad_()
        y, h = gsa.rms_norm(x, w, residual=res)
        dx, dres, dw = torch.autograd.grad([y, h], [x, res, w], [s["dy"], s["dh"]])
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dres": dres, "dw": dw}
    names = ["q", "k", "v", "g", "beta"] + (["s0"] if s["s0"] is not None else [])
    more = dict(scale=s["scale"], cu_seqlens=s.get("cu"), output_final_state=True)
    if case["op"] == "prefill":
        with torch.no_grad():
            o, state = gsa.gated_delta_rule(*(s[n] for n in names[:5]), initial_state=s["s0"],
                                            **more)
        return {"o": o, "state": state}
    leaves = [s[n].detach().requires_grad_() for n in names]
    o, state = gsa.gated_delta_rule(*leaves[:5], initial_state=leaves[5] if len(leaves) > 5
                                    else None, **more)
    grads = torch.autograd.grad([o, state], leaves, [s["do"], s["ds"]])
    return {"o": o.detach(), "state": state.detach(),
            **{"d" + n: x for n, x in zip(names, grads)}}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("norm", "quant", "norm_train"):
        n, w = case["rows"] * case["width"], case["width"] * e
        res = 1 if case["residual"] else 0
        if case["op"] == "norm":
            return {"bytes": n * e * (2 + 2 * res) + w, "flops": n * (4 + res)}
        if case["op"] == "quant":
            scales = 4 * case["rows"] * (case["width"] // case["group"] if case["group"] else 1)
            return {"bytes": n * (e * (1 + 2 * res) + 1) + w + scales, "flops": n * (7 + res)}
        # x, res, dy, dh in; y, h, dx out (the residual's gradient is dx's)
        return {"bytes": n * e * (4 + 3 * res) + 2 * w, "flops": n * (14 + 2 * res)}
    ge = 2 if case["gates"] == "bf16" else 4
    B = 1 if case["packed"] else case["seqs"]
    t, kh, vh, dk, dv = B * case["tokens"], case["kh"], case["vh"], case["dk"], case["dv"]
    ins = t * (2 * kh * dk * e + vh * dv * e + 2 * vh * ge)
    state = case["seqs"] * vh * dk * dv * 4
    out = t * vh * dv * e
    one = t * vh * dk * dv  # one multiply-add of every state element for every token
    if case["op"] == "step":
        return {"bytes": ins + out + 2 * state, "flops": 7 * one}
    states = state * (2 if case["initial"] else 1)
    if case["op"] == "prefill":
        return {"bytes": ins + out + states, "flops": 7 * one}
    # inputs, do and the final state's gradient in; o, the final state and a gradient for each input out
    return {"bytes": 2 * ins + 2 * out + state + 2 * states - (0 if case["initial"] else state),
            "flops": 21 * one}


# ------------------------------------------------------------------ 64 bits, from the definition

def _exact_rows(case, s):
    """fp64 inputs as [N, L, ...] with L tokens a sequence (a padded token changes nothing: its
    decay is 1 and its write strength 0), and the rows of the output they go to."""
    rep = case["vh"] // case["kh"]
    x = {n: s[n].double() for n in ("q", "k", "v", "g", "beta", "do") if n in s}
    x["q"], x["k"] = x["q"].repeat_interleave(rep, 2), x["k"].repeat_interleave(rep, 2)
    if not case["packed"]:
        return x, None
    lens = _lengths(case)
    at, begin = [], 0
    for n in lens:
        at.append(torch.arange(begin, begin + n, device="cuda"))
        begin += n
    long = max(lens)
    y = {n: v.new_zeros((len(lens), long) + tuple(v.shape[2:])) for n, v in x.items()}
    for n, v in x.items():
        for i, rows in enumerate(at):
            y[n][i, :len(rows)] = v[0, rows]
    return y, at


def _exact_back(x, at):
    if at is None:
        return x
    return torch.cat([x[i, :len(rows)] for i, rows in enumerate(at)]).reshape(
        (1, -1) + tuple(x.shape[2:]))


def _exact_token(S, q, k, v, a, b, scale):
    """S <- a S + k (b (v - a S^T k))^T and scale S^T q, for one token of every sequence and head."""
    S = S * a[..., None, None]
    u = b[..., None] * (v - torch.einsum("nhkv,nhk->nhv", S, k))
    S = S + torch.einsum("nhk,nhv->nhkv", k, u)
    return S, scale * torch.einsum("nhkv,nhk->nhv", S, q)


def _exact_delta(case, s):
    x, at = _exact_rows(case, s)
    N, L = x["q"].shape[:2]
    if L > 20000 or (case["op"] == "train" and L > 9000):
        return None
    S = s["s0"].double() if s["s0"] is not None else torch.zeros(
        case["seqs"], case["vh"], case["dk"], case["dv"], dtype=torch.float64, device="cuda")
    scale, a = s["scale"], x["g"].exp()
    train, hold, o = case["op"] == "train", [], torch.zeros_like(x["v"])
    for t in range(L):
        if train and t % CHUNK == 0:
            hold.append(S)
        S, o[:, t] = _exact_token(S, x["q"][:, t], x["k"][:, t], x["v"][:, t], a[:, t],
                                  x["beta"][:, t], scale)
    out = {"o": _exact_back(o, at), "state": S}
    if not train:
        return out
    d = {n: torch.zeros_like(x[n]) for n in ("q", "k", "v", "g", "beta")}
    dS = s["ds"].double()
    for c in reversed(range(len(hold))):
        before = [hold[c]]
        ts = range(c * CHUNK, min(L, (c + 1) * CHUNK))
        for t in ts:
            before.append(_exact_token(before[-1], x["q"][:, t], x["k"][:, t], x["v"][:, t],
                                       a[:, t], x["beta"][:, t], scale)[0])
        for i, t in reversed(list(enumerate(ts))):
            q, k, v, b, do = (x[n][:, t] for n in ("q", "k", "v", "beta", "do"))
            faded = before[i] * a[:, t, :, None, None]
            err = v - torch.einsum("nhkv,nhk->nhv", faded, k)
            dS = dS + scale * torch.einsum("nhk,nhv->nhkv", q, do)
            d["q"][:, t] = scale * torch.einsum("nhkv,nhv->nhk", before[i + 1], do)
            du = torch.einsum("nhkv,nhk->nhv", dS, k)
            d["v"][:, t] = b[..., None] * du
            d["beta"][:, t] = (du * err).sum(-1)
            d["k"][:, t] = torch.einsum("nhkv,nhv->nhk", dS, b[..., None] * err) \
                - torch.einsum("nhkv,nhv->nhk", faded, d["v"][:, t])
            dS = dS - torch.einsum("nhk,nhv->nhkv", k, d["v"][:, t])
            d["g"][:, t] = (dS * faded).sum((-1, -2))
            dS = dS * a[:, t, :, None, None]
    kh, rep = case["kh"], case["vh"] // case["kh"]
    for n in ("q", "k"):
        d[n] = d[n].reshape(N, L, kh, rep, -1).sum(3)
    out |= {"d" + n: _exact_back(v, at) for n, v in d.items()}
    if s["s0"] is not None:
        out["ds0"] = dS
    return out


def _exact_step(case, s):
    rep, real = case["vh"] // case["kh"], s["idx"] >= 0
    rows = s["idx"][real].long()
    pool = s["state"].double()
    S, o = pool[rows], torch.zeros_like(s["v"], dtype=torch.float64)
    for t in range(case["tokens"]):
        q, k = (s[n][real][:, t].double().repeat_interleave(rep, 1) for n in "qk")
        S, got = _exact_token(S, q, k, s["v"][real][:, t].double(), s["g"][real][:, t].double().exp(),
                              s["beta"][real][:, t].double(), s["scale"])
        o[real, t] = got
    pool[rows] = S
    return {"o": o, "state": pool}


def _exact_norm(case, s):
    dt = s["x"].dtype
    x, w = s["x"].double(), s["w"].double()
    h = x if s["res"] is None else (x + s["res"].double()).to(dt).double()  # a rounding of the definition
    r = 1 / torch.sqrt((h * h).sum(-1, keepdim=True) / case["width"] + 1e-6)
    y = h * r * w
    if case["op"] == "norm":
        return {"y": y, "h": h}
    if case["op"] == "quant":
        part = y.reshape(case["rows"], -1, case["group"] or case["width"])
        scale = part.abs().amax(-1).clamp(min=1e-12) / FP8_MAX
        part = (part / scale[..., None]).clamp(-FP8_MAX, FP8_MAX)
        # e4m3: three bits behind the leading one, the smallest step 2^-9
        step = torch.exp2(torch.floor(torch.log2(part.abs().clamp(min=2.0 ** -6))) - 3)
        held = torch.round(part / step) * step
        return {"y": held.reshape(y.shape), "scale": scale, "h": h}
    dy = s["dy"].double()
    dx = r * (dy * w - h * r * ((dy * w * h * r).sum(-1, keepdim=True) / case["width"]))
    if s["res"] is not None:
        dx = dx + s["dh"].double()
    return {"y": y, "h": h, "dx": dx, "dres": dx if s["res"] is not None else None,
            "dw": (dy * h * r).sum(0)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        return _exact_step(case, s)
    if case["op"] in ("prefill", "train"):
        return _exact_delta(case, s)
    return _exact_norm(case, s)
