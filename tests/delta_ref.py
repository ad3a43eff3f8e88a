"""The gated delta rule and the RMS norm in 64 bits, token by token and row by row."""
import torch


def delta_tokens(q, k, v, g, beta, scale, state=None):
    """One sequence: q, k [T, Hk, dk], v [T, Hv, dv], g, beta [T, Hv]; returns (o, S)."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    S = (state.double() if state is not None else
         torch.zeros(v.shape[1], q.shape[2], v.shape[2], dtype=torch.float64, device=v.device))
    out = []
    for t in range(q.shape[0]):
        S = S * g[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
        S = S + torch.einsum("hk,hv->hkv", k[t], u)
        out.append(scale * torch.einsum("hkv,hk->hv", S, q[t]))
    o = torch.stack(out) if out else v.new_zeros(v.shape)
    return o, S


def delta_ref(q, k, v, g, beta, scale, initial=None, bounds=None):
    """A batch [B, T, ...], or with ``bounds`` ([(begin, end), ...]) one packed row of it; rows
    outside every sequence are zero."""
    if bounds is None:
        got = [delta_tokens(q[b], k[b], v[b], g[b], beta[b], scale,
                            None if initial is None else initial[b]) for b in range(q.shape[0])]
        return torch.stack([o for o, _ in got]), torch.stack([s for _, s in got])
    pieces, states, at = [], [], 0
    zeros = v[0].double() * 0
    for n, (b, e) in enumerate(bounds):
        o, s = delta_tokens(q[0, b:e], k[0, b:e], v[0, b:e], g[0, b:e], beta[0, b:e], scale,
                            None if initial is None else initial[n])
        pieces += [zeros[at:b], o]
        states.append(s)
        at = e
    return torch.cat(pieces + [zeros[at:]])[None], torch.stack(states)


def norm_ref(x, w, eps, res=None):
    """(y, h) in 64 bits; h rounded to the inputs' type, as the operator defines it (the sum of
    two values of that type is exact in 64 bits, so this is the one rounding)."""
    h = x.double() if res is None else (x.double() + res.double()).to(x.dtype).double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double(), h


def rel(a, b):
    """2-norm of the difference over 2-norm of the exact result."""
    d, n = (a.double() - b.double()).norm().item(), b.double().norm().item()
    return d / n if n else (0.0 if d == 0 else float("inf"))
