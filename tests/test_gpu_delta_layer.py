"""The norm and the gated delta rule together, as a layer's token mixer uses them: a packed batch
of prompts, tokens after it against a pool of states, and a training step.

Each stage is held to its own tolerance (derived in test_gpu_delta.py and test_gpu_norm.py)
against 64 bits that start from the operators' inputs to that stage; states and outputs of the
tokens behind a prompt against the token-by-token definition over prompt and tokens at once.  The
training step's gradients pass three stages, each off by at most 16e-6 (fp32), and five inputs'
shares, which may cancel to a fifth of their size: 3 * 5 * 16e-6 = 2.4e-4.
"""
import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib
from delta_ref import delta_ref, delta_tokens, norm_ref, rel

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
NORM = {"fp32": 4e-6, "bf16": 2.0 ** -8}
OUT = {"fp32": 8e-6, "bf16": 2.0 ** -8}
STATE = {"fp32": 8e-6, "bf16": 2.0 ** -15}
HK, HV, DK, DV = 2, 4, 64, 96
WIDTH = 2 * HK * DK + HV * DV + 2 * HV  # q, k, v, decay, strength of a token


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


def inputs(n, unit, norm):
    """q, k, v, g, beta from a row of WIDTH values; `norm` makes queries and keys unit-length."""
    q, k, v, g, b = n.split([HK * DK, HK * DK, HV * DV, HV, HV], -1)
    q, k = (norm(t.unflatten(-1, (HK, DK)), unit) for t in (q, k))
    gates = torch.nn.functional.softplus(g.float() - 2), torch.sigmoid(b.float())
    if n.dtype == torch.float64:
        gates = torch.nn.functional.softplus(g - 2), torch.sigmoid(b)
    return q, k, v.unflatten(-1, (HV, DV)), -gates[0], gates[1]


def weights(dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)

    def near_one(n):
        return (1 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(dtype)

    return near_one(WIDTH), torch.full((DK,), DK ** -0.5, device="cuda").to(dtype), near_one(DV)


def rows(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_prompts_then_tokens(dtype):
    dt, lens, steps = DT[dtype], [70, 1, 130], 5
    w_in, unit, w_out = weights(dt)
    total, n = sum(lens), len(lens)
    cu = torch.tensor([0, 70, 71, 201], dtype=torch.int32, device="cuda")
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    pool = torch.full((6, HV, DK, DV), 7.0, device="cuda")

    def mix(x, res, run):
        h_in, h = gsa.rms_norm(x, w_in, residual=res)
        ry, rh = norm_ref(x, w_in, 1e-6, res)
        assert torch.equal(h.double(), rh) and rel(h_in, ry) <= NORM[dtype]
        args = inputs(h_in, unit, gsa.rms_norm)
        o = run(*args)
        y8, scale = gsa.rms_norm_fp8(gsa.rms_norm(o, w_out).flatten(-2), w_in[:HV * DV],
                                     group_size=128)
        got = (y8.float().unflatten(-1, (-1, 128)) * scale[..., None]).flatten(-2)
        want = norm_ref(norm_ref(o, w_out, 1e-6)[0].to(dt).flatten(-2), w_in[:HV * DV], 1e-6)[0]
        # half a step of e4m3, 2^-4, and of the type between the norms
        assert rel(got, want) <= 2.0 ** -4 + 2 * NORM[dtype]
        return args, o

    with torch.no_grad():
        x, res = rows(1, total, WIDTH, dtype=dt, seed=1), rows(1, total, WIDTH, dtype=dt, seed=2)

        def prompt(*a):
            o, S = gsa.gated_delta_rule(*a, cu_seqlens=cu, output_final_state=True)
            pool[slots.long()] = S
            return o

        seen, o = mix(x, res, prompt)
        outs = [[o[0, b:e]] for b, e in ((0, 70), (70, 71), (71, 201))]
        parts = [[[t[0, b:e] for t in seen]] for b, e in ((0, 70), (70, 71), (71, 201))]
        for s in range(steps):
            x, res = rows(n, 1, WIDTH, dtype=dt, seed=10 + s), rows(n, 1, WIDTH, dtype=dt, seed=30 + s)
            seen, o = mix(x, res, lambda *a: gsa.gated_delta_step(*a, pool, state_indices=slots))
            for i in range(n):
                outs[i].append(o[i])
                parts[i].append([t[i] for t in seen])
        for i in range(n):
            whole = [torch.cat(ts) for ts in zip(*parts[i])]
            ro, rS = delta_tokens(*whole, DK ** -0.5)
            assert rel(torch.cat(outs[i]), ro) <= OUT[dtype]
            assert rel(pool[slots[i].item()], rS) <= STATE[dtype]
    assert (pool[[1, 3, 5]] == 7.0).all() and _lib.device_error() == 0


def test_tokens_in_a_graph():
    """A token's whole run captured once and replayed: the states go on as they do without it."""
    dt = torch.bfloat16
    w_in, unit, w_out = weights(dt)
    x, res = rows(3, 1, WIDTH, dtype=dt, seed=1), rows(3, 1, WIDTH, dtype=dt, seed=2)
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")

    def token(pool):
        n, h = gsa.rms_norm(x, w_in, residual=res)
        o = gsa.gated_delta_step(*inputs(n, unit, gsa.rms_norm), pool, state_indices=slots)
        return gsa.rms_norm_fp8(gsa.rms_norm(o, w_out).flatten(-2), w_in[:HV * DV])

    with torch.no_grad():
        a, b = (rows(3, HV, DK, DV, dtype=torch.float32, seed=4) for _ in range(2))
        token(b.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, scale = token(b)
        for seed in (7, 8, 9):
            x.copy_(rows(3, 1, WIDTH, dtype=dt, seed=seed))
            graph.replay()
            ey, escale = token(a)
            assert torch.equal(y.view(torch.uint8), ey.view(torch.uint8))
            assert torch.equal(scale, escale) and torch.equal(a, b)


def test_training_step():
    x, res = (rows(2, 100, WIDTH, dtype=torch.float32, seed=s) for s in (1, 2))
    dy, dh = rows(2, 100, HV, DV, dtype=torch.float32, seed=3), rows(
        2, 100, WIDTH, dtype=torch.float32, seed=4)

    def layer(norm, residual_norm, rule):
        def run(x, res, w_in, unit, w_out):
            n, h = residual_norm(x, w_in, res)
            return norm(rule(*inputs(n, unit, norm)), w_out), h
        return run

    mine = layer(gsa.rms_norm, lambda x, w, r: gsa.rms_norm(x, w, residual=r),
                 lambda *a: gsa.gated_delta_rule(*a)[0])

    def norm64(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    exact = layer(norm64, lambda x, w, r: (norm64(x + r, w), x + r),
                  lambda *a: delta_ref(*a, DK ** -0.5)[0])
    grads = []
    for run, to in ((mine, torch.float32), (exact, torch.float64)):
        leaves = [t.to(to).requires_grad_() for t in (x, res) + weights(torch.float32)]
        grads.append(torch.autograd.grad(run(*leaves), leaves, [dy.to(to), dh.to(to)]))
    for name, a, b in zip(("x", "residual", "w_in", "unit", "w_out"), *grads):
        assert rel(a, b) <= 2.4e-4, (name, rel(a, b))


def test_gradients_of_another_type():
    """Gradients of the outputs in fp32 for operators in bf16, and the other way round."""
    for dtype, other in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        x, res = rows(5, 96, dtype=dtype, seed=1), rows(5, 96, dtype=dtype, seed=2)
        w = weights(dtype)[2]
        up = rows(5, 96, dtype=torch.bfloat16, seed=3)  # the same values in either type
        leaves = [t.requires_grad_() for t in (x, w, res)]
        outs = gsa.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        a = torch.autograd.grad(outs, leaves, [up.to(other)] * 2, retain_graph=True)
        b = torch.autograd.grad(outs, leaves, [up.to(dtype)] * 2)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        mixed = [t.detach().requires_grad_() for t in inputs(
            rows(1, 70, WIDTH, dtype=dtype, seed=4), weights(dtype)[1], gsa.rms_norm)]
        o = gsa.gated_delta_rule(*mixed)[0]
        up = rows(1, 70, HV, DV, dtype=torch.bfloat16, seed=5)
        a = torch.autograd.grad(o, mixed, up.to(other), retain_graph=True)
        b = torch.autograd.grad(o, mixed, up.to(dtype))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
