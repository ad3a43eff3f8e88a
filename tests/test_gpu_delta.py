"""The gated delta rule against the token-by-token definition in 64 bits.

Tolerances (2-norm of the error over 2-norm of the result), derived before the first run:
* fp32: every output is a chain of sums of at most dk + 2 * 64 = 256 products, two such chains
  behind one another (S0 -> N -> o) and T = (I + L)^-1 on top, whose norm stays below 4 for unit
  keys: 4 * 2 * sqrt(256) roundings of 2^-24 = 8e-6.
* bf16 o: the output's own rounding (at most 2^-8, rms 2^-8 / sqrt(3)) and that of the factors
  P and N inside a chunk (two more of the same size): sqrt(3) * 2^-8 / sqrt(3) = 2^-8.
* bf16 gradients: up to five such roundings (two factors of each product, twice in a row, and
  the output's): sqrt(6) * 2^-8 / sqrt(3) < 2^-7.
* states and the initial state's gradient from bf16 inputs: factors held as pairs of bf16, off by
  2^-17 of their value; fewer than eight of them in a row, independent: sqrt(8) * 2^-17 < 2^-15.
"""
import math

import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib
from delta_ref import delta_ref, rel

pytestmark = pytest.mark.gpu

TOL = {("o", "fp32"): 8e-6, ("state", "fp32"): 8e-6, ("grad", "fp32"): 16e-6,
       ("o", "bf16"): 2.0 ** -8, ("state", "bf16"): 2.0 ** -15, ("grad", "bf16"): 2.0 ** -7}
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


def make(B, T, Hk, Hv, dk, dv, dtype="bf16", gates="fp32", seed=0, rate=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    q = torch.nn.functional.normalize(r(B, T, Hk, dk), dim=-1).to(DT[dtype])
    k = torch.nn.functional.normalize(r(B, T, Hk, dk), dim=-1).to(DT[dtype])
    v = r(B, T, Hv, dv).to(DT[dtype])
    g = (-rate * torch.nn.functional.softplus(r(B, T, Hv) - 2)).to(DT[gates])
    beta = torch.sigmoid(r(B, T, Hv)).to(DT[gates])
    return q, k, v, g, beta, r


def check_forward(args, dtype, scale=None, initial=None, bounds=None, cu=None):
    q, k, v, g, beta = args
    with torch.no_grad():
        o, S = gsa.gated_delta_rule(q, k, v, g, beta, scale=scale, initial_state=initial,
                                    cu_seqlens=cu, output_final_state=True)
        ro, rS = delta_ref(q, k, v, g, beta, q.shape[-1] ** -0.5 if scale is None else scale,
                           initial, bounds)
    assert o.dtype == q.dtype and S.dtype == torch.float32
    assert o.shape == v.shape
    assert rel(o, ro) <= TOL["o", dtype], rel(o, ro)
    assert rel(S, rS) <= TOL["state", dtype], rel(S, rS)
    return o, S


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 17, 63, 64, 65, 128, 200])
def test_lengths(dtype, T):
    *a, r = make(2, T, 2, 2, 128, 128, dtype, "fp32", seed=T)
    check_forward(a, dtype, initial=0.5 * r(2, 2, 128, 128))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dims", [(1, 1, 8, 8), (1, 4, 64, 96), (2, 2, 72, 40), (2, 8, 128, 64),
                                  (3, 3, 32, 256), (1, 2, 104, 136), (2, 4, 16, 200)])
def test_head_layouts(dtype, dims):
    Hk, Hv, dk, dv = dims
    *a, r = make(2, 150, Hk, Hv, dk, dv, dtype, "bf16" if dtype == "bf16" else "fp32", seed=dk)
    check_forward(a, dtype, scale=0.3, initial=r(2, Hv, dk, dv))


@pytest.mark.parametrize("shape", [(1, 1024, 1, 1, 128, 128), (1, 1500, 1, 2, 64, 72),
                                   (2, 2111, 2, 2, 104, 200), (1, 3000, 2, 4, 128, 64)])
@pytest.mark.parametrize("start", [False, True])
def test_long_sequences_of_few_heads(shape, start):
    """Long enough to be cut into segments that run side by side: states, outputs, gradients."""
    B, T, Hk, Hv, dk, dv = shape
    *a, r = make(*shape, "bf16", "bf16", seed=T, rate=0.05)  # slow decays: the cuts matter
    S0 = 0.5 * r(B, Hv, dk, dv) if start else None
    check_forward(a, "bf16", initial=S0)
    if not start:
        return
    do, dS = r(B, T, Hv, dv).bfloat16(), r(B, Hv, dk, dv)
    got = grads_of(lambda *x: gsa.gated_delta_rule(*x[:5], initial_state=x[5],
                                                   output_final_state=True), a + [S0], [do, dS])
    want = grads_of(lambda *x: delta_ref(*x[:5], dk ** -0.5, x[5]),
                    [t.double() for t in a + [S0]], [do.double(), dS.double()])
    for name, x, y in zip(("q", "k", "v", "g", "beta", "S0"), got, want):
        tol = TOL["state", "bf16"] if name == "S0" else TOL["grad", "bf16"]
        assert rel(x, y) <= tol, (name, rel(x, y))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lens", [[5], [0, 64, 1, 0, 130, 63], [200, 3], [0, 0], [65, 65, 65]])
@pytest.mark.parametrize("pad", [(0, 0), (7, 70)])
def test_packed(dtype, lens, pad):
    T = sum(lens) + sum(pad)
    if T == 0:
        T = 1
    *a, r = make(1, T, 2, 4, 64, 64, dtype, "fp32", seed=len(lens) + T)
    cu = [pad[0]]
    for n in lens:
        cu.append(cu[-1] + n)
    bounds = list(zip(cu[:-1], cu[1:]))
    o, _ = check_forward(a, dtype, initial=r(len(lens), 4, 64, 64), bounds=bounds,
                         cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    assert not o[0, :cu[0]].any() and not o[0, cu[-1]:].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_packed_neighbours_do_not_meet(dtype):
    """NaN and infinities in one sequence, or in rows of none, reach no other sequence."""
    *a, _ = make(1, 200, 1, 2, 64, 64, dtype, seed=5)
    cu = torch.tensor([3, 70, 133, 190], dtype=torch.int32, device="cuda")
    clean, S = gsa.gated_delta_rule(*a, cu_seqlens=cu, output_final_state=True)
    for t in a:
        t[:, :3] = math.nan
        t[:, 70:133] = math.inf
        t[:, 190:] = math.nan
    o, S2 = gsa.gated_delta_rule(*a, cu_seqlens=cu, output_final_state=True)
    for b, e in ((3, 70), (133, 190)):
        assert torch.equal(o[:, b:e], clean[:, b:e])
    assert torch.equal(S[[0, 2]], S2[[0, 2]])
    assert not o[0, :3].any() and not o[0, 190:].any()


def test_many_sequences():
    """More sequences than the table kernel has threads, most of them empty."""
    lens = [(3 * i) % 7 if i % 5 == 0 else 0 for i in range(2500)]
    T = sum(lens)
    *a, _ = make(1, T, 1, 1, 16, 16, "fp32", seed=2)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    o, S = gsa.gated_delta_rule(*a, cu_seqlens=cu, output_final_state=True)
    at = 0
    for n, ln in enumerate(lens):
        if ln:
            ro, rS = delta_ref(*(t[:, at:at + ln] for t in a), 0.25)
            assert rel(o[:, at:at + ln], ro) <= 8e-6 and rel(S[n], rS[0]) <= 8e-6
            at += ln
        else:
            assert not S[n].any()
    assert _lib.device_error() == 0


def test_bad_cu_seqlens_is_cut_and_reported():
    *a, _ = make(1, 100, 1, 1, 32, 32, "bf16", seed=3)
    cu = torch.tensor([10, 60, 40, 400], dtype=torch.int32, device="cuda")
    o, S = gsa.gated_delta_rule(*a, cu_seqlens=cu, output_final_state=True)
    assert _lib.device_error() == _lib.load().gsa_rms_norm(
        None, 0, None, 0, None, 0, 0.0, 0, -1, 1, None, 0, None, 0, None, None)  # INVALID_ARG
    with torch.no_grad():
        ro, rS = delta_ref(*a, 32 ** -0.5, bounds=[(10, 60), (60, 60), (60, 100)])
    assert rel(o, ro) <= TOL["o", "bf16"] and rel(S, rS) <= TOL["state", "bf16"]
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides(dtype):
    """Views of one projection's columns, heads in front of tokens, unaligned rows, expanded
    gates: the same results as contiguous copies."""
    B, T, H, d = 2, 77, 2, 64
    *a, r = make(B, T, H, H, d, d, dtype, "fp32", seed=9)
    want, wS = gsa.gated_delta_rule(*a, output_final_state=True)
    q, k, v, g, beta = a
    wide = torch.cat([x.flatten(2) for x in (q, k, v)], -1)
    views = [wide[..., i * H * d:(i + 1) * H * d].unflatten(-1, (H, d)) for i in range(3)]
    got, gS = gsa.gated_delta_rule(*views, g, beta, output_final_state=True)
    assert torch.equal(got, want) and torch.equal(gS, wS)
    swap = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, g, beta)]
    got, gS = gsa.gated_delta_rule(*swap, output_final_state=True)
    assert torch.equal(got, want) and torch.equal(gS, wS)
    odd = []
    for x in (q, k, v):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:]
        odd.append(flat.view(x.shape).copy_(x))
    got, gS = gsa.gated_delta_rule(*odd, g, beta, output_final_state=True)
    assert torch.equal(got, want) and torch.equal(gS, wS)
    ge, be = g[:, :1, :1].expand(B, T, H), beta[:, :, :1].expand(B, T, H)
    got = gsa.gated_delta_rule(q, k, v, ge, be)[0]
    assert torch.equal(got, gsa.gated_delta_rule(q, k, v, ge.contiguous(), be.contiguous())[0])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gates_at_their_ends(dtype):
    """Decay -inf wipes the state, far sums keep the neighbours' decays, beta 0 writes nothing."""
    *a, r = make(1, 140, 1, 2, 64, 64, dtype, "fp32", seed=4)
    q, k, v, g, beta = a
    g[:, 10] = -math.inf
    g[:, 11] = -math.inf
    g[:, 30:34] = -300.0
    g[:, 90] = -1e30
    beta[:, 50:70] = 0
    beta[:, 100:] = 1
    g[:, 120:] = 0
    check_forward(a, dtype, initial=r(1, 2, 64, 64))
    g[:, :64] = -math.inf  # every token of a chunk
    check_forward(a, dtype, initial=r(1, 2, 64, 64))


def grads_of(fn, leaves, outs_grad):
    leaves = [t.detach().requires_grad_() for t in leaves]
    outs = fn(*leaves)
    return torch.autograd.grad(outs, leaves, outs_grad, materialize_grads=True)


@pytest.mark.parametrize("dtype,gates", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("shape", [(2, 130, 2, 2, 128, 128), (1, 64, 1, 4, 64, 96),
                                   (1, 1, 2, 2, 32, 40), (2, 75, 2, 4, 104, 200)])
def test_gradients(dtype, gates, shape):
    B, T, Hk, Hv, dk, dv = shape
    *a, r = make(*shape, dtype, gates, seed=T)
    S0, do, dS = r(B, Hv, dk, dv), r(B, T, Hv, dv).to(DT[dtype]), r(B, Hv, dk, dv)
    got = grads_of(lambda *x: gsa.gated_delta_rule(*x[:5], initial_state=x[5],
                                                   output_final_state=True), a + [S0], [do, dS])
    want = grads_of(lambda *x: delta_ref(*x[:5], dk ** -0.5, x[5]),
                    [t.double() for t in a + [S0]], [do.double(), dS.double()])
    for name, x, y, like in zip(("q", "k", "v", "g", "beta", "S0"), got, want, a + [S0]):
        assert x.dtype == like.dtype and x.shape == like.shape
        tol = TOL["state", dtype] if name == "S0" else TOL["grad", dtype]
        assert rel(x, y) <= tol, (name, rel(x, y))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gradients_packed(dtype):
    lens, front, behind = [0, 70, 1, 64], 5, 9
    T = sum(lens) + front + behind
    *a, r = make(1, T, 1, 2, 64, 64, dtype, dtype, seed=8)
    cu = [front]
    for n in lens:
        cu.append(cu[-1] + n)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
    S0, do, dS = r(4, 2, 64, 64), r(1, T, 2, 64).to(DT[dtype]), r(4, 2, 64, 64)
    got = grads_of(lambda *x: gsa.gated_delta_rule(*x[:5], initial_state=x[5], cu_seqlens=cut,
                                                   output_final_state=True), a + [S0], [do, dS])
    want = grads_of(lambda *x: delta_ref(*x[:5], 0.125, x[5], list(zip(cu[:-1], cu[1:]))),
                    [t.double() for t in a + [S0]], [do.double(), dS.double()])
    for name, x, y in zip(("q", "k", "v", "g", "beta", "S0"), got, want):
        tol = TOL["state", dtype] if name == "S0" else TOL["grad", dtype]
        assert rel(x, y) <= tol, (name, rel(x, y))
        if name != "S0":
            assert not x[0, :front].any() and not x[0, T - behind:].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gradients_with_only_one_output_used(dtype):
    *a, r = make(1, 70, 2, 2, 64, 64, dtype, dtype, seed=12)
    do, dS = r(1, 70, 2, 64).to(DT[dtype]), r(1, 2, 64, 64)
    for pick, up in ((0, do), (1, dS)):
        got = grads_of(lambda *x: gsa.gated_delta_rule(*x, output_final_state=True)[pick], a, up)
        want = grads_of(lambda *x: delta_ref(*x, 0.125)[pick], [t.double() for t in a],
                        up.double())
        for name, x, y in zip(("q", "k", "v", "g", "beta"), got, want):
            if not y.any():
                assert not x.any()  # the last state does not depend on the queries
            else:
                assert rel(x, y) <= TOL["grad", dtype], (name, rel(x, y))


def test_gradients_against_differences():
    """fp32, central differences of a step of 2^-7 along a random direction of every input: the
    truncation is h^2 / 6 of the third derivative, about 1e-5 of the slope at these sizes, the
    outputs' own error (8e-6 of a sum near 1) over 2h about 5e-4 of it."""
    *a, r = make(1, 70, 1, 2, 32, 32, "fp32", seed=21)
    S0, wo, wS = r(1, 2, 32, 32), r(1, 70, 2, 32), r(1, 2, 32, 32)
    leaves = a + [S0]

    def f(*x):
        o, S = gsa.gated_delta_rule(*x[:5], initial_state=x[5], output_final_state=True)
        return (o.double() * wo).sum() + (S.double() * wS).sum()

    got = torch.autograd.grad(f(*[t.requires_grad_() for t in leaves]), leaves)
    with torch.no_grad():
        for i, (x, gx) in enumerate(zip(leaves, got)):
            d = torch.randn(x.shape, generator=torch.Generator("cuda").manual_seed(i),
                            device="cuda")
            d = d / d.norm() * min(1.0, x.norm().item())
            h = 2.0 ** -7
            args = lambda s: [t + s * h * d if j == i else t for j, t in enumerate(leaves)]  # noqa
            slope = ((f(*args(1)) - f(*args(-1))) / (2 * h)).item()
            want = (gx.double() * d).sum().item()
            size = gx.double().norm().item() * d.double().norm().item()
            assert abs(slope - want) <= 2e-3 * size, (i, slope, want, size)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_same_bits_every_time(dtype):
    *a, r = make(2, 150, 2, 4, 64, 64, dtype, dtype, seed=30)
    do, dS = r(2, 150, 4, 64).to(DT[dtype]), r(2, 4, 64, 64)
    run = lambda: grads_of(lambda *x: gsa.gated_delta_rule(*x, output_final_state=True), a, [do, dS])  # noqa
    for x, y in zip(run(), run()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,gates", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("dims", [(2, 2, 128, 128), (1, 4, 64, 96), (2, 4, 40, 200)])
def test_step(dtype, gates, T, dims):
    Hk, Hv, dk, dv = dims
    B = 9
    *a, r = make(B, T, Hk, Hv, dk, dv, dtype, gates, seed=T + dk)
    pool = r(14, Hv, dk, dv)
    before = pool.clone()
    idx = torch.tensor([3, -1, 0, 13, 7, -1, 2, 1, 12], dtype=torch.int32, device="cuda")
    o = gsa.gated_delta_step(*a, pool, state_indices=idx)
    live = [i for i in range(B) if idx[i] >= 0]
    rows = idx[live].long()
    ro, rS = delta_ref(*(t[live] for t in a), dk ** -0.5, before[rows])
    assert rel(o[live], ro) <= (8e-6 if dtype == "fp32" else 2.0 ** -8)
    assert rel(pool[rows], rS) <= 1e-6  # dk products and one update, fp32 throughout
    assert not o[idx < 0].any()
    rest = [i for i in range(14) if i not in rows.tolist()]
    assert torch.equal(pool[rest], before[rest])
    assert _lib.device_error() == 0


def test_step_follows_the_whole_sequence():
    """A prompt through gated_delta_rule, then token by token: the same as the whole at once."""
    *a, _ = make(3, 90, 2, 4, 128, 128, "bf16", "bf16", seed=40)
    o, S = gsa.gated_delta_rule(*a, output_final_state=True)
    head = [t[:, :65] for t in a]
    o1, state = gsa.gated_delta_rule(*head, output_final_state=True)
    outs = [o1]
    for t in range(65, 90):
        outs.append(gsa.gated_delta_step(*(x[:, t:t + 1] for x in a), state))
    assert rel(torch.cat(outs, 1), o) <= 2.0 ** -7  # both within 2^-8 of the exact one
    assert rel(state, S) <= 2.0 ** -14


def test_step_refuses_bad_and_repeated_slots_on_the_device():
    *a, r = make(6, 1, 1, 2, 64, 64, "bf16", seed=41)
    pool = r(4, 2, 64, 64)
    before = pool.clone()
    idx = torch.tensor([2, 4, 2, -5, 0, 2], dtype=torch.int32, device="cuda")
    o = gsa.gated_delta_step(*a, pool, state_indices=idx)
    assert _lib.device_error() == 1 and _lib.device_error() == 0
    assert o[[1, 2, 3, 5]].isnan().all()
    ro, rS = delta_ref(*(t[[0, 4]] for t in a), 0.125, before[[2, 0]])
    assert rel(o[[0, 4]], ro) <= 2.0 ** -8 and rel(pool[[2, 0]], rS) <= 1e-6
    assert torch.equal(pool[[1, 3]], before[[1, 3]])


def test_step_without_indices_and_with_infinite_decay():
    *a, r = make(2, 1, 2, 2, 32, 32, "fp32", seed=42)
    a[3][0] = -math.inf
    pool = r(5, 2, 32, 32)
    before = pool.clone()
    o = gsa.gated_delta_step(*a, pool)
    ro, rS = delta_ref(*a, 32 ** -0.5, before[:2])
    assert rel(o, ro) <= 8e-6 and rel(pool[:2], rS) <= 1e-6
    assert torch.equal(pool[2:], before[2:])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_empty_batches(dtype):
    for B, T in ((0, 5), (2, 0)):
        *a, r = make(B, T, 2, 2, 64, 64, dtype)
        S0 = r(B, 2, 64, 64)
        leaves = [t.requires_grad_() for t in a + [S0]]
        o, S = gsa.gated_delta_rule(*leaves[:5], initial_state=leaves[5], output_final_state=True)
        assert o.shape == (B, T, 2, 64) and torch.equal(S, S0)
        grads = torch.autograd.grad(S.sum(), leaves, allow_unused=True)
        assert torch.equal(grads[5], torch.ones_like(S0))
        with torch.no_grad():
            assert gsa.gated_delta_step(*a, S0.clone()).shape == (B, T, 2, 64)


def test_other_stream_and_graph():
    """Captured and replayed with new inputs, on a stream of its own; two graphs at once."""
    *a, _ = make(2, 100, 2, 2, 128, 128, "bf16", seed=50)
    *b, _ = make(2, 100, 2, 2, 128, 128, "bf16", seed=51)
    want = [gsa.gated_delta_rule(*x, output_final_state=True) for x in (a, b)]
    bufs = [[t.clone() for t in a] for _ in range(2)]
    graphs, outs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.no_grad():
        gsa.gated_delta_rule(*bufs[0])
        for x in bufs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(gsa.gated_delta_rule(*x, output_final_state=True))
            graphs.append(g)
    for t, n in zip(bufs[1], b):
        t.copy_(n)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for g, st in zip(graphs, (s, other)):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for (o, S), (wo, wS) in zip(outs, want):
        assert torch.equal(o, wo) and torch.equal(S, wS)


def test_training_step_in_a_graph():
    *a, r = make(1, 130, 2, 2, 64, 64, "bf16", "bf16", seed=52)
    do = r(1, 130, 2, 64).bfloat16()
    want = grads_of(lambda *x: gsa.gated_delta_rule(*x)[0], a, do)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        grads_of(lambda *x: gsa.gated_delta_rule(*x)[0], a, do)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = grads_of(lambda *x: gsa.gated_delta_rule(*x)[0], a, do)
        g.replay()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_inputs_changed_before_the_backward_are_noticed():
    *a, _ = make(1, 40, 1, 1, 32, 32, "fp32", seed=60)
    a[0].requires_grad_()
    v = a[2]
    o = gsa.gated_delta_rule(*a)[0]
    v.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()


def test_two_calls_at_once():
    """Forward and backward on two streams side by side: each the same bits as alone."""
    def run(leaves, do):
        o, S = gsa.gated_delta_rule(*leaves, output_final_state=True)
        return (o, S) + torch.autograd.grad(o, leaves, do)

    work = []
    for seed, (B, T, H) in enumerate([(1, 1500, 8), (4, 333, 16)]):
        *a, r = make(B, T, H, H, 128, 128, seed=seed)
        work.append(([t.requires_grad_() for t in a], r(B, T, H, 128).bfloat16()))
    alone = [run(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(5):
        got = []
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(run(*w))
        torch.cuda.synchronize()
        for x, y in zip(alone, got):
            assert all(torch.equal(p, q) for p, q in zip(x, y))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_states_off_the_grid_and_inputs_that_are_one_tensor(dtype):
    q, _, v, g, beta, r = make(2, 90, 2, 2, 64, 64, dtype, "fp32", seed=8)
    S0 = r(2 * 2 * 64 * 64 + 1)[1:].view(2, 2, 64, 64)
    check_forward((q, q, v, g, g.exp()), dtype, initial=S0)
    dS = r(2 * 2 * 64 * 64 + 1)[1:].view(2, 2, 64, 64)
    leaves = [t.requires_grad_() for t in (q, v, g)] + [S0.requires_grad_()]
    got = torch.autograd.grad(
        gsa.gated_delta_rule(q, q, v, g, beta, initial_state=S0, output_final_state=True)[1],
        leaves, dS)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(
        delta_ref(exact[0], exact[0], exact[1], exact[2], beta, 0.125, exact[3])[1], exact,
        dS.double())
    for name, x, y in zip(("q and k", "v", "g", "S0"), got, want):
        assert rel(x, y) <= (TOL["state", dtype] * 2 if name == "S0" else TOL["grad", dtype]), name


def test_offsets_past_32_bits():
    """More than 2^31 values a tensor.  The last 128 tokens start from a wiped state, so they, and
    their gradients, are those of a call on them alone."""
    T, H, d, tail = 2 ** 20 + 128, 16, 128, 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, do = (torch.randn(1, T, H, d, generator=gen, device="cuda", dtype=torch.bfloat16)
                   for _ in range(4))
    q.mul_(d ** -0.5), k.mul_(d ** -0.5)
    g = torch.full((1, T, H), -0.05, device="cuda")
    g[:, T - tail] = -math.inf
    beta = torch.full((1, T, H), 0.5, device="cuda")
    results = []
    for part in (slice(0, T), slice(T - tail, T)):
        leaves = [t[:, part].detach().requires_grad_() for t in (q, k, v, beta)]
        o, S = gsa.gated_delta_rule(*leaves[:3], g[:, part], leaves[3], output_final_state=True)
        grads = torch.autograd.grad(o, leaves, do[:, part])
        results.append([o[:, -tail:].clone(), S.clone()] + [t[:, -tail:].clone() for t in grads])
        del o, S, grads, leaves
    for name, a, b in zip(("o", "S", "q", "k", "v", "beta"), *results):
        assert torch.isfinite(a).all()
        assert rel(a, b) <= TOL["o" if name == "o" else "state" if name == "S" else "grad", "bf16"]
    del q, k, v, do, results
    torch.cuda.empty_cache()


def test_slots_past_32_bits():
    *a, r = make(3, 2, 16, 16, 128, 128, seed=11)
    pool = torch.zeros(8195, 16, 128, 128, device="cuda")  # 2^31 values and 3 states
    few = r(3, 16, 128, 128)
    slots = torch.tensor([8194, 0, 8192], dtype=torch.int32, device="cuda")
    pool[slots.long()] = few
    o = gsa.gated_delta_step(*a, pool, state_indices=slots)
    want = gsa.gated_delta_step(*a, few)
    assert torch.equal(o, want) and torch.equal(pool[slots.long()], few)
    assert not pool[1].any() and not pool[8193].any() and not pool[8191].any()
    del pool
    torch.cuda.empty_cache()
