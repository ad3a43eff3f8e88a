"""Calls of the gated delta rule and the norm at the borders of what their documentation allows.
Tolerances as derived in test_gpu_delta.py."""
import math

import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib
from delta_ref import delta_ref, norm_ref, rel
from test_gpu_delta import DT, TOL, check_forward, grads_of, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


def test_wide_indices_and_bounds_are_refused_on_the_device():
    """int64 slots and bounds that would come round to valid ones in 32 bits."""
    *a, r = make(6, 1, 1, 2, 64, 64, "bf16", seed=43)
    pool = r(4, 2, 64, 64)
    before = pool.clone()
    idx = torch.tensor([2, 2 ** 32 + 1, 2 ** 32 - 1, -2 ** 32, -1, 0], device="cuda")
    o = gsa.gated_delta_step(*a, pool, state_indices=idx)
    assert _lib.device_error() == 1 and _lib.device_error() == 0
    assert o[[1, 2, 3]].isnan().all() and not o[4].any()
    ro, rS = delta_ref(*(t[[0, 5]] for t in a), 0.125, before[[2, 0]])
    assert rel(o[[0, 5]], ro) <= 2.0 ** -8 and rel(pool[[2, 0]], rS) <= 1e-6
    assert torch.equal(pool[[1, 3]], before[[1, 3]])

    *a, _ = make(1, 100, 1, 1, 32, 32, "bf16", seed=44)
    for cu, bounds in (([0, 60, 2 ** 32 + 80], [(0, 60), (60, 100)]),
                       ([-2 ** 32 + 10, 60, 100], [(0, 60), (60, 100)]),
                       ([0, 2 ** 32 + 30, 100], [(0, 100), (100, 100)])):
        o, S = gsa.gated_delta_rule(*a, cu_seqlens=torch.tensor(cu, device="cuda"),
                                    output_final_state=True)
        assert _lib.device_error() == 1
        with torch.no_grad():
            ro, rS = delta_ref(*a, 32 ** -0.5, bounds=bounds)
        assert rel(o, ro) <= TOL["o", "bf16"] and rel(S, rS) <= TOL["state", "bf16"]


def check_gradients(a, S0, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    do = torch.randn(a[2].shape, generator=gen, device="cuda").to(DT[dtype])
    dS = torch.randn(S0.shape, generator=gen, device="cuda")
    got = grads_of(lambda *x: gsa.gated_delta_rule(*x[:5], initial_state=x[5],
                                                   output_final_state=True), [*a, S0], [do, dS])
    want = grads_of(lambda *x: delta_ref(*x[:5], a[0].shape[-1] ** -0.5, x[5]),
                    [t.double() for t in (*a, S0)], [do.double(), dS.double()])
    for name, x, y in zip(("q", "k", "v", "g", "beta", "S0"), got, want):
        assert torch.isfinite(x).all(), name
        if not y.any():  # wiped before it reaches anything
            assert not x.any(), name
            continue
        tol = TOL["state", dtype] if name == "S0" else TOL["grad", dtype]
        assert rel(x, y) <= tol, (name, rel(x, y))


@pytest.mark.parametrize("dtype,gates", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("whole", [False, True])
def test_gradients_with_gates_at_their_ends(dtype, gates, whole):
    """All six gradients where decays wipe the state: a product of an overflowing exponential and
    a zero must show nowhere, and nothing may flow back past a wiped state."""
    *a, r = make(1, 140, 1, 2, 64, 64, dtype, gates, seed=4)
    q, k, v, g, beta = a
    g[:, 10:12] = -math.inf
    g[:, 30:34] = -300.0
    g[:, 90] = -1e30
    beta[:, 50:70] = 0
    beta[:, 100:] = 1
    g[:, 120:] = 0
    if whole:
        g[:, :64] = -math.inf  # every token of a chunk
    check_gradients(a, r(1, 2, 64, 64), dtype, 14)


@pytest.mark.parametrize("shape", [(1, 2049, 1, 1, 128, 128), (1, 4097, 1, 2, 128, 128),
                                   (2, 2700, 1, 3, 72, 256), (1, 2100, 4, 16, 64, 128)])
@pytest.mark.parametrize("wiped", [False, True])
def test_segments(shape, wiped):
    """Sequences that are cut into 4 to 9 segments, the last one short, down to one token; with
    `wiped` the state is lost inside one segment and at the first token of another."""
    B, T, Hk, Hv, dk, dv = shape
    *a, r = make(*shape, "bf16", "fp32", seed=T, rate=0.02)
    if wiped:
        a[3][:, 700] = -math.inf
        a[3][:, 1152] = -math.inf
    check_forward(a, "bf16", initial=0.5 * r(B, Hv, dk, dv))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_norm_of_many_short_rows(dtype):
    """Queries and keys of a long prompt: a row a head."""
    x = torch.randn(4099, 16, 128, generator=torch.Generator("cuda").manual_seed(1),
                    device="cuda").to(DT[dtype])
    w = torch.full((128,), 128 ** -0.5, device="cuda").to(DT[dtype])
    dy = torch.randn(x.shape, generator=torch.Generator("cuda").manual_seed(2),
                     device="cuda").to(DT[dtype])
    leaf, weight = x.requires_grad_(), w.requires_grad_()
    y = gsa.rms_norm(leaf, weight)
    dx, dw = torch.autograd.grad(y, [leaf, weight], dy)
    with torch.no_grad():
        ry, _ = norm_ref(x, w, 1e-6)
        # tolerances of test_gpu_norm.py, element by element for y
        eps = 4e-6 + (2.0 ** -8 if dtype == "bf16" else 0)
        assert ((y.double() - ry).abs() <= eps * ry.abs()).all()
        h, p = x.double(), dy.double() * w.double()
        rstd = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        assert rel(dx, rstd * (p - h * rstd ** 2 * (p * h).mean(-1, keepdim=True))) <= eps
        want = (dy.double() * h * rstd).flatten(0, 1).sum(0)
        assert rel(dw, want) <= (1e-5 if dtype == "fp32" else 2.0 ** -8)


def test_step_is_noticed_and_tangents_are_refused():
    """On the device as on the host (test_operator_host.py)."""
    *a, r = make(2, 1, 1, 2, 64, 64, "bf16", seed=45)
    pool = r(4, 2, 64, 64)
    w = torch.ones_like(pool, requires_grad=True)
    loss = (pool * w).sum()
    gsa.gated_delta_step(*a, pool)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        q = torch.autograd.forward_ad.make_dual(a[0], torch.ones_like(a[0]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gsa.gated_delta_rule(q, *a[1:])
        with pytest.raises(RuntimeError, match="forward-mode"):
            gsa.rms_norm(q, torch.ones(64, device="cuda"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_packed_batch_without_rows(dtype):
    """T = 0 and N sequences of none: the states, and their gradients, pass through."""
    *a, r = make(1, 0, 2, 4, 64, 40, dtype, "fp32")
    S0 = r(3, 4, 64, 40)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (*a, S0)]
    o, S = gsa.gated_delta_rule(*leaves[:5], initial_state=S0, cu_seqlens=cu,
                                output_final_state=True)
    assert o.shape == (1, 0, 4, 40) and torch.equal(S, S0)
    dS = r(3, 4, 64, 40)
    grads = torch.autograd.grad(S, leaves, dS, allow_unused=True)
    assert torch.equal(grads[5], dS) and all(x.numel() == 0 for x in grads[:5])
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dims", [(1, 1, 8, 8), (1, 8, 16, 256), (2, 2, 128, 256), (1, 2, 104, 136),
                                  (3, 3, 72, 128)])
def test_gradients_of_head_layouts(dtype, dims):
    Hk, Hv, dk, dv = dims
    *a, r = make(2, 70, Hk, Hv, dk, dv, dtype, "fp32", seed=dk + dv)
    check_gradients(a, r(2, Hv, dk, dv), dtype, 15)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_backward_twice_and_through_saved_tensor_hooks(dtype):
    """What the forward pass kept is only read, and may come back at another address."""
    *a, r = make(1, 130, 1, 2, 64, 72, dtype, "fp32", seed=46)
    do = r(1, 130, 2, 72).to(DT[dtype])
    leaves = [t.requires_grad_() for t in a]
    o = gsa.gated_delta_rule(*leaves)[0]
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    second = torch.autograd.grad(o, leaves, do)
    with torch.autograd.graph.save_on_cpu():
        o = gsa.gated_delta_rule(*leaves)[0]
    third = torch.autograd.grad(o, leaves, do)
    for x, y, z in zip(first, second, third):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_step_of_many_rows_with_repeated_slots():
    """More rows than a block has threads, the repeated slots far apart: the first row has it."""
    B, slots = 300, 280
    *a, r = make(B, 1, 1, 1, 16, 32, "fp32", seed=47)
    pool = r(slots, 1, 16, 32)
    before = pool.clone()
    idx = torch.randperm(slots, generator=torch.Generator().manual_seed(3)).tolist()
    idx += [idx[0], idx[128], idx[255], -1] + idx[1:17]
    live = list(range(slots))
    o = gsa.gated_delta_step(*a, pool, state_indices=torch.tensor(idx, device="cuda"))
    assert _lib.device_error() == 1
    ro, rS = delta_ref(*(t[live] for t in a), 0.25, before[idx[:slots]])
    assert rel(o[live], ro) <= 8e-6 and rel(pool[idx[:slots]], rS) <= 1e-6
    assert o[[280, 281, 282]].isnan().all() and o[284:].isnan().all() and not o[283].any()
