"""What the gated delta rule and the RMS norm refuse, on the host and before any device work."""
import ctypes

import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib, delta, norm
from gsa_gdn_benchmarkstudy_b200.build import build


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def args(**over):
    a = _lib.DeltaArgs()
    a.B, a.T, a.Hk, a.Hv, a.dk, a.dv, a.N = 2, 100, 2, 4, 64, 96, 2
    a.dtype, a.gate_dtype, a.scale = 0, 1, 1.0
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), 1), (dict(T=-1), 1), (dict(Hk=0), 1), (dict(Hv=3), 1), (dict(dk=0), 1),
    (dict(dtype=2), 3), (dict(gate_dtype=7), 3), (dict(dk=136), 3), (dict(dk=60), 3),
    (dict(dv=264), 3), (dict(dv=12), 3), (dict(N=3), 1), (dict(cu_seqlens=16), 1),
    (dict(cu_seqlens=16, B=1, N=0), 1), (dict(Hk=70000, Hv=70000), 3),
    (dict(T=2 ** 31 - 1), 3)])
def test_delta_sizes(lib, over, code):
    a = args(**over)
    assert lib.gsa_delta_rule_workspace_size(ctypes.byref(a), 0) == -1
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), None, None, 0, None, 0, None) == code
    assert lib.gsa_delta_rule_backward(ctypes.byref(a), None, None, None, 0, None, 0, None, None,
                                       None, None, None, None, None) == code


def test_delta_null_alignment_and_workspace(lib):
    assert lib.gsa_delta_rule_forward(None, None, None, 0, None, 0, None) == 1
    a = args()
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), None, None, 0, None, 0, None) == 1
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), None, None, 2, None, 0, None) == 1
    assert lib.gsa_delta_rule_workspace_size(ctypes.byref(a), 9) == -1
    sizes = [lib.gsa_delta_rule_workspace_size(ctypes.byref(a), u) for u in (0, 1, 2)]
    assert 0 < sizes[0] < sizes[1] and sizes[2] > 0
    for n in ("q", "k", "v", "g", "beta"):
        setattr(a, n, 4096)
    a.q_stride[1] = 4
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, 4096, 1 << 40, None) == 2
    a.q_stride[1] = 0  # an expanded dimension
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, 4096, 1 << 40, None) == 2
    for n in ("q", "k", "v"):
        getattr(a, n + "_stride")[:] = [1 << 20, 1 << 10, 128]
    a.k = 4098
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, 4096, 1 << 40, None) == 2
    a.k = 4096
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, None, 1 << 40, None) == 1
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, 4096, sizes[0] - 1, None) == 1
    assert lib.gsa_delta_rule_forward(ctypes.byref(a), 4096, None, 0, 4100, 1 << 40, None) == 2
    assert lib.gsa_delta_rule_backward(ctypes.byref(a), None, None, 4096, sizes[0], 4096, 1 << 40,
                                       4096, 4096, 4096, 4096, 4096, None, None) == 1
    # empty work is a success
    assert lib.gsa_delta_rule_forward(ctypes.byref(args(B=0, N=0)), None, None, 0, None, 0,
                                      None) == 0


def test_step_sizes(lib):
    a = args()
    assert lib.gsa_delta_step(ctypes.byref(a), None, -1, None, None, None) == 1
    assert lib.gsa_delta_step(ctypes.byref(a), 4096, 1, None, 4096, None) == 1  # two rows, one slot
    assert lib.gsa_delta_step(ctypes.byref(a), 4096, 2, None, 4096, None) == 1  # q is NULL
    assert lib.gsa_delta_step(ctypes.byref(args(T=0)), 4096, 2, None, 4096, None) == 0


def test_norm_sizes(lib):
    call = lib.gsa_rms_norm
    ok = dict(x=4096, xs=8, res=None, rs=0, w=4096, wd=0, eps=1e-6, d=0, rows=2, width=8, y=4096,
              ys=8, h=None, hs=0, rstd=None, st=None)
    for over, code in ((dict(rows=-1), 1), (dict(width=0), 1), (dict(width=32769), 3),
                       (dict(d=5), 3), (dict(wd=5), 3), (dict(x=None), 1), (dict(ys=7), 1),
                       (dict(res=4096, rs=8), 1), (dict(rows=2 ** 31), 3), (dict(rows=0), 0)):
        assert call(*(ok | over).values()) == code, over
    assert lib.gsa_rms_norm_fp8(4096, 8, None, 0, 4096, 0, 1e-6, 0, 2, 64, 4096, 64, 4096, 128,
                                None, 0, None) == 3
    assert lib.gsa_rms_norm_fp8(4096, 8, None, 0, 4096, 0, 1e-6, 0, 2, 64, 4096, 64, None, 0,
                                None, 0, None) == 1
    assert lib.gsa_rms_norm_backward_workspace_size(0, 64) == 0
    assert lib.gsa_rms_norm_backward(4096, 8, None, 0, 4096, 8, 4096, 0, 4096, 0, 2, 8, 4096, 8,
                                     4096, None, 0, None) == 1


def cpu(B=1, T=4, Hk=1, Hv=2, dk=16, dv=16, dtype=torch.float32, gates=torch.float32):
    return (torch.zeros(B, T, Hk, dk, dtype=dtype), torch.zeros(B, T, Hk, dk, dtype=dtype),
            torch.zeros(B, T, Hv, dv, dtype=dtype), torch.zeros(B, T, Hv, dtype=gates),
            torch.zeros(B, T, Hv, dtype=gates))


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="only on CUDA"):
        gsa.gated_delta_rule(*cpu())
    with pytest.raises(RuntimeError, match="only on CUDA"):
        gsa.gated_delta_step(*cpu(), torch.zeros(1, 2, 16, 16))
    for f in (gsa.rms_norm, gsa.rms_norm_fp8):
        with pytest.raises(RuntimeError, match="only on CUDA"):
            f(torch.zeros(2, 8), torch.zeros(8))


@pytest.fixture
def no_device_check(monkeypatch):
    """The checks that follow the device's, on CPU tensors."""
    for m in (delta, norm):
        monkeypatch.setattr(m, "_cuda", lambda *t: None)


def test_delta_shapes(no_device_check):
    q, k, v, g, b = cpu()
    f = gsa.gated_delta_rule
    for bad in ((q[0], k, v, g, b), (q, k[:, :2], v, g, b), (q, k, v[:, :2], g, b),
                (q, k, v, g[..., :1], b), (q, k, v, g, b[:, :1]), (q, k.bfloat16(), v, g, b),
                (q, k, v, g.bfloat16(), b), (q, k, v[..., :12], g, b),
                (q[..., :12], k[..., :12], v, g, b)):
        with pytest.raises(ValueError):
            f(*bad)
    two = cpu(Hk=2, Hv=3)
    with pytest.raises(ValueError, match="multiple of 2"):
        f(*two)
    with pytest.raises(RuntimeError, match="bfloat16 and float32"):
        f(*cpu(dtype=torch.float16))
    with pytest.raises(ValueError, match="dk <= 128"):
        f(*cpu(dk=136))
    with pytest.raises(ValueError, match="initial_state"):
        f(*cpu(), initial_state=torch.zeros(1, 2, 16, 8))
    with pytest.raises(ValueError, match="initial_state"):
        f(*cpu(), initial_state=torch.zeros(1, 2, 16, 16).bfloat16())
    with pytest.raises(ValueError, match="cu_seqlens must"):
        f(*cpu(), cu_seqlens=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="cu_seqlens must"):
        f(*cpu(), cu_seqlens=torch.zeros(3))
    with pytest.raises(ValueError, match="batch of 1"):
        f(*cpu(B=2), cu_seqlens=torch.zeros(3, dtype=torch.int32))


def test_step_shapes(no_device_check):
    f = gsa.gated_delta_step
    state = torch.zeros(2, 2, 16, 16)
    with pytest.raises(ValueError, match="state must"):
        f(*cpu(), state.bfloat16())
    with pytest.raises(ValueError, match="state must"):
        f(*cpu(), state.transpose(2, 3))
    with pytest.raises(ValueError, match="state must"):
        f(*cpu(), torch.zeros(2, 2, 16, 8))
    with pytest.raises(ValueError, match="as many states"):
        f(*cpu(B=3), state)
    with pytest.raises(ValueError, match="state_indices"):
        f(*cpu(), state, state_indices=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="state_indices"):
        f(*cpu(), state, state_indices=torch.zeros(1))
    q, *rest = cpu()
    with pytest.raises(RuntimeError, match="no gradients"):
        f(q.requires_grad_(), *rest, state)


def test_norm_shapes(no_device_check):
    x, w = torch.zeros(4, 8), torch.zeros(8)
    for f in (gsa.rms_norm, gsa.rms_norm_fp8):
        with pytest.raises(ValueError, match="weight"):
            f(x, torch.zeros(9))
        with pytest.raises(ValueError, match="residual"):
            f(x, w, residual=torch.zeros(4, 9))
        with pytest.raises(ValueError, match="residual"):
            f(x, w, residual=torch.zeros(4, 8).bfloat16())
        with pytest.raises(RuntimeError, match="bfloat16 and float32"):
            f(x.half(), w)
        with pytest.raises(ValueError, match="32768"):
            f(torch.zeros(1, 32769), torch.zeros(32769))
        with pytest.raises(ValueError, match="last dim"):
            f(torch.zeros(3, 0), torch.zeros(0))
    with pytest.raises(ValueError, match="group_size"):
        gsa.rms_norm_fp8(x, w, group_size=64)
    with pytest.raises(ValueError, match="multiple of 128"):
        gsa.rms_norm_fp8(x, w, group_size=128)
    with pytest.raises(RuntimeError, match="no gradients"):
        gsa.rms_norm_fp8(x.requires_grad_(), w)


# Addresses between two elements, which a kernel could only fault on: refused before any device
# work.  4096 stands for a good address; nothing reads it, because each call has one bad one.
def test_delta_addresses_between_elements(lib):
    for dtype, gates in ((0, 0), (0, 1), (1, 0), (1, 1)):
        def make(**over):
            a = args(dtype=dtype, gate_dtype=gates)
            for n in ("q", "k", "v"):
                setattr(a, n, 4096)
                getattr(a, n + "_stride")[:] = [1 << 20, 1 << 10, 128]
            a.g = a.beta = 4096
            for n, v in over.items():
                setattr(a, n, v)
            return a

        word, gate = (2 if dtype == 0 else 4), (2 if gates == 0 else 4)
        inputs = {"q": word, "k": word, "v": word, "g": gate, "beta": gate}

        def forward(a, o=4096, final=4096):
            return lib.gsa_delta_rule_forward(ctypes.byref(a), o, final, 0, 4096, 1 << 40, None)

        def backward(a, at=None):
            p = [4096] * 10
            if at is not None:
                p[at[0]] = at[1]
            dout, dfinal, dq, dk, dv, dg, dbeta, dinitial = p[:8]
            return lib.gsa_delta_rule_backward(
                ctypes.byref(a), dout, dfinal, 4096, 1 << 40, 4096, 1 << 40, dq, dk, dv, dg,
                dbeta, dinitial, None)

        def step(a, indices=4096, o=4096):
            return lib.gsa_delta_step(ctypes.byref(a), 4096, 9, indices, o, None)

        for name, size in inputs.items():
            bad = make(**{name: 4096 + size // 2})
            assert forward(bad) == 2 and backward(bad) == 2 and step(bad) == 2, name
        assert forward(make(initial_state=4098)) == 2
        assert forward(make(initial_state=4098, T=0)) == 2
        assert forward(make(cu_seqlens=4098, B=1)) == 2
        assert backward(make(cu_seqlens=4098, B=1)) == 2
        assert forward(make(), o=4096 + word // 2) == 2
        assert forward(make(), final=4098) == 2 and forward(make(T=0), final=4098) == 2
        for i, size in enumerate((word, 4, word, word, word, gate, gate, 4)):
            assert backward(make(), (i, 4096 + size // 2)) == 2, i
        assert backward(make(T=0), (1, 4098)) == 2 and backward(make(T=0), (7, 4098)) == 2
        assert step(make(), indices=4098) == 2 and step(make(), o=4096 + word // 2) == 2


def test_norm_addresses_between_elements(lib):
    for dtype, wdtype in ((0, 0), (0, 1), (1, 0), (1, 1)):
        word, weight = (2 if dtype == 0 else 4), (2 if wdtype == 0 else 4)

        def off(sizes, call):
            good = [4096] * len(sizes)
            for i, size in enumerate(sizes):
                if size > 1:
                    assert call(*(good[:i] + [4096 + size // 2] + good[i + 1:])) == 2, i

        off([word, word, weight, word, word, 4], lambda x, r, w, y, h, rstd: lib.gsa_rms_norm(
            x, 8, r, 8, w, wdtype, 1e-6, dtype, 2, 8, y, 8, h, 8, rstd, None))
        off([word, word, weight, 1, 4, word], lambda x, r, w, y, s, h: lib.gsa_rms_norm_fp8(
            x, 8, r, 8, w, wdtype, 1e-6, dtype, 2, 8, y, 8, s, 0, h, 8, None))
        off([word, word, word, weight, 4, word, weight],
            lambda dy, dh, h, w, rstd, dx, dw: lib.gsa_rms_norm_backward(
                dy, 8, dh, 8, h, 8, w, wdtype, rstd, dtype, 2, 8, dx, 8, dw, 4096, 1 << 40, None))
