"""What the gated delta rule's and the norm's entry points do on the host: the arguments that
reach the library, and what autograd is told.  CPU tensors against a stand-in for the library."""
import contextlib
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib, delta, norm


@pytest.fixture(autouse=True)
def _gradients():
    """Other test modules switch gradients off for the whole process."""
    with torch.enable_grad():
        yield


class Library:
    """Takes every call as a success and keeps the int32 values that it was handed."""

    def __init__(self):
        self.indices = self.cu_seqlens = None

    def gsa_delta_rule_workspace_size(self, a, use):
        return 256

    def gsa_delta_rule_forward(self, a, *rest):
        p = _lib.DeltaArgs.from_buffer_copy(a)
        if p.cu_seqlens:
            self.cu_seqlens = list((ctypes.c_int32 * (p.N + 1)).from_address(p.cu_seqlens))
        return 0

    def gsa_delta_step(self, a, state, slots, indices, o, stream):
        p = _lib.DeltaArgs.from_buffer_copy(a)
        if indices:
            self.indices = list((ctypes.c_int32 * p.B).from_address(indices))
        return 0


@pytest.fixture
def library(monkeypatch):
    fake = Library()
    monkeypatch.setattr(_lib, "load", lambda path=None: fake)
    for m in (delta, norm):
        monkeypatch.setattr(m, "_cuda", lambda *t: None)
        monkeypatch.setattr(m, "_on", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(m, "_raw_stream", lambda index: 0)
    return fake


def inputs(B=1, T=4, Hk=1, Hv=2, dk=16, dv=16):
    return (torch.zeros(B, T, Hk, dk), torch.zeros(B, T, Hk, dk), torch.zeros(B, T, Hv, dv),
            torch.zeros(B, T, Hv), torch.zeros(B, T, Hv))


def test_wide_state_indices_stay_outside_the_pool(library):
    """What int32 cannot hold must not come round to a slot, or to -1, an empty row."""
    slots = 5
    good = [3, -1, 0, 4]
    bad = [2 ** 32 + 2, 2 ** 32 - 1, 2 ** 31, -2 ** 32 + 1, -2 ** 31 - 1, 2 ** 63 - 1, -2 ** 63, -2]
    idx = torch.tensor([x for pair in zip(good * 2, bad) for x in pair])
    for t in (idx, torch.stack([idx, idx], 1)[:, 0]):
        gsa.gated_delta_step(*inputs(B=len(idx), T=1), torch.zeros(slots, 2, 16, 16),
                             state_indices=t)
        assert library.indices[0::2] == good * 2
        assert all(x < -1 or x >= slots for x in library.indices[1::2])
    narrow = torch.tensor(good, dtype=torch.int32)
    gsa.gated_delta_step(*inputs(B=4, T=1), torch.zeros(slots, 2, 16, 16), state_indices=narrow)
    assert library.indices == good


@pytest.mark.parametrize("cu", [[0, 2 ** 32 + 60, 100], [0, 60, 2 ** 32 + 100], [2 ** 32, 60, 100],
                                [-2 ** 32, 60, 100], [0, 60, 2 ** 63 - 1], [-2 ** 63, 60, 100],
                                [0, 2 ** 33, 2 ** 32], [-2 ** 33, -2 ** 32, 100]])
def test_wide_cu_seqlens_stay_wrong(library, cu):
    """Bounds that int32 cannot hold still decrease or leave [0, T], which the device reports."""
    T = 100
    gsa.gated_delta_rule(*inputs(T=T), cu_seqlens=torch.tensor(cu))
    got = library.cu_seqlens
    assert [x for x, y in zip(got, cu) if 0 <= y <= T] == [y for y in cu if 0 <= y <= T]
    assert all(x < 0 or x > T for x, y in zip(got, cu) if not 0 <= y <= T)


def test_step_counts_as_a_change_of_the_state(library):
    """A graph that saved the states must notice that the step has overwritten them."""
    pool = torch.zeros(3, 2, 16, 16)
    w = torch.ones_like(pool, requires_grad=True)
    loss = (pool * w).sum()
    gsa.gated_delta_step(*inputs(T=1), pool)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    base = torch.zeros(2, 3, 2, 16, 16)  # a view's base and its other views share the count
    loss = (base[1] * w).sum()
    gsa.gated_delta_step(*inputs(T=1), base[0])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_step_in_inference_mode(library):
    """States made in inference mode carry no count."""
    with torch.inference_mode():
        pool = torch.zeros(3, 2, 16, 16)
        gsa.gated_delta_step(*inputs(T=1), pool)
    outside = torch.zeros(3, 2, 16, 16)
    with torch.inference_mode():
        gsa.gated_delta_step(*inputs(T=1), outside)
    gsa.gated_delta_step(*inputs(T=1), outside)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("at", range(6))
def test_forward_mode_derivatives_are_refused(library, grad, at):
    """A tangent must not be dropped, whether reverse mode is on or not."""
    from torch.autograd import forward_ad
    x = [*inputs(T=1), torch.zeros(1, 2, 16, 16)]
    rows = [torch.ones(4, 128), torch.ones(128), torch.ones(4, 128)]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x[at] = forward_ad.make_dual(x[at], torch.ones_like(x[at]))
        for call in (lambda: gsa.gated_delta_rule(*x[:5], initial_state=x[5]),
                     lambda: gsa.gated_delta_step(*x)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        if at < 3:
            rows[at] = forward_ad.make_dual(rows[at], torch.ones_like(rows[at]))
            for norm_of in (gsa.rms_norm, gsa.rms_norm_fp8):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    norm_of(rows[0], rows[1], residual=rows[2])
    with torch.no_grad(), forward_ad.dual_level():  # no tangents: an ordinary call
        gsa.gated_delta_step(*inputs(T=1), torch.zeros(1, 2, 16, 16))


def test_function_transforms_are_refused(library):
    x = [*inputs(T=1), torch.zeros(1, 2, 16, 16)]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: gsa.gated_delta_rule(q, *x[1:5])[0], (x[0],), (x[0],))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: gsa.rms_norm(v, torch.ones(16)), (x[2],), (x[2],))


def test_import_without_cuda_in_torch():
    """A torch built without CUDA has no raw streams; the package's host parts still import."""
    code = ("import torch\n"
            "if hasattr(torch._C, '_cuda_getCurrentRawStream'):\n"
            "    del torch._C._cuda_getCurrentRawStream\n"
            "import gsa_gdn_benchmarkstudy_b200 as gsa\n"
            "try:\n"
            "    gsa.rms_norm(torch.zeros(2, 8), torch.zeros(8))\n"
            "except RuntimeError as e:\n"
            "    assert 'only on CUDA' in str(e)\n"
            "else:\n"
            "    raise SystemExit('no error')\n")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent)
    assert got.returncode == 0, got.stderr
