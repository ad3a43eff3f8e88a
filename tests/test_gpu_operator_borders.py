"""Calls of the gated delta rule and the norm at the borders of what their documentation allows.
Tolerances as derived in test_gpu_delta.py."""
import pytest
import torch

import gsa_gdn_benchmarkstudy_b200 as gsa
from gsa_gdn_benchmarkstudy_b200 import _lib
from delta_ref import delta_ref, rel
from test_gpu_delta import TOL, make

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
