"""The gated delta rule: whole sequences with gradients, and decoding steps.

The token mixer that the benchmark study sets beside gated sparse attention
(the reference's benchmark_models.ipynb:187-225 states it token by token).  Per
sequence and value head, with a state S [dk, dv]:

    S_t = exp(g_t) S_{t-1} + k_t u_t^T
    u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t)
    o_t = scale S_t^T q_t

``gated_delta_rule`` computes it chunk by chunk for training and prompts,
``gated_delta_step`` token by token against a pool of states for decoding.
Both run on the tensors' device and its current stream; there is no CPU path.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _DTYPES, _cuda, _dtype_code, _no_tangents, _on, _ptr, _raw_stream


def _rows_ok(t: torch.Tensor) -> torch.Tensor:
    """t [B, T, H, d] as the kernels read it: unit inner stride; in bf16 rows on 16 bytes and no
    dimension expanded.  Copied where it is not."""
    b, r, h, c = t.stride()
    if t.dtype is torch.bfloat16:
        if c == 1 and b > 0 and r > 0 and h > 0 and (b | r | h) % 8 == 0 and t.data_ptr() % 16 == 0:
            return t
        steps = [x for x, n in zip((b, r, h), t.shape) if n > 1]
        bad = t.data_ptr() % 16 or any(x % 8 or x <= 0 for x in steps)
    else:
        bad = False
    if t.numel() and (bad or (c != 1 and t.shape[3] > 1)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _gates_ok(t: torch.Tensor) -> torch.Tensor:
    if t.numel() and t.shape[2] > 1 and t.stride(2) != 1:
        return t.contiguous()
    return t


def _int32(t: torch.Tensor, least: int) -> torch.Tensor:
    """Whole numbers as contiguous int32.  What int32 does not hold becomes ``least`` or 2^31 - 1,
    which the kernels refuse as they would the number itself: no pool has 2^31 states (the smallest
    is 256 bytes) and no call so many tokens."""
    if t.dtype is not torch.int32:
        t = t.clamp(least, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _check(q, k, v, g, beta, *others) -> None:
    _no_tangents(q, k, v, g, beta, *others)
    if not q.is_cuda:
        _cuda(q, k, v, g, beta, *others)
    device = q.get_device()
    for t in (k, v, g, beta, *others):
        if t is not None and t.get_device() != device:
            _cuda(q, k, v, g, beta, *others)
            raise ValueError("all tensors must be on one device")
    q_shape, v_shape, g_shape = q.shape, v.shape, g.shape
    for name, shape in (("q", q_shape), ("v", v_shape)):
        if len(shape) != 4:
            raise ValueError(f"{name}: expected 4 dims, got {tuple(shape)}")
    dtype, gates = q.dtype, g.dtype
    if dtype not in _DTYPES or gates not in _DTYPES:
        _dtype_code(q), _dtype_code(g)
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must share a dtype")
    if beta.dtype is not gates:
        raise ValueError("g and beta must share a dtype")
    B, T, Hk, dk = q_shape
    vB, vT, Hv, dv = v_shape
    if k.shape != q_shape:
        raise ValueError(f"k must be [{B}, {T}, {Hk}, {dk}], got {tuple(k.shape)}")
    if vB != B or vT != T or Hk == 0 or Hv == 0 or Hv % Hk:
        raise ValueError(f"v must be [{B}, {T}, Hv, dv] with Hv a multiple of {Hk}, got "
                         f"{tuple(v_shape)}")
    if g_shape != (B, T, Hv) or beta.shape != g_shape:
        raise ValueError(f"g and beta must be [{B}, {T}, {Hv}], got {tuple(g_shape)} and "
                         f"{tuple(beta.shape)}")
    if dk % 8 or dv % 8 or not 0 < dk <= 128 or not 0 < dv <= 256:
        raise ValueError(f"dk and dv must be multiples of 8, dk <= 128 and dv <= 256, got "
                         f"{dk} and {dv}")


def _args(q, k, v, g, beta, scale, N, cu, initial) -> bytes:
    """gsa_delta_t."""
    B, T, Hk, dk = q.shape
    _, _, Hv, dv = v.shape
    q0, q1, q2, _ = q.stride()
    k0, k1, k2, _ = k.stride()
    v0, v1, v2, _ = v.stride()
    g0, g1, _ = g.stride()
    b0, b1, _ = beta.stride()
    return _lib.DELTA_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
        q0, q1, q2, k0, k1, k2, v0, v1, v2, g0, g1, b0, b1,
        0 if cu is None else cu.data_ptr(), 0 if initial is None else initial.data_ptr(),
        _DTYPES[q.dtype], _DTYPES[g.dtype], scale, B, T, Hk, Hv, dk, dv, N)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(
        t.shape, dtype=t.dtype, device=t.device)


def _workspace(a: bytes, use: int, device) -> torch.Tensor:
    need = int(_lib.load().gsa_delta_rule_workspace_size(a, use))
    if need < 0:
        raise RuntimeError(f"gsa_delta_rule_workspace_size failed: {_lib.last_error()}")
    return torch.empty(need, dtype=torch.uint8, device=device)


def _forward(q, k, v, g, beta, initial, cu, scale, N, want_final, use):
    B, T, _, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    a = _args(q, k, v, g, beta, scale, N, cu, initial)
    ws = _workspace(a, use, q.device)
    o = _like(v)
    final = (torch.empty(N, Hv, dk, dv, dtype=torch.float32, device=q.device) if want_final
             else None)
    rc = _lib.load().gsa_delta_rule_forward(
        a, o.data_ptr(), _ptr(final), use, ws.data_ptr(), ws.numel(),
        _raw_stream(q.device.index))
    _lib.check(rc, "gsa_delta_rule_forward")
    return o, final, ws


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial, cu, scale, N, want_final):
        with _on(q.device):
            o, final, ws = _forward(q, k, v, g, beta, initial, cu, scale, N, want_final,
                                    _lib.GSA_DELTA_TRAINING)
        ctx.save_for_backward(q, k, v, g, beta, cu, ws)
        ctx.scale, ctx.N, ctx.has_initial = scale, N, initial is not None
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dfinal):
        q, k, v, g, beta, cu, ws = ctx.saved_tensors
        if do is not None:
            do = do.to(q.dtype).contiguous()
            if do.data_ptr() % 16:
                do = do.clone()
        if dfinal is not None:
            dfinal = dfinal.float().contiguous()
        with _on(q.device):
            a = _args(q, k, v, g, beta, ctx.scale, ctx.N, cu, None)
            scratch = _workspace(a, _lib.GSA_DELTA_BACKWARD, q.device)
            dq, dk, dv, dg, dbeta = _like(q), _like(k), _like(v), _like(g), _like(beta)
            dinitial = (torch.empty(ctx.N, v.shape[2], q.shape[3], v.shape[3],
                                    dtype=torch.float32, device=q.device)
                        if ctx.has_initial and ctx.needs_input_grad[5] else None)
            rc = _lib.load().gsa_delta_rule_backward(
                a, _ptr(do), _ptr(dfinal), ws.data_ptr(), ws.numel(),
                scratch.data_ptr(), scratch.numel(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                dg.data_ptr(), dbeta.data_ptr(), _ptr(dinitial),
                _raw_stream(q.device.index))
        _lib.check(rc, "gsa_delta_rule_backward")
        return dq, dk, dv, dg, dbeta, dinitial, None, None, None, None


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                     beta: torch.Tensor, scale: float | None = None,
                     initial_state: torch.Tensor | None = None,
                     cu_seqlens: torch.Tensor | None = None, output_final_state: bool = False):
    """The gated delta rule over whole sequences, with gradients.

    q, k [B, T, Hk, dk] and v [B, T, Hv, dv] (bf16 or fp32), Hv a multiple of Hk
    (value head h reads key head h // (Hv // Hk)), dk <= 128 and dv <= 256,
    multiples of 8; g (log decay, at most 0) and beta [B, T, Hv], both bf16 or
    both fp32; scale defaults to dk ** -0.5.  ``initial_state`` [N, Hv, dk, dv]
    fp32 (default zeros).  With ``cu_seqlens`` (int32 or int64 [N + 1] on the device, as
    ``[0, n_0, n_0 + n_1, ...]``) B is 1 and the N sequences lie one behind the
    other; rows of no sequence come out, and in the gradients, as zeros.

    Returns (o [B, T, Hv, dv] in q's dtype, final state [N, Hv, dk, dv] fp32 or
    None).  Differentiable once, in reverse mode, in q, k, v, g, beta and the initial state; the
    gradients have the inputs' dtypes and add up in a fixed order.  States, decays
    and sums are held in fp32.  From bf16 inputs the products take pairs of bf16 for
    the state, which comes out within about 5e-6 of exact, and single ones for the
    gradients: dq and dk are within about 3e-3, dg and dbeta within about 2e-3 where
    the gates, and so they, are fp32.  fp32 inputs keep fp32 throughout.
    Keys are expected near unit length (``rms_norm`` with weight dk ** -0.5 makes
    them), values finite."""
    _check(q, k, v, g, beta, initial_state, cu_seqlens)
    B, T, _, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    N = B
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (
                torch.int32, torch.int64):
            raise ValueError("cu_seqlens must be int32 or int64 [N + 1] with N >= 1")
        if B != 1:
            raise ValueError("cu_seqlens needs a batch of 1")
        cu_seqlens = _int32(cu_seqlens, -1)
        N = cu_seqlens.numel() - 1
    if initial_state is not None:
        if initial_state.shape != (N, Hv, dk, dv) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be float32 [{N}, {Hv}, {dk}, {dv}]")
        initial_state = initial_state.contiguous()
    scale = dk ** -0.5 if scale is None else float(scale)
    q, k, v, g, beta = _rows_ok(q), _rows_ok(k), _rows_ok(v), _gates_ok(g), _gates_ok(beta)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state)):
        return _GatedDeltaRule.apply(q, k, v, g, beta, initial_state, cu_seqlens, scale, N,
                                     output_final_state)
    with _on(q.device):
        return _forward(q, k, v, g, beta, initial_state, cu_seqlens, scale, N,
                        output_final_state, _lib.GSA_DELTA_INFERENCE)[:2]


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                     beta: torch.Tensor, state: torch.Tensor, scale: float | None = None,
                     state_indices: torch.Tensor | None = None) -> torch.Tensor:
    """One or a few tokens of each of B sequences, against states updated in place.

    Inputs as ``gated_delta_rule`` with T the tokens of the step (usually 1).
    ``state`` [slots, Hv, dk, dv] fp32, contiguous: sequence b has the slot
    ``state_indices[b]`` (int32 or int64 [B] on the device; default b); -1 marks an empty
    row of the batch, whose output is zero.  An index outside [-1, slots) or one
    that an earlier row has already is refused on the device: that row comes out
    as NaN, no state changes for it, and ``_lib.device_error()`` reports it.
    Autograd counts the call as a change of ``state`` in place.
    Returns o [B, T, Hv, dv].  No gradients."""
    _check(q, k, v, g, beta, state, state_indices)
    B, T, _, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or g.requires_grad or beta.requires_grad
                                    or state.requires_grad):
        raise RuntimeError("gated_delta_step has no gradients; use gated_delta_rule")
    slots = state.shape[0] if state.dim() == 4 else -1
    if (state.shape != (slots, Hv, dk, dv) or state.dtype is not torch.float32
            or not state.is_contiguous() or state.data_ptr() % 16):
        raise ValueError(f"state must be contiguous float32 [slots, {Hv}, {dk}, {dv}], 16-byte "
                         "aligned")
    if state_indices is not None:
        if state_indices.shape != (B,) or state_indices.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"state_indices must be int32 or int64 [{B}]")
        if state_indices.dtype is not torch.int32 or not state_indices.is_contiguous():
            state_indices = _int32(state_indices, -2)
    elif slots < B:
        raise ValueError(f"{B} rows need as many states, got {slots}")
    scale = dk ** -0.5 if scale is None else float(scale)
    q, k, v, g, beta = _rows_ok(q), _rows_ok(k), _rows_ok(v), _gates_ok(g), _gates_ok(beta)
    with _on(q.device):
        a = _args(q, k, v, g, beta, scale, B, None, None)
        o = _like(v)
        rc = _lib.load().gsa_delta_step(
            a, state.data_ptr(), slots, _ptr(state_indices), o.data_ptr(),
            _raw_stream(q.device.index))
    if rc:
        _lib.check(rc, "gsa_delta_step")
    if not state.is_inference():
        increment_version(state)  # graphs that saved it notice
    return o
