"""Selective state-space scan, for training and for packed serving batches.

Per token t, channel d and state n, with the channel's group f = d // (D / F):

  dt        = softplus(delta[t, d] + delta_bias[d])      (softplus and bias optional)
  h[n]      = exp(dt A[d, n]) h[n] + dt u[t, d] B[t, f, n]
  y         = sum_n C[t, f, n] h[n] + skip[d] u[t, d]
  out[t, d] = y SiLU(gate[t, d])                          (skip, gate optional)

  selective_scan          packed sequences (cu_seqlens), zero initial states, with autograd
                          -> greta_ssm_scan_fwd / greta_ssm_scan_bwd
  packed_selective_scan   a serving batch with cache-slot states, prompts and
                          single tokens in any mix -> greta_ssm_scan_packed

u, delta, gate, B and C have one type (fp32, fp16, bf16) and may be column
views of wider projection outputs (contiguous innermost dimension, any row
stride); B and C are compact per group, [T, F, N], as this package's filters
are [T, W, D/G]. A, skip, delta_bias and the states are fp32, and so are all
sums. The reference has no state-space mixer; the conv ahead of the scan is
causal_conv.py.

There is no CPU fallback: non-CUDA tensors raise ValueError.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi
from .causal_conv import channel_rows, check_disjoint, packed_metadata, packed_out
from .dynamic_conv import _cu

MAX_STATES = 128
SAVE_EVERY = 8  # tokens per saved state


def _check(u, delta, A, B, C, skip, gate, delta_bias):
    """Shapes, types and devices of the operands ([T, D] rows); (T, D, N, F)."""
    T, D = u.shape
    _capi.dtype_code(u)
    if tuple(delta.shape) != (T, D):
        raise ValueError(f"delta shape {tuple(delta.shape)} must match u's {(T, D)}")
    if gate is not None and tuple(gate.shape) != (T, D):
        raise ValueError(f"gate shape {tuple(gate.shape)} must match u's {(T, D)}")
    if A.dim() != 2 or A.shape[0] != D:
        raise ValueError(f"A must be [{D}, N], got {tuple(A.shape)}")
    N = A.shape[1]
    if not 1 <= N <= MAX_STATES:
        raise ValueError(f"the number of states must be between 1 and {MAX_STATES}, got {N}")
    if B.dim() != 3 or B.shape[0] != T or B.shape[2] != N or B.shape[1] < 1 or D % B.shape[1] != 0:
        raise ValueError(f"B must be [{T}, F, {N}] with F dividing {D}, got {tuple(B.shape)}")
    if tuple(C.shape) != tuple(B.shape):
        raise ValueError(f"C shape {tuple(C.shape)} must match B's {tuple(B.shape)}")
    for name, t in (("skip", skip), ("delta_bias", delta_bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must be [{D}], got {tuple(t.shape)}")
    for name, t in (("delta", delta), ("gate", gate), ("B", B), ("C", C)):
        if t is not None and t.dtype != u.dtype:
            raise ValueError(f"{name} dtype {t.dtype} must match u dtype {u.dtype}")
    for name, t in (("delta", delta), ("A", A), ("B", B), ("C", C), ("skip", skip), ("gate", gate),
                    ("delta_bias", delta_bias)):
        if t is not None and t.device != u.device:
            raise ValueError(f"{name} is on {t.device}, u on {u.device}")
    return T, D, N, B.shape[1]


def _group_rows(t):
    """B or C [T, F, N] as (tensor, token-row stride): read in place when each
    token's F x N block is contiguous."""
    T, F, N = t.shape
    if (t.stride(2) == 1 or N == 1) and (t.stride(1) == N or F == 1) and (t.stride(0) >= F * N or T == 1):
        return t, max(t.stride(0), F * N)
    return t.contiguous(), F * N


def _fp32(t):
    """fp32, contiguous and on a 16-byte boundary, as the kernels read it."""
    if t is None:
        return None
    t = (t if t.dtype == torch.float32 else t.float()).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _Operands:
    """The operands of a call as the kernels take them: tensors (kept alive)
    and the leading arguments of the C calls."""

    def __init__(self, u, delta, A, B, C, skip, gate, delta_bias):
        self.u, ldu = channel_rows(u)
        self.delta, ldd = channel_rows(delta)
        self.gate, ldg = (None, 0) if gate is None else channel_rows(gate)
        self.B, ldb = _group_rows(B)
        self.C, ldc = _group_rows(C)
        self.A, self.skip, self.delta_bias = _fp32(A), _fp32(skip), _fp32(delta_bias)
        p = _capi.ptr
        self.args = (_capi.dtype_code(u), p(self.u), ldu, p(self.delta), ldd, p(self.gate), ldg, p(self.B), ldb,
                     p(self.C), ldc, p(self.A), p(self.skip), p(self.delta_bias))


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _scan_forward(ops, T, D, N, F, cu_seqlens, softplus, saved):
    u = ops.u
    out = torch.empty(T, D, dtype=u.dtype, device=u.device)
    cu, cu64, nseq = _cu(cu_seqlens, u.device)
    ranges = _capi.token_ranges()
    L = _capi.lib()
    with torch.cuda.device(u.device.index):
        ws = _workspace(L.greta_ssm_scan_workspace(nseq, T, D, N, F, ranges), u.device)
        st = L.greta_ssm_scan_fwd(*ops.args, _capi.ptr(out), _capi.ptr(saved), _capi.ptr(cu), cu64, nseq, T, D, N, F,
                                  int(softplus), ranges, _capi.ptr(ws), 0 if ws is None else ws.numel(),
                                  _capi.stream_of(u))
    _capi.check("greta_ssm_scan_fwd", st)
    return out


class SelectiveScanFunction(torch.autograd.Function):
    """u, delta, gate [T, D]; A [D, N]; B, C [T, F, N]; skip, delta_bias [D]."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, skip, gate, delta_bias, cu_seqlens, softplus):
        (T, D), (_, F, N) = u.shape, B.shape
        ops = _Operands(u, delta, A, B, C, skip, gate, delta_bias)
        saved = None
        if any(ctx.needs_input_grad):
            saved = torch.empty(T // SAVE_EVERY + 1, D, N, dtype=torch.float32, device=u.device)
        cu, _, _ = _cu(cu_seqlens, u.device)
        out = _scan_forward(ops, T, D, N, F, cu, softplus, saved)
        ctx.save_for_backward(u, delta, A, B, C, skip, gate, delta_bias, cu, saved)
        ctx.softplus = softplus
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        u, delta, A, B, C, skip, gate, delta_bias, cu, saved = ctx.saved_tensors
        (T, D), (_, F, N) = u.shape, B.shape
        ops = _Operands(u, delta, A, B, C, skip, gate, delta_bias)
        dout = (dout if dout.dtype == u.dtype else dout.to(u.dtype)).contiguous()
        dev, dt, f32 = u.device, u.dtype, torch.float32
        du, ddelta = torch.empty(T, D, dtype=dt, device=dev), torch.empty(T, D, dtype=dt, device=dev)
        dgate = None if gate is None else torch.empty(T, D, dtype=dt, device=dev)
        dB, dC = torch.empty(T, F, N, dtype=dt, device=dev), torch.empty(T, F, N, dtype=dt, device=dev)
        dA = torch.empty(D, N, dtype=f32, device=dev)
        dskip = None if skip is None else torch.empty(D, dtype=f32, device=dev)
        dbias = None if delta_bias is None else torch.empty(D, dtype=f32, device=dev)
        cu, cu64, nseq = _cu(cu, dev)
        ranges = _capi.token_ranges()
        L, p = _capi.lib(), _capi.ptr
        with torch.cuda.device(dev.index):
            ws = _workspace(L.greta_ssm_scan_bwd_workspace(nseq, T, D, N, F, ranges), dev)
            st = L.greta_ssm_scan_bwd(
                *ops.args, p(saved), p(dout), p(du), p(ddelta), p(dgate), p(dB), p(dC), p(dA), p(dskip), p(dbias),
                p(cu), cu64, nseq, T, D, N, F, int(ctx.softplus), ranges, p(ws), 0 if ws is None else ws.numel(),
                _capi.stream_of(u))
        _capi.check("greta_ssm_scan_bwd", st)
        like = lambda g, t: g if g is None or g.dtype == t.dtype else g.to(t.dtype)  # noqa: E731
        return (du, ddelta, like(dA, A), dB, dC, like(dskip, skip), dgate, like(dbias, delta_bias), None, None)


@torch.compiler.disable(recursive=True)
def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   skip: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                   cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scan of packed sequences, differentiable in every operand.

    u, delta, gate (or None): [1, T, D]; A: [D, N] with N <= 128 (negative for
    a decaying state); B, C: [T, F, N], F groups of D / F consecutive channels
    each; skip, delta_bias: [D] or None; cu_seqlens: [N + 1] offsets (None: one
    sequence). Returns [1, T, D] contiguous. Every sequence starts from a zero
    state; rows that no sequence holds give zeros and zero gradients. When a
    gradient is needed, the forward keeps the states ahead of every 8th token
    (fp32 [T / 8 + 1, D, N]) for the backward.
    """
    if u.dim() != 3 or u.shape[0] != 1:
        raise ValueError(f"u must be [1, T, D], got {tuple(u.shape)}")
    for name, t in (("delta", delta), ("gate", gate)):
        if t is not None and tuple(t.shape) != tuple(u.shape):
            raise ValueError(f"{name} shape {tuple(t.shape)} must match u's {tuple(u.shape)}")
    # squeeze, not u[0], whose gradient would be copied into zeros
    u, delta, gate = u.squeeze(0), delta.squeeze(0), None if gate is None else gate.squeeze(0)
    _check(u, delta, A, B, C, skip, gate, delta_bias)
    if not u.is_cuda:
        raise ValueError("selective_scan requires CUDA tensors")
    if cu_seqlens is not None and (cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1):
        raise ValueError(f"cu_seqlens must be [N + 1], got {tuple(cu_seqlens.shape)}")
    return SelectiveScanFunction.apply(u, delta, A, B, C, skip, gate, delta_bias, cu_seqlens,
                                       delta_softplus).unsqueeze(0)


def _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out, flags):
    if u.dim() != 2:
        raise ValueError(f"u must be [T, D], got {tuple(u.shape)}")
    T, D, N, F = _check(u, delta, A, B, C, skip, gate, delta_bias)
    if state.dim() != 3 or tuple(state.shape[1:]) != (D, N):
        raise ValueError(f"state must be [slots, {D}, {N}], got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise ValueError(f"state must be float32, got {state.dtype}")
    if not u.is_cuda:
        raise ValueError("packed_selective_scan requires CUDA tensors")
    starts, slots, has_initial = packed_metadata(u, state, starts, slots, has_initial)
    out, new = packed_out(u, out)
    if T == 0:
        return out
    check_disjoint(out, u=u, delta=delta, gate=gate, B=B, C=C, state=state)
    ops = _Operands(u, delta, A, B, C, skip, gate, delta_bias)
    s_slot, s_d, s_n = state.stride()
    ranges = _capi.token_ranges()
    n = slots.numel()
    L = _capi.lib()
    with torch.cuda.device(u.device.index):
        ws = _workspace(L.greta_ssm_scan_workspace(n, T, D, N, F, ranges), u.device)
        st = L.greta_ssm_scan_packed(
            *ops.args, _capi.ptr(out), _capi.ptr(state) if state.numel() else None, state.shape[0], s_slot, s_d, s_n,
            _capi.ptr(starts), _capi.ptr(slots), _capi.ptr(has_initial), n, T, D, N, F, int(delta_softplus), new,
            ranges, _capi.ptr(flags), _capi.ptr(ws), 0 if ws is None else ws.numel(), _capi.stream_of(u))
    _capi.check("greta_ssm_scan_packed", st)
    return out


def packed_selective_scan(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial,
                          delta_softplus=False, out=None):
    """Scan of a packed serving batch with cache-slot states, prompts and single
    tokens in any mix.

    u, delta, gate (or None): [T, D]; B, C: [T, F, N]; A: [D, N]; skip,
    delta_bias: [D] or None; state: fp32 [slots, D, N], any strides, updated in
    place: each request starts from its slot's state (zeros without one, or
    where has_initial is 0) and leaves its last state there. starts: [N+1]
    offsets; slots, has_initial: [N], as in packed_dynamic_conv_triton: a
    negative slot has no state and is not written. A request without tokens
    leaves its slot as it was, and the requests of one batch have different
    slots. Returns [T, D]: `out` when given, whose rows behind the last request
    stay as they were (they are zeros in a new tensor).
    """
    return _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out,
                   None)


def packed_selective_scan_checked(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial,
                                  delta_softplus=False, out=None):
    """packed_selective_scan, reporting slots >= state.shape[0] (which the kernel
    skips) as IndexError. Waits for the device: for debugging and tests."""
    flags = torch.zeros(1, dtype=torch.int32, device=u.device)
    out = _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out,
                  flags)
    if int(flags.item()) & 1:
        raise IndexError(f"a cache slot index is >= the number of cache slots ({state.shape[0]})")
    return out


__all__ = ["selective_scan", "SelectiveScanFunction", "packed_selective_scan", "packed_selective_scan_checked"]
