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

import functools
from typing import Optional

import torch

from . import _capi
from .causal_conv import channel_rows, check_disjoint, longest, packed_metadata, packed_out, same_device, to_real
from .dynamic_conv import _cu

MAX_STATES = 128
SAVE_EVERY = 8  # tokens per saved state


def _check(u, delta, A, B, C, skip, gate, delta_bias):
    """Shapes, types and devices of the operands ([T, D] rows, with or without a
    leading 1); (T, D, N, F)."""
    rows = u.shape
    T, D = rows[-2:]
    dt = u.dtype
    _capi.dtype_code(u)
    if delta.shape != rows:
        raise ValueError(f"delta shape {tuple(delta.shape)} must match u's {tuple(rows)}")
    if gate is not None and gate.shape != rows:
        raise ValueError(f"gate shape {tuple(gate.shape)} must match u's {tuple(rows)}")
    if A.dim() != 2 or A.shape[0] != D:
        raise ValueError(f"A must be [{D}, N], got {tuple(A.shape)}")
    N = A.shape[1]
    if not 1 <= N <= MAX_STATES:
        raise ValueError(f"the number of states must be between 1 and {MAX_STATES}, got {N}")
    groups = B.shape
    if len(groups) != 3 or groups[0] != T or groups[2] != N or groups[1] < 1 or D % groups[1] != 0:
        raise ValueError(f"B must be [{T}, F, {N}] with F dividing {D}, got {tuple(groups)}")
    if C.shape != groups:
        raise ValueError(f"C shape {tuple(C.shape)} must match B's {tuple(groups)}")
    if skip is not None and (skip.dim() != 1 or skip.shape[0] != D):
        raise ValueError(f"skip must be [{D}], got {tuple(skip.shape)}")
    if delta_bias is not None and (delta_bias.dim() != 1 or delta_bias.shape[0] != D):
        raise ValueError(f"delta_bias must be [{D}], got {tuple(delta_bias.shape)}")
    if delta.dtype != dt or B.dtype != dt or C.dtype != dt or (gate is not None and gate.dtype != dt):
        for name, t in (("delta", delta), ("gate", gate), ("B", B), ("C", C)):
            if t is not None and t.dtype != dt:
                raise ValueError(f"{name} dtype {t.dtype} must match u dtype {dt}")
    same_device("u", u, delta=delta, A=A, B=B, C=C, skip=skip, gate=gate, delta_bias=delta_bias)
    return T, D, N, groups[1]


def _group_rows(t):
    """B or C [T, F, N] as (tensor, token-row stride): read in place when each
    token's F x N block is contiguous."""
    T, F, N = t.shape
    row, group, state = t.stride()
    if (state == 1 or N == 1) and (group == N or F == 1) and (row >= F * N or T == 1):
        return t, max(row, F * N)
    return t.contiguous(), F * N


def _fp32(t):
    """fp32, contiguous and on a 16-byte boundary, as the kernels read it."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or not t.is_contiguous():
        t = to_real(t, torch.float32).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _operands(u, delta, A, B, C, skip, gate, delta_bias):
    """(tensors to keep alive, the leading arguments of the C calls)."""
    u, ldu = channel_rows(u)
    delta, ldd = channel_rows(delta)
    gate, ldg = (None, 0) if gate is None else channel_rows(gate)
    B, ldb = _group_rows(B)
    C, ldc = _group_rows(C)
    A, skip, delta_bias = _fp32(A), _fp32(skip), _fp32(delta_bias)
    p = _capi.addr
    return (u, delta, gate, B, C, A, skip, delta_bias), (
        _capi.dtype_code(u), u.data_ptr(), ldu, delta.data_ptr(), ldd, p(gate), ldg, B.data_ptr(), ldb, C.data_ptr(),
        ldc, A.data_ptr(), p(skip), p(delta_bias))


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(kind, device, nseq, T, D, N, F, ranges):
    """Bytes of workspace of a call on `device` (the sizes decide it alone). kind:
    "bwd", or the `packed` of greta_ssm_scan_workspace."""
    L = _capi.lib()
    with torch.cuda.device(device):
        if kind == "bwd":
            return L.greta_ssm_scan_bwd_workspace(nseq, T, D, N, F, ranges)
        return L.greta_ssm_scan_workspace(kind, nseq, T, D, N, F, ranges)


def _workspace(kind, device, *sizes):
    """(workspace or None, its bytes)"""
    n = _workspace_bytes(kind, device.index, *sizes)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


class SelectiveScanFunction(torch.autograd.Function):
    """u, delta, gate [1, T, D]; A [D, N]; B, C [T, F, N]; skip, delta_bias [D].
    (The views to [T, D] are made in here: outside they would be nodes of their
    own.)"""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, skip, gate, delta_bias, cu_seqlens, softplus, keep_states):
        u, delta, gate = u.squeeze(0), delta.squeeze(0), None if gate is None else gate.squeeze(0)
        (T, D), (_, F, N) = u.shape, B.shape
        keep, args = _operands(u, delta, A, B, C, skip, gate, delta_bias)
        saved = None
        if keep_states and any(ctx.needs_input_grad):
            saved = torch.empty(T // SAVE_EVERY + 1, D, N, dtype=torch.float32, device=u.device)
        cu, cu64, nseq = _cu(cu_seqlens, u.device)
        out = torch.empty(1, T, D, dtype=u.dtype, device=u.device)
        ranges = _capi.token_ranges()
        ws, n = _workspace(0, u.device, nseq, T, D, N, F, ranges)
        p = _capi.addr
        _capi.call("greta_ssm_scan_fwd", u, *args, p(out), p(saved), p(cu), cu64, nseq, T, D, N, F, int(softplus),
                   ranges, p(ws), n)
        ctx.save_for_backward(u, delta, A, B, C, skip, gate, delta_bias, cu, saved)
        ctx.softplus, ctx.ranges = softplus, ranges
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        u, delta, A, B, C, skip, gate, delta_bias, cu, saved = ctx.saved_tensors
        (T, D), (_, F, N) = u.shape, B.shape
        keep, args = _operands(u, delta, A, B, C, skip, gate, delta_bias)
        dev, dt, f32 = u.device, u.dtype, torch.float32
        dout = (dout if dout.dtype == dt else dout.to(dt)).contiguous()
        du, ddelta = torch.empty(1, T, D, dtype=dt, device=dev), torch.empty(1, T, D, dtype=dt, device=dev)
        dgate = None if gate is None else torch.empty(1, T, D, dtype=dt, device=dev)
        dB, dC = torch.empty(T, F, N, dtype=dt, device=dev), torch.empty(T, F, N, dtype=dt, device=dev)
        dA = torch.empty(D, N, dtype=f32, device=dev)
        dskip = None if skip is None else torch.empty(D, dtype=f32, device=dev)
        dbias = None if delta_bias is None else torch.empty(D, dtype=f32, device=dev)
        cu, cu64, nseq = _cu(cu, dev)
        ranges = ctx.ranges  # the forward call's: autograd runs this on a thread of its own
        ws, n = _workspace("bwd", dev, nseq, T, D, N, F, ranges)
        p = _capi.addr
        _capi.call("greta_ssm_scan_bwd", u, *args, p(saved), p(dout), p(du), p(ddelta), p(dgate), p(dB), p(dC), p(dA),
                   p(dskip), p(dbias), p(cu), cu64, nseq, T, D, N, F, int(ctx.softplus), ranges, p(ws), n)
        like = lambda g, t: g if g is None or g.dtype == t.dtype else g.to(t.dtype)  # noqa: E731
        return (du, ddelta, like(dA, A), dB, dC, like(dskip, skip), dgate, like(dbias, delta_bias), None, None, None)


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
    (fp32 [T / 8 + 1, D, N]) for the backward, which besides takes up to about
    2 GB for its sums of dB and dC (10 GB at 131072 tokens, 4096 x 128).
    """
    if u.dim() != 3 or u.shape[0] != 1:
        raise ValueError(f"u must be [1, T, D], got {tuple(u.shape)}")
    _check(u, delta, A, B, C, skip, gate, delta_bias)
    if not u.is_cuda:
        raise ValueError("selective_scan requires CUDA tensors")
    if cu_seqlens is not None and (cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1):
        raise ValueError(f"cu_seqlens must be [N + 1], got {tuple(cu_seqlens.shape)}")
    # (inside the node gradients are always off, and needs_input_grad is set without them too)
    return SelectiveScanFunction.apply(u, delta, A, B, C, skip, gate, delta_bias, cu_seqlens, delta_softplus,
                                       torch.is_grad_enabled())


def _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out,
            max_query_len, flags):
    if u.dim() != 2:
        raise ValueError(f"u must be [T, D], got {tuple(u.shape)}")
    T, D, N, F = _check(u, delta, A, B, C, skip, gate, delta_bias)
    most = 0 if max_query_len is None else longest(max_query_len)
    if state.dim() != 3 or state.shape[1] != D or state.shape[2] != N:
        raise ValueError(f"state must be [slots, {D}, {N}], got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise ValueError(f"state must be float32, got {state.dtype}")
    if not u.is_cuda:
        raise ValueError("packed_selective_scan requires CUDA tensors")
    starts, slots, has_initial = packed_metadata(u, state, starts, slots, has_initial)
    out, new = packed_out(u, out)
    if T == 0:
        return out
    if not new:
        check_disjoint(out, u=u, delta=delta, gate=gate, B=B, C=C, state=state)
    keep, args = _operands(u, delta, A, B, C, skip, gate, delta_bias)
    ranges, n = _capi.token_ranges(), slots.numel()
    ws, nbytes = _workspace(1 | most, u.device, n, T, D, N, F, ranges)
    p = _capi.addr
    _capi.call("greta_ssm_scan_packed", u, *args, p(out), p(state) or None, state.shape[0], *state.stride(), p(starts),
               p(slots), p(has_initial), n, T, D, N, F, int(delta_softplus), new | most, ranges, p(flags), p(ws),
               nbytes)
    return out


def packed_selective_scan(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial,
                          delta_softplus=False, out=None, max_query_len=None):
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

    max_query_len: the most tokens of any request, where the host knows it. A
    batch of at most 32 rows more than requests is taken for a decode step and
    walked request by request; with this, one long request in a table of empty
    ones is not (256 tokens beside 255 empty requests, 4096 x 16: 266 us without
    it, 35 with it). It has no say in the result, but for rounding.
    """
    return _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out,
                   max_query_len, None)


def packed_selective_scan_checked(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial,
                                  delta_softplus=False, out=None, max_query_len=None):
    """packed_selective_scan, reporting slots >= state.shape[0] (which the kernel
    skips) as IndexError. Waits for the device: for debugging and tests."""
    flags = torch.zeros(1, dtype=torch.int32, device=u.device)
    out = _packed(u, delta, A, B, C, skip, gate, delta_bias, state, starts, slots, has_initial, delta_softplus, out,
                  max_query_len, flags)
    if int(flags.item()) & 1:
        raise IndexError(f"a cache slot index is >= the number of cache slots ({state.shape[0]})")
    return out


__all__ = ["selective_scan", "SelectiveScanFunction", "packed_selective_scan", "packed_selective_scan_checked"]
