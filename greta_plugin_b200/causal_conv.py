"""Short causal depthwise convolution with static filters (the one ahead of a
selective scan), for training and for packed serving batches.

  pre[t, d] = bias[d] + sum_k weight[k, d] x[t + k - W + 1, d]   (tap W-1 = current token)
  out[t, d] = SiLU(pre) or pre

  causal_conv1d          packed sequences (cu_seqlens), zero history, with autograd
                         -> greta_ssm_conv_fwd / greta_ssm_conv_bwd
  packed_causal_conv1d   a serving batch with cache-slot state, prompts and single
                         tokens in any mix -> greta_ssm_conv_packed

Filters are tap-major [W, D], as this package's per-token filters are
[T, W, D/G]; a checkpoint's [D, 1, W] weight is passed as
`weight.squeeze(1).t()`, which the kernels read in place. x may be a column
view of a wider projection output (contiguous channels, any row stride). The
reference has no such convolution; its dynamic one is dynamic_conv.py.

There is no CPU fallback: non-CUDA tensors raise ValueError.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi
from .dynamic_conv import _cu

MAX_WIDTH = 16
GRADS_F32 = 0x100  # GRETA_SSM_GRADS_F32
LONGEST_BIT = 8  # GRETA_SSM_LONGEST


def _activation(activation) -> int:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return int(activation == "silu")


def channel_rows(t):
    """[T, D] as (tensor, row stride): read in place when the channels are
    contiguous and rows do not overlap, else made contiguous. Rows that start
    on whole vectors take the vector path; others are read by element."""
    T, D = t.shape
    row, col = t.stride()
    if (col == 1 or D == 1) and (row >= D or T == 1):
        return t, max(row, D)
    return t.contiguous(), D


def _check_weight(x, weight, bias):
    D = x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != D:
        raise ValueError(f"weight must be [W, {D}] (taps, channels), got {tuple(weight.shape)}")
    W = weight.shape[0]
    if not 1 <= W <= MAX_WIDTH:
        raise ValueError(f"kernel size must be between 1 and {MAX_WIDTH}, got {W}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != D):
        raise ValueError(f"bias must be [{D}], got {tuple(bias.shape)}")
    same_device("x", x, weight=weight, bias=bias)
    return W


def same_device(name, t, **others):
    dev = t.get_device()
    for o in others.values():
        if o is not None and o.get_device() != dev:
            k = next(k for k, v in others.items() if v is o)
            raise ValueError(f"{k} is on {o.device}, {name} on {t.device}")


def to_real(t, dtype):
    """t.to(dtype) for a real type, which would drop an imaginary part."""
    if t.is_complex():
        raise ValueError(f"parameters must be real, got {t.dtype}")
    return t.to(dtype)


def _as_type(t, dtype):
    return t if t is None or t.dtype == dtype else to_real(t, dtype)


def _bias(bias, dtype):
    return None if bias is None else _as_type(bias, dtype).contiguous()


class CausalConv1dFunction(torch.autograd.Function):
    """x [1, T, D] (rows may be strided), weight [W, D], bias [D] or None. (The
    views to [T, D] are made in here: outside they would be nodes of their own.)"""

    @staticmethod
    def forward(ctx, x, weight, bias, cu_seqlens, silu):
        x, ldx = channel_rows(x.squeeze(0))
        T, D = x.shape
        w, b = _as_type(weight, x.dtype), _bias(bias, x.dtype)
        y = torch.empty(1, T, D, dtype=x.dtype, device=x.device)
        cu, cu64, nseq = _cu(cu_seqlens, x.device)
        p = _capi.addr
        _capi.call("greta_ssm_conv_fwd", x, _capi.dtype_code(x), p(x), ldx, p(w), *w.stride(), p(b), p(y), p(cu), cu64,
                   nseq, T, D, w.shape[0], silu)
        ctx.save_for_backward(x, weight, bias, cu)
        ctx.silu = silu
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, weight, bias, cu = ctx.saved_tensors
        x, ldx = channel_rows(x)
        dt, dev = x.dtype, x.device
        w, b = _as_type(weight, dt), _bias(bias, dt)
        (T, D), W = x.shape, w.shape[0]
        dout = _as_type(dout, dt).contiguous()
        dx = torch.empty(1, T, D, dtype=dt, device=dev)
        # parameters of another type than x's take the fp32 sums, not sums rounded to x's type
        f32 = weight.dtype != dt or (bias is not None and bias.dtype != dt)
        sums = torch.float32 if f32 else dt
        dw = torch.empty(W, D, dtype=sums, device=dev)
        db = None if b is None else torch.empty(D, dtype=sums, device=dev)
        ws = torch.empty(_capi.lib().greta_ssm_conv_bwd_workspace(T, D, W), dtype=torch.uint8, device=dev)
        cu, cu64, nseq = _cu(cu, dev)
        p = _capi.addr
        _capi.call("greta_ssm_conv_bwd", x, _capi.dtype_code(x), p(x), ldx, p(w), *w.stride(), p(b), p(dout), p(dx),
                   p(dw), p(db), p(cu), cu64, nseq, T, D, W, ctx.silu | (GRADS_F32 if f32 else 0), p(ws), ws.numel())
        return dx, _as_type(dw, weight.dtype), None if b is None else _as_type(db, bias.dtype), None, None


@torch.compiler.disable(recursive=True)
def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  cu_seqlens: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
    """Convolution of packed sequences, differentiable in x, weight and bias.

    x: [1, T, D]; weight: [W, D]; bias: [D] or None; cu_seqlens: [N + 1]
    offsets (None: one sequence); activation: None or "silu". Returns
    [1, T, D] contiguous. Each sequence starts with zero history; rows that no
    sequence holds give zeros and zero gradients. weight and bias are used in
    x's type (fp32 ones beside 16-bit x are rounded to it, as its products are
    taken there); their gradients are summed in fp32 and rounded once, to the
    parameter's own type.
    """
    if x.dim() != 3 or x.shape[0] != 1:
        raise ValueError(f"x must be [1, T, D], got {tuple(x.shape)}")
    _check_weight(x, weight, bias)
    silu = _activation(activation)
    _capi.dtype_code(x)
    if not x.is_cuda:
        raise ValueError("causal_conv1d requires CUDA tensors")
    if cu_seqlens is not None and (cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1):
        raise ValueError(f"cu_seqlens must be [N + 1], got {tuple(cu_seqlens.shape)}")
    return CausalConv1dFunction.apply(x, weight, bias, cu_seqlens, silu)


def _as_meta(t, x, dtype):
    if t.dtype is dtype and t.get_device() == x.get_device() and t.dim() == 1 and t.is_contiguous():
        return t
    if dtype is torch.int8 and t.dtype not in (torch.bool, torch.uint8, torch.int8):
        t = t.ne(0)  # (a count, 256 say, has no place in 8 bits)
    elif t.dtype is torch.int64:
        t = t.clamp(-1, 2 ** 31 - 1)  # (past 32 bits there is no row and no slot, and not another one's)
    return t.to(device=x.device, dtype=dtype).reshape(-1).contiguous()


def packed_metadata(x, state, starts, slots, has_initial):
    """The request tensors on x's device in the kernels' types, checked against
    one another."""
    n = slots.numel()
    if starts.numel() != n + 1 or has_initial.numel() != n:
        raise ValueError(f"starts must hold one offset more than slots ({n}) and has_initial as many, got "
                         f"{starts.numel()} and {has_initial.numel()}")
    same_device("x", x, state=state)
    if 0 in state.stride() and state.numel() and any(st == 0 and size > 1 for st, size in zip(state.stride(), state.shape)):
        raise ValueError("state is updated in place and must not be expanded")
    return (_as_meta(starts, x, torch.int32), _as_meta(slots, x, torch.int32),
            _as_meta(has_initial, x, torch.int8))


def longest(max_query_len) -> int:
    """GRETA_SSM_LONGEST of max_query_len."""
    n = int(max_query_len)
    if n < 0:
        raise ValueError(f"max_query_len must not be negative, got {n}")
    return min(max(n, 1), 2 ** 22 - 1) << LONGEST_BIT


def packed_out(x, out):
    """(output of a packed call, whether it is new): `out`, checked, whose rows
    outside every request stay as they were, or a new tensor, where the kernel
    writes zeros to them."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device), 1
    if out.dtype != x.dtype or out.shape != x.shape or not out.is_contiguous() or out.get_device() != x.get_device():
        raise ValueError("out must be a contiguous tensor shaped and typed like the input, on its device")
    return out, 0


def check_disjoint(out, **inputs):
    """`out` is written while other rows of the inputs are still read."""
    a0 = out.data_ptr()
    a1 = a0 + out.numel() * out.element_size()
    for name, t in inputs.items():
        if t is None:
            continue
        b0 = t.data_ptr()
        if b0 >= a1 or t.numel() == 0 or a0 == a1:
            continue
        span = t.numel()
        if not t.is_contiguous():
            span = 1
            for n, s in zip(t.shape, t.stride()):
                span += (n - 1) * s
        if a0 < b0 + span * t.element_size():
            raise ValueError(f"out must not overlap {name}")


def _packed(x, weight, bias, state, starts, slots, has_initial, activation, out, max_query_len, flags):
    if x.dim() != 2:
        raise ValueError(f"x must be [T, D], got {tuple(x.shape)}")
    T, D = x.shape
    W = _check_weight(x, weight, bias)
    silu = _activation(activation)
    most = 0 if max_query_len is None else longest(max_query_len)
    if state.dim() != 3 or state.shape[1] != D or state.shape[2] != W - 1:
        raise ValueError(f"state must be [slots, {D}, {W - 1}], got {tuple(state.shape)}")
    if state.dtype != x.dtype:
        raise ValueError(f"state dtype {state.dtype} must match x dtype {x.dtype}")
    _capi.dtype_code(x)
    if not x.is_cuda:
        raise ValueError("packed_causal_conv1d requires CUDA tensors")
    starts, slots, has_initial = packed_metadata(x, state, starts, slots, has_initial)
    out, new = packed_out(x, out)
    if T == 0:
        return out
    if not new:
        check_disjoint(out, x=x, state=state)
    x, ldx = channel_rows(x)
    w, b = _as_type(weight, x.dtype), _bias(bias, x.dtype)
    p = _capi.addr
    _capi.call("greta_ssm_conv_packed", x, _capi.dtype_code(x), p(x), ldx, p(w), *w.stride(), p(b), p(out),
               p(state) or None, state.shape[0], *state.stride(), p(starts), p(slots), p(has_initial), slots.numel(),
               T, D, W, silu, new | most, p(flags))
    return out


def packed_causal_conv1d(x, weight, bias, state, starts, slots, has_initial, activation=None, out=None,
                         max_query_len=None):
    """Convolution of a packed serving batch with cache-slot history, in one launch.

    x: [T, D]; weight: [W, D]; bias: [D] or None; state: [slots, D, W-1] of x's
    type, any strides, updated in place. starts: [N+1] offsets of the N
    requests, prompts and single tokens in any mix; slots, has_initial: [N],
    with the meaning they have in packed_dynamic_conv_triton (a negative slot
    has no history and is not written). A request without tokens leaves its
    slot as it was, and the requests of one batch have different slots. Returns
    [T, D]: `out` when given, whose rows behind the last request stay as they
    were (they are zeros in a new tensor).

    max_query_len: the most tokens of any request, where the host knows it. A
    batch of at most 8 rows more than requests is taken for a decode step and
    walked request by request; with this, one long request in a table of empty
    ones is not. It has no say in the result.
    """
    return _packed(x, weight, bias, state, starts, slots, has_initial, activation, out, max_query_len, None)


def packed_causal_conv1d_checked(x, weight, bias, state, starts, slots, has_initial, activation=None, out=None,
                                 max_query_len=None):
    """packed_causal_conv1d, reporting slots >= state.shape[0] (which the kernel
    skips) as IndexError. Waits for the device: for debugging and tests."""
    flags = torch.zeros(1, dtype=torch.int32, device=x.device)
    out = _packed(x, weight, bias, state, starts, slots, has_initial, activation, out, max_query_len, flags)
    if int(flags.item()) & 1:
        raise IndexError(f"a cache slot index is >= the number of cache slots ({state.shape[0]})")
    return out


__all__ = ["causal_conv1d", "packed_causal_conv1d", "packed_causal_conv1d_checked", "CausalConv1dFunction"]
