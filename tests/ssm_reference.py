"""Plain 64-bit forms of the state-space operators, from their formulas, and the
error bounds that the kernels are held to.

Every function also computes magnitudes: the same sums with every product taken
absolute. A kernel that computes in fp32 and rounds its output once to type T
is off by at most half a step of T relative to the value, plus a number of fp32
roundings (2^-24 each) of the magnitude:

  convolution   W + 8 (taps, bias, sigmoid), plus the number of tokens in the
                sums of dw and dbias
  scan          32 per token of the longest sequence, + 64, + the terms of a
                sum over channels or tokens. Per token the state is multiplied
                by a decay exp(dt A): 2 ulp = 4 roundings from the exponential,
                one each from argument, product, input and sum (8), and
                dt's own error, up to 2^-21 = 8 roundings relative, which moves
                the argument by 8 |dt A|; the inputs keep |dt A| <= 3 (24). 64
                covers softplus, SiLU and the sum over states (up to 128 terms
                are added in a tree of depth 7 over 4 sums)
"""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ROUNDING = 2.0 ** -24


def assert_within(got, ref, mag, dtype, roundings, what=""):
    got, ref, mag = got.detach().double().cpu(), ref.double().cpu(), mag.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-37  # fp16 subnormals; fp32 flushes them
    tol = HALF_STEP[dtype] * ref.abs() + roundings * ROUNDING * mag * (1 + HALF_STEP[dtype]) + tiny
    off = (got - ref).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = int(torch.nan_to_num(off / tol, nan=1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst at {i}: got "
                             f"{got.flatten()[i]:.9g}, expected {ref.flatten()[i]:.9g} +- {tol.flatten()[i]:.3g}")


def _silu(v):
    return v * torch.sigmoid(v)


def _dsilu(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def segments(cu, tokens):
    """[(request, first, end)] of the sequences that have tokens."""
    if cu is None:
        return [(0, 0, tokens)]
    cu = [min(max(int(v), 0), tokens) for v in cu]
    return [(i, a, b) for i, (a, b) in enumerate(zip(cu, cu[1:])) if b > a]


def conv(x, w, bias, silu, cu=None, history=None, dout=None):
    """x [T, D], w [W, D]; history {request: [W-1, D]}. Returns (values,
    magnitudes), dicts with out, and with dout dx, dw, dbias."""
    x, w = x.double(), w.double()
    W, (T, D) = w.shape[0], x.shape
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    val = {"out": torch.zeros_like(x)}
    mag = {"out": torch.zeros_like(x)}
    if dout is not None:
        for d in (val, mag):
            d["dx"], d["dw"], d["dbias"] = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i, a, e in segments(cu, T):
        past = torch.zeros(W - 1, D, dtype=torch.float64, device=x.device)
        if history is not None and i in history:
            past = history[i].double()
        rows = torch.cat([past, x[a:e]])
        n = e - a
        taps = torch.stack([rows[k:k + n] for k in range(W)], 1)  # [n, W, D]
        pre = (taps * w).sum(1) + b
        pmag = (taps.abs() * w.abs()).sum(1) + b.abs()
        val["out"][a:e] = _silu(pre) if silu else pre
        # |SiLU'| <= 1.1
        mag["out"][a:e] = 1.1 * pmag
        if dout is None:
            continue
        g = dout[a:e].double()
        dpre = g * _dsilu(pre) if silu else g
        # SiLU'' is below 0.5: an error of pre moves dpre by half of it
        dmag = g.abs() * (1.1 + 0.5 * pmag) if silu else g.abs()
        for k in range(W):
            j = W - 1 - k  # token t + j reads x[t] with tap k
            if j < n:
                val["dx"][a:e - j] += w[k] * dpre[j:]
                mag["dx"][a:e - j] += w[k].abs() * dmag[j:]
        val["dw"] += (taps * dpre[:, None]).sum(0)
        mag["dw"] += (taps.abs() * dmag[:, None]).sum(0)
        val["dbias"] += dpre.sum(0)
        mag["dbias"] += dmag.sum(0)
    return val, mag


def _scan_pass(u, dt, slope, A, B, C, skip, gate, segs, before, dout, absolute):
    """One evaluation of the scan's formulas, with every factor absolute or not."""
    sign = (lambda v: v.abs()) if absolute else (lambda v: v)
    T, D = u.shape
    F, N = B.shape[1:]
    per = D // F
    dev = u.device
    decay = A
    u, B, C, skip, A = sign(u), sign(B), sign(C), sign(skip), sign(A)
    z = None if gate is None else sign(_silu(gate))
    out = {"out": torch.zeros(T, D, dtype=torch.float64, device=dev), "last": {}}
    if dout is not None:
        dout = sign(dout)
        for k in ("du", "ddelta", "dgate"):
            out[k] = torch.zeros(T, D, dtype=torch.float64, device=dev)
        for k in ("dB", "dC"):
            out[k] = torch.zeros(T, F, N, dtype=torch.float64, device=dev)
        out["dA"] = torch.zeros(D, N, dtype=torch.float64, device=dev)
        out["dskip"] = torch.zeros(D, dtype=torch.float64, device=dev)
        out["ddelta_bias"] = torch.zeros(D, dtype=torch.float64, device=dev)
    for i, a, e in segs:
        h = sign(before[i]) if before is not None and i in before else torch.zeros(D, N, dtype=torch.float64, device=dev)
        hs, ys = [h], []
        for t in range(a, e):
            bt, ct = B[t].repeat_interleave(per, 0), C[t].repeat_interleave(per, 0)
            h = torch.exp(dt[t][:, None] * decay) * h + (dt[t] * u[t])[:, None] * bt
            hs.append(h)
            ys.append((ct * h).sum(-1) + skip * u[t])
        out["last"][i] = h
        y = torch.stack(ys)
        out["out"][a:e] = y if z is None else y * z[a:e]
        if dout is None:
            continue
        dy = dout[a:e] if z is None else dout[a:e] * z[a:e]
        if gate is not None:
            # |SiLU'| and the move of SiLU' by an error of the gate
            d = _dsilu(gate[a:e])
            out["dgate"][a:e] = dout[a:e] * y * (d.abs() + 0.5 if absolute else d)
        r = torch.zeros(D, N, dtype=torch.float64, device=dev)
        for t in range(e - 1, a - 1, -1):
            bt, ct = B[t].repeat_interleave(per, 0), C[t].repeat_interleave(per, 0)
            g = ct * dy[t - a][:, None] + r
            r = torch.exp(dt[t][:, None] * decay) * g
            kept = r * hs[t - a]
            gb = (g * bt).sum(-1)
            out["dC"][t] = (dy[t - a][:, None] * hs[t - a + 1]).view(F, per, N).sum(1)
            out["dB"][t] = (g * (dt[t] * u[t])[:, None]).view(F, per, N).sum(1)
            out["du"][t] = skip * dy[t - a] + dt[t] * gb
            out["ddelta"][t] = ((kept * A).sum(-1) + u[t] * gb) * slope[t]
            out["dA"] += kept * dt[t][:, None]
        out["dskip"] += (dy * u[a:e]).sum(0)
        out["ddelta_bias"] += out["ddelta"][a:e].sum(0)
    return out


def scan(u, delta, A, B, C, skip=None, gate=None, delta_bias=None, softplus=False, cu=None, before=None, dout=None):
    """u, delta, gate [T, D]; B, C [T, F, N]; before {request: [D, N]}. Returns
    (values, magnitudes): dicts with out, last {request: state} and, with dout,
    the gradients by name."""
    T, D = u.shape
    d64 = lambda v: None if v is None else v.detach().double()  # noqa: E731
    u, delta, A, B, C, skip, gate, delta_bias = map(d64, (u, delta, A, B, C, skip, gate, delta_bias))
    zero = torch.zeros(D, dtype=torch.float64, device=u.device)
    raw = delta + (zero if delta_bias is None else delta_bias)
    dt = torch.nn.functional.softplus(raw, threshold=1000) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    before = None if before is None else {k: v.double() for k, v in before.items()}
    args = (A, B, C, zero if skip is None else skip, gate, segments(cu, T), before, d64(dout))
    return (_scan_pass(u, dt, slope, *args, absolute=False), _scan_pass(u, dt.abs(), slope, *args, absolute=True))
