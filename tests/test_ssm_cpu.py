"""State-space operators without a GPU: the plain 64-bit forms that the GPU
tests compare with are checked against automatic differentiation and
differences, the C ABI and the Python entry points refuse bad calls before any
launch, and workspace sizes follow the shapes."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

import ssm_reference as R

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "greta_ssm.h"
P = ctypes.c_void_p
FAKE = P(0x1000)  # never dereferenced: validation fails before any use


@pytest.fixture(scope="module")
def lib():
    from greta_plugin_b200 import _capi

    return _capi.lib()


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _scan_autograd(u, delta, A, B, C, skip, gate, bias, cu):
    """The recurrence in differentiable torch, token by token."""
    T, D = u.shape
    per = D // B.shape[1]
    dt = torch.nn.functional.softplus(delta + bias)
    out = []
    for _, a, e in R.segments(cu, T):
        h = torch.zeros(D, A.shape[1], dtype=torch.float64)
        for t in range(a, e):
            h = torch.exp(dt[t][:, None] * A) * h + (dt[t] * u[t])[:, None] * B[t].repeat_interleave(per, 0)
            out.append(((C[t].repeat_interleave(per, 0) * h).sum(-1) + skip * u[t]) * gate[t] * torch.sigmoid(gate[t]))
    return torch.stack(out)


def _scan_case(seed=0, T=9, D=6, N=3, F=2):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return dict(u=r(T, D), delta=r(T, D), A=-torch.rand(D, N, generator=g, dtype=torch.float64) - 0.1, B=r(T, F, N),
                C=r(T, F, N), skip=r(D), gate=r(T, D), delta_bias=r(D)), r(T, D)


def test_scan_reference_gradients_equal_autograd():
    case, dout = _scan_case()
    cu = [0, 4, 4, 9]
    val, _ = R.scan(**case, softplus=True, cu=cu, dout=dout)
    leaves = {k: v.clone().requires_grad_() for k, v in case.items()}
    out = _scan_autograd(leaves["u"], leaves["delta"], leaves["A"], leaves["B"], leaves["C"], leaves["skip"],
                         leaves["gate"], leaves["delta_bias"], cu)
    torch.testing.assert_close(val["out"], out.detach(), rtol=1e-12, atol=1e-12)
    grads = torch.autograd.grad(out, list(leaves.values()), dout)
    for k, gr in zip(leaves, grads):
        torch.testing.assert_close(val["d" + k], gr, rtol=1e-10, atol=1e-10)


def test_scan_reference_gradients_equal_differences():
    case, dout = _scan_case(seed=1)
    val, _ = R.scan(**case, softplus=True, cu=[0, 5, 9], dout=dout)
    eps = 1e-6
    for name in case:
        flat = case[name].flatten()
        for i in (0, flat.numel() // 2, flat.numel() - 1):
            side = []
            for s in (eps, -eps):
                v = flat.clone()
                v[i] += s
                o, _ = R.scan(**{**case, name: v.view_as(case[name])}, softplus=True, cu=[0, 5, 9])
                side.append((o["out"] * dout).sum())
            diff = (side[0] - side[1]) / (2 * eps)
            torch.testing.assert_close(val["d" + name].flatten()[i], diff, rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("silu", [False, True])
def test_conv_reference_gradients(silu):
    g = torch.Generator().manual_seed(3)
    x, w, b, dout = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((11, 5), (4, 5), (5,), (11, 5)))
    cu = [0, 2, 2, 10, 11]
    val, _ = R.conv(x, w, b, silu, cu=cu, dout=dout)
    lx, lw, lb = (t.clone().requires_grad_() for t in (x, w, b))
    parts = []
    for _, a, e in R.segments(cu, 11):
        rows = torch.cat([torch.zeros(3, 5, dtype=torch.float64), lx[a:e]])
        pre = torch.nn.functional.conv1d(rows.t()[None], lw.t()[:, None], lb, groups=5)[0].t()
        parts.append(torch.nn.functional.silu(pre) if silu else pre)
    out = torch.cat(parts)
    torch.testing.assert_close(val["out"], out.detach(), rtol=1e-12, atol=1e-12)
    for k, gr in zip(("dx", "dw", "dbias"), torch.autograd.grad(out, (lx, lw, lb), dout)):
        torch.testing.assert_close(val[k], gr, rtol=1e-10, atol=1e-10)


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------
def test_every_declared_symbol_is_exported_and_bound(lib):
    names = sorted(set(re.findall(r"GRETA_API\s+[\w\s\*]+?\b(greta_ssm_\w+)\s*\(", HEADER.read_text())))
    assert len(names) == 10
    for n in names:
        assert getattr(lib, n).argtypes is not None, n


def test_conv_rejects_bad_arguments(lib):
    from greta_plugin_b200 import _capi as C

    def fwd(dtype=C.DT_BF16, x=FAKE, ldx=64, w=FAKE, y=FAKE, cu=None, n=0, T=10, D=64, W=4):
        return lib.greta_ssm_conv_fwd(dtype, x, ldx, w, D, 1, None, y, cu, 0, n, T, D, W, 0, None)

    assert fwd(dtype=7) == C.ERR_UNSUPPORTED
    assert fwd(W=17) == C.ERR_UNSUPPORTED
    assert fwd(W=0) == C.ERR_INVALID_ARG
    assert fwd(D=0) == C.ERR_INVALID_ARG
    assert fwd(T=-1) == C.ERR_INVALID_ARG
    assert fwd(T=2 ** 31) == C.ERR_INVALID_ARG
    assert fwd(x=None) == C.ERR_INVALID_ARG
    assert fwd(y=None) == C.ERR_INVALID_ARG
    assert fwd(ldx=63) == C.ERR_INVALID_ARG
    assert fwd(n=2) == C.ERR_INVALID_ARG  # sequences without offsets
    assert fwd(T=0, x=None, w=None, y=None) == C.OK

    def bwd(dw=FAKE, bias=None, dbias=None, dout=FAKE, ws=FAKE, nbytes=1 << 40):
        return lib.greta_ssm_conv_bwd(C.DT_BF16, FAKE, 64, FAKE, 64, 1, bias, dout, FAKE, dw, dbias, None, 0, 0, 10,
                                      64, 4, 0, ws, nbytes, None)

    assert bwd(dw=None) == C.ERR_INVALID_ARG
    assert bwd(bias=FAKE) == C.ERR_INVALID_ARG
    assert bwd(dbias=FAKE) == C.ERR_INVALID_ARG
    assert bwd(dout=None) == C.ERR_INVALID_ARG
    assert bwd(ws=None) == C.ERR_INVALID_ARG
    assert bwd(nbytes=lib.greta_ssm_conv_bwd_workspace(10, 64, 4) - 1) == C.ERR_INVALID_ARG
    assert bwd(ws=P(0x1008)) == C.ERR_ALIGNMENT

    def packed(state=FAKE, slots_n=8, starts=FAKE, slots=FAKE, init=FAKE, n=2, W=4):
        return lib.greta_ssm_conv_packed(C.DT_BF16, FAKE, 64, FAKE, 64, 1, None, FAKE, state, slots_n, 192, 3, 1,
                                         starts, slots, init, n, 10, 64, W, 0, 0, None, None)

    assert packed(starts=None) == C.ERR_INVALID_ARG
    assert packed(slots=None) == C.ERR_INVALID_ARG
    assert packed(init=None) == C.ERR_INVALID_ARG
    assert packed(state=None) == C.ERR_INVALID_ARG
    assert packed(slots_n=-1) == C.ERR_INVALID_ARG


def test_scan_rejects_bad_arguments(lib):
    from greta_plugin_b200 import _capi as C

    def fwd(dtype=C.DT_BF16, u=FAKE, ldu=64, A=FAKE, B=FAKE, ldb=16, T=10, D=64, N=16, F=1, ranges=0, out=FAKE,
            saved=None, ws=FAKE, nbytes=1 << 40):
        return lib.greta_ssm_scan_fwd(dtype, u, ldu, FAKE, D, None, 0, B, ldb, FAKE, F * N, A, None, None, out, saved,
                                      None, 0, 0, T, D, N, F, 0, ranges, ws, nbytes, None)

    assert fwd(dtype=5) == C.ERR_UNSUPPORTED
    assert fwd(N=129, ldb=129) == C.ERR_UNSUPPORTED
    assert fwd(N=0) == C.ERR_INVALID_ARG
    assert fwd(F=3, ldb=48) == C.ERR_INVALID_ARG  # does not divide D
    assert fwd(F=0) == C.ERR_INVALID_ARG
    assert fwd(ranges=-1) == C.ERR_INVALID_ARG
    assert fwd(u=None) == C.ERR_INVALID_ARG
    assert fwd(A=None) == C.ERR_INVALID_ARG
    assert fwd(out=None) == C.ERR_INVALID_ARG
    assert fwd(ldu=63) == C.ERR_INVALID_ARG
    assert fwd(ldb=15) == C.ERR_INVALID_ARG
    assert fwd(T=2 ** 31) == C.ERR_INVALID_ARG
    assert fwd(A=P(0x1004)) == C.ERR_ALIGNMENT
    assert fwd(saved=P(0x1004)) == C.ERR_ALIGNMENT
    # several ranges need a workspace
    need = lib.greta_ssm_scan_workspace(0, 0, 64, 64, 16, 1, 3)
    assert need > 0
    assert fwd(T=64, ranges=3, ws=None) == C.ERR_INVALID_ARG
    assert fwd(T=64, ranges=3, nbytes=need - 1) == C.ERR_INVALID_ARG
    assert fwd(T=64, ranges=3, ws=P(0x1008)) == C.ERR_ALIGNMENT
    assert fwd(T=0, u=None, A=None, B=None, out=None) == C.OK

    def bwd(saved=FAKE, dA=FAKE, dgate=None, gate=None, skip=None, dskip=None, ws=FAKE):
        return lib.greta_ssm_scan_bwd(C.DT_BF16, FAKE, 64, FAKE, 64, gate, 64, FAKE, 16, FAKE, 16, FAKE, skip, None,
                                      saved, FAKE, FAKE, FAKE, dgate, FAKE, FAKE, dA, dskip, None, None, 0, 0, 10, 64,
                                      16, 1, 0, 0, ws, 1 << 40, None)

    assert bwd(saved=None) == C.ERR_INVALID_ARG
    assert bwd(dA=None) == C.ERR_INVALID_ARG
    assert bwd(gate=FAKE) == C.ERR_INVALID_ARG
    assert bwd(skip=FAKE) == C.ERR_INVALID_ARG
    assert bwd(ws=None) == C.ERR_INVALID_ARG
    assert bwd(saved=P(0x1004)) == C.ERR_ALIGNMENT

    def packed(state=FAKE, nslots=4, starts=FAKE, slots=FAKE, init=FAKE):
        return lib.greta_ssm_scan_packed(C.DT_BF16, FAKE, 64, FAKE, 64, None, 0, FAKE, 16, FAKE, 16, FAKE, None, None,
                                         FAKE, state, nslots, 1024, 16, 1, starts, slots, init, 2, 10, 64, 16, 1, 0,
                                         0, 0, None, FAKE, 1 << 40, None)

    assert packed(state=None) == C.ERR_INVALID_ARG
    assert packed(nslots=-1) == C.ERR_INVALID_ARG
    assert packed(starts=None) == C.ERR_INVALID_ARG
    assert packed(slots=None) == C.ERR_INVALID_ARG
    assert packed(init=None) == C.ERR_INVALID_ARG


def test_batch_metadata_rejects_bad_arguments(lib):
    from greta_plugin_b200 import _capi as C

    def f(q=FAKE, n=4, T=8, starts=FAKE, seq=FAKE, tables=None, row=8, width=8, bs=16, free=FAKE, nfree=4,
          slots=FAKE, used=FAKE):
        return lib.greta_ssm_batch_metadata(q, FAKE, n, T, starts, FAKE, seq, FAKE, tables, row, width, bs, free,
                                            nfree, slots, used, None)

    assert f(n=-1) == C.ERR_INVALID_ARG
    assert f(n=16385) == C.ERR_UNSUPPORTED
    assert f(T=-1) == C.ERR_INVALID_ARG
    assert f(q=None) == C.ERR_INVALID_ARG
    assert f(starts=None) == C.ERR_INVALID_ARG
    assert f(seq=None) == C.ERR_INVALID_ARG
    assert f(tables=FAKE, bs=0) == C.ERR_INVALID_ARG
    assert f(tables=FAKE, row=7) == C.ERR_INVALID_ARG
    assert f(tables=FAKE, free=None) == C.ERR_INVALID_ARG
    assert f(tables=FAKE, slots=None) == C.ERR_INVALID_ARG
    assert f(tables=FAKE, used=None) == C.ERR_INVALID_ARG


def test_workspaces_follow_the_shapes(lib):
    assert lib.greta_ssm_scan_workspace(0, 0, 100, 64, 16, 1, 1) == 0  # one range carries nothing
    assert lib.greta_ssm_scan_workspace(0, 0, 0, 64, 16, 1, 4) == 0
    assert lib.greta_ssm_scan_workspace(1, 64, 70, 64, 16, 1, 0) == 0  # single tokens
    two = lib.greta_ssm_scan_workspace(0, 0, 100, 64, 16, 1, 2)
    assert two >= 2 * (2 * 64 * 16 + 64) * 4
    assert lib.greta_ssm_scan_bwd_workspace(0, 100, 64, 16, 1, 1) >= 100 * 2 * 16 * 4 + 64 * 18 * 4
    assert lib.greta_ssm_conv_bwd_workspace(1, 64, 4) == 5 * 64 * 4


# ---------------------------------------------------------------------------
# Python entry points: refusals on CPU tensors, before the device is needed
# ---------------------------------------------------------------------------
def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _ints(*v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype)


@pytest.mark.parametrize("kw, match", [
    (dict(x=_t(2, 5, 8)), "x must be"),
    (dict(x=_t(5, 8)), "x must be"),
    (dict(weight=_t(4, 9)), "weight must be"),
    (dict(weight=_t(17, 8)), "kernel size"),
    (dict(bias=_t(9)), "bias must be"),
    (dict(activation="relu"), "activation"),
    (dict(x=_t(1, 5, 8, dtype=torch.float64)), "unsupported dtype"),
    (dict(), "requires CUDA"),
])
def test_causal_conv1d_refuses(kw, match):
    from greta_plugin_b200 import causal_conv1d

    with pytest.raises(ValueError, match=match):
        causal_conv1d(**{**dict(x=_t(1, 5, 8), weight=_t(4, 8)), **kw})


@pytest.mark.parametrize("kw, match", [
    (dict(x=_t(1, 5, 8)), "x must be"),
    (dict(state=_t(3, 8, 4)), "state must be"),
    (dict(state=_t(3, 8, 3, dtype=torch.float32)), "must match x dtype"),
    (dict(), "requires CUDA"),
])
def test_packed_causal_conv1d_refuses(kw, match):
    from greta_plugin_b200 import packed_causal_conv1d

    args = dict(x=_t(5, 8), weight=_t(4, 8), bias=None, state=_t(3, 8, 3), starts=_ints(0, 2, 5), slots=_ints(0, 1),
                has_initial=_ints(1, 1, dtype=torch.int8))
    with pytest.raises(ValueError, match=match):
        packed_causal_conv1d(**{**args, **kw})


def _scan_args(T=5, D=8, N=4, F=2, dtype=torch.bfloat16):
    return dict(u=_t(T, D, dtype=dtype), delta=_t(T, D, dtype=dtype), A=_t(D, N, dtype=torch.float32),
                B=_t(T, F, N, dtype=dtype), C=_t(T, F, N, dtype=dtype), skip=None, gate=None, delta_bias=None)


SCAN_REFUSALS = [
    (dict(A=_t(9, 4, dtype=torch.float32)), "A must be"),
    (dict(A=_t(8, 129, dtype=torch.float32)), "number of states"),
    (dict(B=_t(5, 3, 4)), "B must be"),
    (dict(B=_t(5, 2, 5)), "B must be"),
    (dict(C=_t(5, 1, 4)), "C shape"),
    (dict(skip=_t(7)), "skip must be"),
    (dict(delta_bias=_t(7)), "delta_bias must be"),
    (dict(C=_t(5, 2, 4, dtype=torch.float32)), "must match u dtype"),
    (dict(), "requires CUDA"),
]


@pytest.mark.parametrize("kw, match", SCAN_REFUSALS)
def test_selective_scan_refuses(kw, match):
    from greta_plugin_b200 import selective_scan

    args = {**_scan_args(), **kw}
    for k in ("u", "delta"):
        args[k] = args[k][None]
    with pytest.raises(ValueError, match=match):
        selective_scan(**args)


def test_selective_scan_refuses_batches_and_shapes():
    from greta_plugin_b200 import selective_scan

    a = _scan_args()
    with pytest.raises(ValueError, match="u must be"):
        selective_scan(**a)
    a["u"], a["delta"] = a["u"][None], _t(1, 5, 7)
    with pytest.raises(ValueError, match="delta shape"):
        selective_scan(**a)
    a["delta"], a["gate"] = _t(1, 5, 8), _t(1, 4, 8)
    with pytest.raises(ValueError, match="gate shape"):
        selective_scan(**a)


@pytest.mark.parametrize("kw, match", SCAN_REFUSALS + [
    (dict(gate=_t(5, 7)), "gate shape"),
    (dict(delta=_t(5, 7)), "delta shape"),
    (dict(state=_t(3, 8, 5, dtype=torch.float32)), "state must be"),
    (dict(state=_t(3, 8, 4)), "must be float32"),
])
def test_packed_selective_scan_refuses(kw, match):
    from greta_plugin_b200 import packed_selective_scan

    args = {**_scan_args(), "state": _t(3, 8, 4, dtype=torch.float32), "starts": _ints(0, 2, 5),
            "slots": _ints(0, 1), "has_initial": _ints(1, 1, dtype=torch.int8), **kw}
    with pytest.raises(ValueError, match=match):
        packed_selective_scan(**args)


def test_expanded_state_is_refused():
    """A state that several slots or channels share cannot be updated in place."""
    from greta_plugin_b200.causal_conv import packed_metadata

    meta = (_ints(0, 2, 5), _ints(0, 1), _ints(1, 1, dtype=torch.int8))
    for state in (_t(1, 8, 3).expand(4, 8, 3), _t(4, 1, 3).expand(4, 8, 3)):
        with pytest.raises(ValueError, match="expanded"):
            packed_metadata(_t(5, 8), state, *meta)
    for state in (_t(4, 8, 3), _t(1, 8, 3).expand(1, 8, 3), _t(4, 8, 0), _t(1, 8, 0).expand(4, 8, 0)):
        packed_metadata(_t(5, 8), state, *meta)


@pytest.mark.parametrize("kw, match", [
    (dict(query_lens=_ints(1, 2, dtype=torch.int64)), "query_lens"),
    (dict(context_lens=_ints(1)), "context_lens has"),
    (dict(num_tokens=-1), "num_tokens"),
    (dict(block_tables=_t(3, 4, dtype=torch.int32)), "block_tables must be"),
    (dict(block_tables=_t(2, 4, dtype=torch.int64)), "block_tables must be"),
    (dict(block_tables=_t(4, 2, dtype=torch.int32).t()), "contiguous"),
    (dict(block_tables=_t(2, 4, dtype=torch.int32)), "block_size"),
    (dict(block_tables=_t(2, 4, dtype=torch.int32), block_size=16), "free_blocks"),
    (dict(free_blocks=_ints(1)), "without block_tables"),
    (dict(), "requires CUDA"),
])
def test_packed_batch_metadata_refuses(kw, match):
    from greta_plugin_b200 import packed_batch_metadata

    args = dict(query_lens=_ints(1, 2), context_lens=_ints(0, 5), num_tokens=3)
    with pytest.raises(ValueError, match=match):
        packed_batch_metadata(**{**args, **kw})


def test_overlap_of_out_is_refused():
    from greta_plugin_b200.causal_conv import check_disjoint

    buf = torch.zeros(10, 16)
    check_disjoint(buf[:5], x=buf[5:], state=None, other=torch.zeros(0))
    with pytest.raises(ValueError, match="overlap x"):
        check_disjoint(buf[:6], x=buf[5:])
    with pytest.raises(ValueError, match="overlap x"):
        check_disjoint(buf, x=buf[:, 8:])  # a strided view inside
