"""State-space operators on the GPU at the edges of what a call may be: operands
on odd addresses, offsets that fall, request tables with many empty rows, mixed
batches of many requests, token ranges chosen by hand, rows and slots past 2^31
elements on the prompts' kernels, parameters of another type than the inputs,
calls from two threads. The plain forms and bounds are those of
ssm_reference.py, the cases' helpers those of the operators' own test files."""
import pytest
import torch

import ssm_reference as R
import test_gpu_ssm_conv as conv_tests
import test_gpu_ssm_scan as scan_tests
from gpu_helpers import DEV, rand, ragged_cu

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def odd(t):
    """`t` [T, ...] as a view whose rows begin on odd elements (an odd offset and
    an odd row stride)."""
    flat = t.reshape(t.shape[0], -1)
    T, n = flat.shape
    ld = n + 1 + n % 2  # odd
    view = torch.zeros(T * ld + 2, dtype=t.dtype, device=t.device)[1:1 + T * ld].view(T, ld)[:, :n]
    view.copy_(flat)
    return view.unflatten(1, t.shape[1:]) if t.dim() > 2 else view


def odd_operands(s):
    return {k: odd(v) if v is not None and k in ("u", "delta", "gate", "B", "C") else v for k, v in s.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D, N, F", [(61, 9, 1), (64, 16, 1), (40, 20, 2), (12, 65, 1)])
def test_scan_operands_on_odd_addresses(dtype, D, N, F):
    """Column views that start on no vector: partial tiles, slices and groups of
    states have elements that are not there, which no copy may name an
    unaligned address for."""
    lens = [30, 1, 41]
    s, dout = scan_tests.make(sum(lens), D, N, F, dtype, D)
    s = odd_operands(s)
    assert all(s[k].data_ptr() % 4 == 2 for k in ("u", "B")) or dtype == torch.float32
    cu = ragged_cu(lens).to(DEV)
    val, mag = R.scan(**s, softplus=True, cu=cu.tolist(), dout=dout)
    got = scan_tests.run_train(s, dout, cu)
    scan_tests.compare(got, val, mag, dtype, max(lens), sum(lens), D, F)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1] * 9, [50, 1, 37]])
def test_packed_scan_operands_on_odd_addresses(dtype, lens):
    from greta_plugin_b200 import packed_selective_scan

    n, T = len(lens), sum(lens)
    for D, N in ((61, 9), (64, 16)):
        s, _ = scan_tests.make(T, D, N, 1, dtype, N)
        s = odd_operands(s)
        state = torch.randn(n, D, N, generator=torch.Generator().manual_seed(N)).to(DEV)
        before = {i: state[i].clone() for i in range(n)}
        starts = ragged_cu(lens)
        out = packed_selective_scan(**s, state=state, starts=starts.to(DEV),
                                    slots=torch.arange(n, dtype=torch.int32, device=DEV),
                                    has_initial=torch.ones(n, dtype=torch.int8, device=DEV), delta_softplus=True)
        val, mag = R.scan(**s, softplus=True, cu=starts.tolist(), before=before)
        R.assert_within(out, val["out"], mag["out"], dtype, 32 * max(lens) + 64, "out")
        for i in range(n):
            R.assert_within(state[i], val["last"][i], mag["last"][i], torch.float32, 32 * max(lens) + 64, f"state {i}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D, W, wide", [(256, 4, "both"), (100, 3, "weight"), (64, 7, "bias")])
def test_conv_gradients_of_fp32_parameters(dtype, D, W, wide):
    """fp32 filters or bias beside 16-bit inputs: their gradients keep the fp32
    sums' bits (a sum rounded to the inputs' type on the way is off by 2^-9)."""
    from greta_plugin_b200 import causal_conv1d

    g = torch.Generator().manual_seed(W)
    lens = [150, 1, 89]
    T = sum(lens)
    x, dout = (rand(g, T, D, dtype=dtype).to(DEV) for _ in range(2))
    w = rand(g, W, D, scale=W ** -0.5, dtype=torch.float32).to(DEV)
    b = rand(g, D, dtype=torch.float32).to(DEV)
    w, b = w.to(dtype if wide == "bias" else w.dtype), b.to(dtype if wide == "weight" else b.dtype)
    w, b = w.requires_grad_(), b.requires_grad_()
    cu = ragged_cu(lens).to(DEV)
    causal_conv1d(x[None], w, b, cu, "silu").backward(dout[None])
    val, mag = R.conv(x, w.detach().to(dtype), b.detach().to(dtype), True, cu=cu.tolist(), dout=dout)
    # the sums' own roundings, and the sigmoid of 16-bit inputs: 20 for arguments
    # up to 10 (10 from the argument, 4 from the power, 3 from sum and
    # reciprocal), twice in SiLU'
    n = 2 * (W + 8) + T + 40
    assert w.grad.dtype == w.dtype and b.grad.dtype == b.dtype
    R.assert_within(w.grad, val["dw"], mag["dw"], w.dtype, n, "dw")
    R.assert_within(b.grad, val["dbias"], mag["dbias"], b.dtype, n, "dbias")


def test_conv_gradients_of_fp32_parameters_over_no_tokens():
    from greta_plugin_b200 import causal_conv1d

    x = torch.zeros(1, 0, 64, device=DEV, dtype=torch.bfloat16)
    w, b = torch.ones(4, 64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True)
    causal_conv1d(x, w, b, None, "silu").sum().backward()
    assert w.grad.dtype == torch.float32 and not w.grad.any() and not b.grad.any()


def meta(lens, slots, init=None):
    """(starts, slots, has_initial) on the device."""
    init = [1] * len(lens) if init is None else init
    return (ragged_cu(lens).to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV),
            torch.tensor(init, dtype=torch.int8, device=DEV))


@pytest.mark.parametrize("lens", [[1, 1], [100, 1]])  # the single tokens' kernels, the prompts'
@pytest.mark.parametrize("slots, bad", [([0, 5], True), ([5, 0], True), ([-1, 0], False)])
def test_checked_calls_report_slots_out_of_range(lens, slots, bad):
    """Also where there is no state to look at: no slots, or filters of one tap."""
    import greta_plugin_b200 as greta

    T, D, N = sum(lens), 64, 16
    s, _ = scan_tests.make(T, D, N, 1, torch.bfloat16, 1)
    x = s["u"]
    for rows in (2, 0):
        for W in (4, 1):
            w = torch.ones(W, D, dtype=x.dtype, device=DEV)
            state = torch.full((rows, D, W - 1), 3.0, dtype=x.dtype, device=DEV)
            call = lambda: greta.packed_causal_conv1d_checked(x, w, None, state, *meta(lens, slots))  # noqa: E731
            if bad or rows == 0:
                with pytest.raises(IndexError, match="cache slot"):
                    call()
            else:
                call()
            assert rows == 0 or (state[1] == 3).all()
        state = torch.full((rows, D, N), 3.0, device=DEV)
        st, sl, init = meta(lens, slots)
        call = lambda: greta.packed_selective_scan_checked(**s, state=state, starts=st, slots=sl,  # noqa: E731
                                                           has_initial=init, delta_softplus=True)
        if bad or rows == 0:
            with pytest.raises(IndexError, match="cache slot"):
                call()
        else:
            call()
        assert rows == 0 or (state[1] == 3).all()


def test_checked_calls_without_slots():
    """Requests that have no slot need none."""
    import greta_plugin_b200 as greta

    s, _ = scan_tests.make(51, 64, 16, 1, torch.bfloat16, 1)
    st, sl, init = meta([50, 1], [-1, -1])
    greta.packed_selective_scan_checked(**s, state=torch.zeros(0, 64, 16, device=DEV), starts=st, slots=sl,
                                        has_initial=init, delta_softplus=True)
    greta.packed_causal_conv1d_checked(s["u"], s["u"][:4], None, s["u"].new_zeros(0, 64, 3), st, sl, init)


@pytest.mark.parametrize("starts", [[0, 1, 10, 3], [0, 1, 2, 14, 5, 6], [0, 9, 4, 0, 0, 0], [3, 1, 12, 2, 40]])
@pytest.mark.parametrize("W", [4, 16])
def test_packed_conv_offsets_that_fall_read_no_other_rows(starts, W):
    """Offsets that fall name no valid batch, but its reads stay inside x: what
    lies around x reaches no slot and no output. (Rows that such offsets give to
    no run stay as `out` was: of 0, 9, 4, 0, 0, 0 the search gives token 1 to
    request 3, whose first three tokens belong to the run of its first, 0, which
    the search gives to request 3 as well, to end at 1.)"""
    from greta_plugin_b200 import packed_causal_conv1d

    n = len(starts) - 1
    for T, D in ((14, 64), (40, 64), (40, 8192)):  # (runs of one token, and of three)
        around = torch.full((T + 64, D), 777.0, dtype=torch.bfloat16, device=DEV)
        x = around[32:32 + T]
        x.fill_(1.0)
        state = torch.full((n, D, W - 1), 1.0, dtype=torch.bfloat16, device=DEV)
        meta_ = (torch.tensor(starts, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV),
                 torch.ones(n, dtype=torch.int8, device=DEV))
        out = torch.zeros_like(x)
        packed_causal_conv1d(x, torch.ones(W, D, dtype=torch.bfloat16, device=DEV), None, state, *meta_, out=out)
        assert float(out.max()) <= W and float(state.max()) <= 1.0


def test_scan_more_groups_than_a_grid_dimension():
    """F may be any divisor of D."""
    lens, D = [2, 1], 70000
    s, dout = scan_tests.make(3, D, 1, D, torch.float32, 2)
    cu = ragged_cu(lens).to(DEV)
    val, mag = R.scan(**s, softplus=True, cu=cu.tolist(), dout=dout)
    scan_tests.compare(scan_tests.run_train(s, dout, cu), val, mag, torch.float32, 2, 3, D, D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("table, at, n", [(256, 128, 256), (300, 0, 301), (64, 63, 60)])
def test_request_tables_with_many_empty_rows(dtype, table, at, n):
    """A long request in a table of empty ones has the rows of a batch of single
    tokens, and is walked by the kernels of those, or, with max_query_len, not."""
    from greta_plugin_b200 import packed_causal_conv1d, packed_selective_scan

    lens = [0] * table
    lens[at] = n
    if n < 100:
        lens[5], lens[40] = 1, 3
    T, D, N, W = sum(lens), 72, 16, 4
    slots = [int(v) for v in torch.randperm(table + 2, generator=torch.Generator().manual_seed(n))[:table]]
    scan_tests.check_packed(lens, slots, [1] * table, D, N, 1, dtype, seed=n)
    conv_tests.check_packed(lens, slots, [1] * table, D, W, dtype, seed=n)
    s, _ = scan_tests.make(T, D, N, 1, dtype, n)
    st, sl, init = meta(lens, slots)
    state = torch.randn(table + 2, D, N, generator=torch.Generator().manual_seed(n)).to(DEV)
    before = {i: state[k].clone() for i, k in enumerate(slots)}
    val, mag = R.scan(**s, softplus=True, cu=st.tolist(), before=before)
    for most in (n, 10 ** 6):
        now = state.clone()
        out = packed_selective_scan(**s, state=now, starts=st, slots=sl, has_initial=init, delta_softplus=True,
                                    max_query_len=most)
        R.assert_within(out, val["out"], mag["out"], dtype, 32 * n + 64, "out")
        for i in val["last"]:
            R.assert_within(now[slots[i]], val["last"][i], mag["last"][i], torch.float32, 32 * n + 64, f"state {i}")
    w, history = s["u"][:W], torch.ones(table + 2, D, W - 1, dtype=dtype, device=DEV)
    want = packed_causal_conv1d(s["u"], w, None, history.clone(), st, sl, init)
    assert torch.equal(want, packed_causal_conv1d(s["u"], w, None, history, st, sl, init, max_query_len=n))
