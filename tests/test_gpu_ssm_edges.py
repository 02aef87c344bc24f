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


# ---------------------------------------------------------------------------
# which kernels run: the prompts' (ranges, with a workspace) or the single tokens'
# ---------------------------------------------------------------------------
@pytest.fixture
def calls(monkeypatch):
    """The scan's packed calls, as the bytes of workspace that they took: 0 is the
    single tokens' kernel (or one range, which these cases do not have)."""
    from greta_plugin_b200 import _capi

    taken, call = [], _capi.call

    def record(name, t, *args):
        if name == "greta_ssm_scan_packed":
            taken.append(args[-1])
        return call(name, t, *args)

    monkeypatch.setattr(_capi, "call", record)
    return taken


def mixed_batch(n, seed):
    """n requests: single tokens, idle ones, and four prompts of up to 90 tokens;
    distinct slots, some requests without one, some that start anew."""
    g = torch.Generator().manual_seed(seed)
    draw = lambda lo, hi, k: torch.randint(lo, hi, (k,), generator=g).tolist()  # noqa: E731
    lens = [int(v > 0) for v in draw(0, 8, n)]
    for at, m in zip(draw(0, n, 4), (90, 33, 17, 64)):
        lens[at] = m
    slots = torch.randperm(n + 3, generator=g)[:n].tolist()
    for at in draw(0, n, 1 + n // 10):
        slots[at] = -1
    return lens, slots, [int(v > 0) for v in draw(0, 4, n)]


@pytest.mark.parametrize("n", [40, 300, 1000])
@pytest.mark.parametrize("ranges", [0, 1, 7])
def test_packed_scan_prompts_beside_many_single_tokens(n, ranges, calls):
    """32 requests and more (the offsets come from memory, not from a lane)."""
    lens, slots, init = mixed_batch(n, n)
    scan_tests.check_packed(lens, slots, init, 72, 16, 1, torch.bfloat16, ranges=ranges, tail=5, seed=n)
    assert sum(lens) + 5 > n + 32 and (ranges == 1 or calls[-1] > 0)


@pytest.mark.parametrize("n", [40, 300, 1000])
@pytest.mark.parametrize("D, W, dtype", [(72, 4, torch.bfloat16), (512, 4, torch.float32), (61, 7, torch.float16)])
def test_packed_conv_prompts_beside_many_single_tokens(n, D, W, dtype):
    lens, slots, init = mixed_batch(n, n + 1)
    assert sum(lens) + 5 > n + 8
    conv_tests.check_packed(lens, slots, init, D, W, dtype, tail=5, seed=n)


def test_packed_scan_in_long_chunks_continues_like_one_call(calls):
    """A prompt in chunks of both kernels' lengths leaves what one call leaves."""
    from greta_plugin_b200 import packed_selective_scan

    chunks = [60, 1, 90, 33, 120, 1, 1]
    total = sum(chunks)
    s, _ = scan_tests.make(total, 64, 16, 1, torch.float32, 13)
    rows, rest = ("u", "delta", "B", "C", "gate"), {k: s[k] for k in ("A", "skip", "delta_bias")}
    val, mag = R.scan(**s, softplus=True)
    state = torch.full((1, 64, 16), 9.0, device=DEV)
    got, at = [], 0
    for n in chunks:
        st, sl, init = meta([n], [0], [int(at > 0)])
        got.append(packed_selective_scan(**{k: s[k][at:at + n] for k in rows}, **rest, state=state, starts=st, slots=sl,
                                         has_initial=init, delta_softplus=True))
        at += n
    assert [n > 0 for n in calls] == [n > 33 for n in chunks]
    base = 32 * total + 64
    R.assert_within(torch.cat(got), val["out"], mag["out"], torch.float32, base, "out")
    R.assert_within(state[0], val["last"][0], mag["last"][0], torch.float32, base, "state")


def test_packed_scan_slot_out_of_range_on_a_long_request(calls):
    """The prompts' kernels skip the slot and flag it, split over ranges or not."""
    from greta_plugin_b200 import _capi, packed_selective_scan_checked

    lens = [100, 1, 60]
    s, _ = scan_tests.make(161, 32, 16, 1, torch.bfloat16, 0)
    state = torch.ones(2, 32, 16, device=DEV)
    for ranges in (0, 6):
        for slots in ([5, 0, -1], [0, -1, 2]):
            st, sl, init = meta(lens, slots)
            with _capi.launch_options(rows_ranges=ranges), pytest.raises(IndexError, match="cache slot"):
                packed_selective_scan_checked(**s, state=state, starts=st, slots=sl, has_initial=init)
            assert (state[1] == 1).all() and calls[-1] > 0


def test_serving_steps_in_long_chunks_equal_one_training_call(calls):
    """Metadata, convolution and scan together in steps past the single tokens'
    kernels, against the formulas on the whole sequences."""
    import greta_plugin_b200 as greta

    D, N, W, total, f32 = 64, 16, 4, [170, 83, 121], torch.float32
    g = torch.Generator().manual_seed(0)
    seqs = [{k: rand(g, n, *s, dtype=f32).to(DEV) for k, s in
             (("x", (D,)), ("delta", (D,)), ("gate", (D,)), ("B", (1, N)), ("C", (1, N)))} for n in total]
    w, b = rand(g, W, D, scale=0.5, dtype=f32).to(DEV), rand(g, D, dtype=f32).to(DEV)
    A = -(torch.rand(D, N, generator=g) * 2 + 0.05).to(DEV)
    skip, bias = rand(g, D, dtype=f32).to(DEV), (rand(g, D, dtype=f32) - 2).to(DEV)
    conv_state, scan_state = torch.full((5, D, W - 1), 3.0, device=DEV), torch.full((5, D, N), 3.0, device=DEV)
    slots, context, got = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV), [0, 0, 0], [[], [], []]
    for step in ([70, 0, 40], [1, 80, 1], [98, 1, 79], [1, 2, 1]):
        T = sum(step) + 3
        rows = {k: torch.cat([s[k][c:c + n] for s, c, n in zip(seqs, context, step)] +
                             [torch.full_like(seqs[0][k][:3], float("nan"))]) for k in seqs[0]}
        m = greta.packed_batch_metadata(torch.tensor(step, dtype=torch.int32, device=DEV),
                                        torch.tensor(context, dtype=torch.int32, device=DEV), T)
        xc = greta.packed_causal_conv1d(rows["x"], w, b, conv_state, m.starts, slots, m.has_initial, "silu")
        y = greta.packed_selective_scan(xc, rows["delta"], A, rows["B"], rows["C"], skip, rows["gate"], bias,
                                        scan_state, m.starts, slots, m.has_initial, True)
        assert not y[sum(step):].any()
        at = 0
        for i, n in enumerate(step):
            got[i].append(y[at:at + n])
            at += n
            context[i] += n
    assert context == total and [n > 0 for n in calls] == [True, True, True, False]
    cu = ragged_cu(total).tolist()
    whole = {k: torch.cat([s[k] for s in seqs]) for k in seqs[0]}
    u, umag = R.conv(whole["x"], w, b, True, cu=cu)
    val, mag = R.scan(u["out"], whole["delta"], A, whole["B"], whole["C"], skip, whole["gate"], bias, True, cu)
    # the scan is linear in u, whose own error is W + 8 roundings of its magnitude
    _, by_u = R.scan(umag["out"], whole["delta"], A, whole["B"], whole["C"], skip, whole["gate"], bias, True, cu)
    n = 32 * max(total) + 64
    R.assert_within(torch.cat([torch.cat(v) for v in got]), val["out"], torch.maximum(mag["out"], by_u["out"]), f32,
                    n + W + 8, "serving")


def far_rows(s, T, ld):
    """The operands of `s` as column blocks of one buffer whose rows lie `ld`
    elements apart."""
    wide = {k: v for k, v in s.items() if v is not None and k in ("u", "delta", "gate", "B", "C")}
    sizes = {k: v[0].numel() for k, v in wide.items()}
    dt = s["u"].dtype
    buf = torch.empty((T - 1) * ld + sum(sizes.values()), dtype=dt, device=DEV)
    buf = buf.as_strided((T, sum(sizes.values())), (ld, 1))
    out, at = dict(s), 0
    for k, v in wide.items():
        view = buf[:, at:at + sizes[k]]
        view.copy_(v.reshape(T, -1))
        out[k] = view.unflatten(1, v.shape[1:]) if v.dim() > 2 else view
        at += sizes[k]
    return out


def test_scan_far_rows_and_slots_on_the_prompts_kernels(calls):
    """Rows of all operands and slots more than 2^31 elements apart give the near
    ones' bits: in split ranges, as the test before the single tokens' kernel."""
    from greta_plugin_b200 import _capi, packed_selective_scan

    lens, D, N = [9, 1, 1, 7], 64, 16
    T = sum(lens)
    s, _ = scan_tests.make(T, D, N, 1, torch.bfloat16, 21)
    far = far_rows(s, T, 2 ** 28 + 8)
    starts, slots, init = meta(lens, [1, 0, -1, 2])
    state = torch.randn(3, D, N, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    far_state = torch.empty(2 * (2 ** 30 + 64) + D * N, device=DEV).as_strided((3, D, N), (2 ** 30 + 64, N, 1))
    far_state.copy_(state)
    kw = dict(starts=starts, slots=slots, has_initial=init, delta_softplus=True)
    with _capi.launch_options(rows_ranges=3):
        want = packed_selective_scan(**s, state=state, **kw)
        got = packed_selective_scan(**far, state=far_state, **kw)
    assert all(n > 0 for n in calls)
    assert torch.equal(got, want) and torch.equal(far_state, state)


def test_scan_training_far_rows():
    """Forward and backward with rows more than 2^31 elements apart."""
    from greta_plugin_b200 import _capi

    lens, D, N = [9, 1, 8], 64, 16
    T = sum(lens)
    s, dout = scan_tests.make(T, D, N, 1, torch.bfloat16, 22)
    far, cu = far_rows(s, T, 2 ** 28 + 8), ragged_cu(lens).to(DEV)
    for ranges in (1, 3):
        with _capi.launch_options(rows_ranges=ranges):
            want = scan_tests.run_train(s, dout, cu)
            got = far_train(far, dout, cu)
        for k in got:
            assert torch.equal(got[k], want[k]), (k, ranges)


def far_train(s, dout, cu):
    """Outputs and gradients through the autograd node itself, which keeps the
    operands as they lie."""
    from greta_plugin_b200 import selective_scan

    leaf = {k: v.detach().requires_grad_() for k, v in s.items()}
    a = {**leaf, **{k: leaf[k][None] for k in ("u", "delta", "gate")}}
    out = selective_scan(**a, delta_softplus=True, cu_seqlens=cu)
    names = ("u", "delta", "gate", "A", "B", "C", "skip", "delta_bias")
    grads = torch.autograd.grad(out, [a[k] for k in names], dout[None])
    return {"out": out[0].detach(), **{"d" + k: g[0] if k in ("u", "delta", "gate") else g
                                       for k, g in zip(names, grads)}}


# ---------------------------------------------------------------------------
# ranges of whole sequences, and wide states
# ---------------------------------------------------------------------------
def takes_whole(lens, D, N, T):
    """The host's rule (ranges of whole sequences): the longest is at most 0.4 of
    what each scheduler has to walk in all."""
    lanes = 4 if N <= 16 else 8 if N <= 32 else 16 if N <= 64 else 32
    slices = -(-D // (32 // lanes * 4))
    return len(lens) < 32 and max(lens) <= int(0.4 * T * slices / (4 * torch.cuda.get_device_properties(0)
                                                                    .multi_processor_count))


WHOLE = [([23] * 20, 4096), ([5, 0, 40, 1, 1, 33, 17, 8, 64, 2, 0, 30] * 2, 8192), ([9, 31, 14, 1, 22] * 6, 4096)]


@pytest.mark.parametrize("lens, D", WHOLE)
@pytest.mark.parametrize("head, tail", [(0, 0), (13, 21)])
def test_train_ranges_of_whole_sequences(lens, D, head, tail):
    assert takes_whole(lens, D, 16, sum(lens) + head + tail)
    scan_tests.check_train(lens, D, 16, dtype=torch.bfloat16, head=head, tail=tail)


@pytest.mark.parametrize("lens, D", WHOLE)
def test_packed_ranges_of_whole_sequences(lens, D):
    assert takes_whole(lens, D, 16, sum(lens) + 9)
    n = len(lens)
    slots = [(7 * i) % n if i % 5 else -1 for i in range(n)] if n % 7 else list(range(n))
    scan_tests.check_packed(lens, slots, [1, 0] * (n // 2), D, 16, tail=9)


def test_ranges_of_whole_sequences_do_not_mix():
    """Two ranges share a tile where one ends and the next begins inside it: NaN in
    a sequence and in the rows outside change no bit of the others, forward and
    backward (sums over tokens apart)."""
    lens, D, tail = [23] * 20, 4096, 9
    T = sum(lens) + tail
    assert takes_whole(lens, D, 16, T)
    s, dout = scan_tests.make(T, D, 16, 1, torch.bfloat16, 5)
    cu = ragged_cu(lens).to(DEV)
    clean = scan_tests.run_train(s, dout, cu)
    for bad in (1, 6, 19):
        a, b = 23 * bad, 23 * (bad + 1)
        t = {k: v.clone() if v is not None else None for k, v in s.items()}
        for k in ("u", "delta", "B", "C", "gate"):
            t[k][a:b] = float("nan")
            t[k][-tail:] = float("nan")
        t["u"][a + 5] = float("inf")
        d = dout.clone()
        d[a:b] = float("nan")
        got = scan_tests.run_train(t, d, cu)
        for k in ("out", "du", "ddelta", "dgate", "dB", "dC"):
            assert torch.equal(got[k][:a], clean[k][:a]) and torch.equal(got[k][b:], clean[k][b:]), (k, bad)
            assert got[k][a:b].isnan().any(), (k, bad)


@pytest.mark.parametrize("N, F", [(64, 1), (128, 2)])
def test_train_wide_states_over_many_blocks(N, F):
    """Wide states beside many channels: hundreds of parts of dB and dC a token."""
    scan_tests.check_train([150, 1, 90], 2048, N, F, torch.bfloat16, seed=N)


@pytest.mark.parametrize("ranges", [1, 2, 5, 25])
@pytest.mark.parametrize("lens", [[200], [90, 1, 109], [1] * 40 + [150, 3]])
def test_train_ranges_reach_the_backward(ranges, lens, monkeypatch):
    """The forward's ranges in the backward too: adjoints carried over each."""
    from greta_plugin_b200 import _capi

    seen, call = [], _capi.call
    monkeypatch.setattr(_capi, "call", lambda name, t, *a: (seen.append((name, a[-3])), call(name, t, *a))[1])
    scan_tests.check_train(lens, 40, 16, seed=ranges, ranges=ranges)
    assert seen == [("greta_ssm_scan_fwd", ranges), ("greta_ssm_scan_bwd", ranges)]


def test_train_wide_states_in_several_launches():
    """So many tokens, channels and states that the backward takes its blocks of
    channels in several launches: channels have their halves' bits, and the sums
    over all channels those of the halves but for rounding. (Positive operands: no
    sum is smaller than its parts, of which 512 are added.)"""
    from greta_plugin_b200 import _capi, selective_scan

    T, D, N, ranges = 4200, 4096, 128, 6
    assert _capi.lib().greta_ssm_scan_bwd_workspace(1, T, D, N, 1, ranges) < T * 2 * N * 4 * 512  # rows of all blocks
    g = torch.Generator(DEV).manual_seed(0)
    one = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    u, dt, dout = one(1, T, D), one(1, T, D) * 0.2, one(1, T, D)
    A, B, C = -one(D, N) * 4 - 0.05, one(T, 1, N), one(T, 1, N)
    cu = torch.tensor([0, 1800, 1801, T], dtype=torch.int32, device=DEV)

    def grads(c):
        leaf = [v.contiguous().requires_grad_() for v in (u[..., c], dt[..., c], A[c], B.clone(), C.clone())]
        with _capi.launch_options(rows_ranges=ranges):
            out = selective_scan(*leaf, cu_seqlens=cu)
        return torch.autograd.grad(out, leaf, dout[..., c].contiguous())

    whole, halves = grads(slice(0, D)), [grads(slice(0, D // 2)), grads(slice(D // 2, D))]
    for i, dim in ((0, 2), (1, 2), (2, 0)):
        assert torch.equal(whole[i], torch.cat([h[i] for h in halves], dim))
    for i in (3, 4):
        want = halves[0][i].double() + halves[1][i].double()
        assert ((whole[i].double() - want).abs() <= 2 * 520 * R.ROUNDING * want).all()


@pytest.mark.parametrize("head, tail", [(0, 3000), (2500, 0), (900, 2100)])
def test_short_sequences_among_many_rows_outside(head, tail):
    """Short sequences beside long runs of rows that none holds, which are dealt to
    the ranges as a long sequence would be."""
    lens, D = [60, 100, 3, 80], 1024
    T = sum(lens) + head + tail
    got = scan_tests.check_train(lens, D, 16, dtype=torch.bfloat16, head=head, tail=tail)
    for k in ("out", "du", "ddelta", "dgate", "dB", "dC"):
        assert not got[k][:head].any() and not got[k][T - tail:].any(), k
    if head == 0:
        scan_tests.check_packed(lens, [2, 0, -1, 1], [1, 0, 1, 1], D, 16, tail=tail)
        scan_tests.check_packed(lens, [2, 0, -1, 1], [1, 0, 1, 1], D, 16, tail=tail, given_out=False)


def test_complex_parameters_are_refused():
    import greta_plugin_b200 as greta

    s, _ = scan_tests.make(5, 8, 4, 1, torch.bfloat16, 0)
    rows = {k: v[None] if k in ("u", "delta", "gate") else v for k, v in s.items()}
    st, sl, init = meta([5], [0])
    for k in ("A", "skip", "delta_bias"):
        z = s[k].to(torch.complex64)
        with pytest.raises(ValueError, match="must be real"):
            greta.selective_scan(**{**rows, k: z})
        with pytest.raises(ValueError, match="must be real"):
            greta.packed_selective_scan(**{**s, k: z}, state=torch.zeros(2, 8, 4, device=DEV), starts=st, slots=sl,
                                        has_initial=init)
    x, w, b = s["u"], s["u"][:3], s["u"][0]
    for kw in (dict(weight=w.to(torch.complex64), bias=b), dict(weight=w, bias=b.to(torch.complex64))):
        with pytest.raises(ValueError, match="must be real"):
            greta.causal_conv1d(x[None], **kw)
        with pytest.raises(ValueError, match="must be real"):
            greta.packed_causal_conv1d(x, **kw, state=x.new_zeros(2, 8, 2), starts=st, slots=sl, has_initial=init)


def test_growing_states_that_are_zero_for_ranges():
    """Positive rates: over a range the growth is past what fp32 holds, but the
    state that it multiplies is zero until the first input. (Gradients are not
    looked at: theirs go back to the first token, e^100 and more.)"""
    from greta_plugin_b200 import _capi, packed_selective_scan, selective_scan

    T, D, N = 104, 32, 16
    s, _ = scan_tests.make(T, D, N, 1, torch.float32, 3, options=("skip", "gate"))
    s["A"] = s["A"].abs() * 2 + 1  # up to 5, steps of 1: e^5 a token
    s["delta"] = torch.ones_like(s["delta"])
    s["u"][:100] = 0
    val, mag = R.scan(**s)
    # |dt A| of 5 takes 8 * 5 + 8 roundings a token, over the four tokens with a state
    n = 4 * 48 + 64
    st, sl, init = meta([T], [0], [0])
    for ranges in (0, 1, 6):
        state = torch.zeros(1, D, N, device=DEV)
        with _capi.launch_options(rows_ranges=ranges):
            out = selective_scan(**{k: v[None] if k in ("u", "delta", "gate") else v for k, v in s.items()})
            packed = packed_selective_scan(**s, state=state, starts=st, slots=sl, has_initial=init)
        R.assert_within(out[0], val["out"], mag["out"], torch.float32, n, f"out {ranges}")
        R.assert_within(packed, val["out"], mag["out"], torch.float32, n, f"packed {ranges}")
        R.assert_within(state[0], val["last"][0], mag["last"][0], torch.float32, n, f"state {ranges}")
