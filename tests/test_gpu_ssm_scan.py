"""Selective scan on the GPU against its plain 64-bit form (ssm_reference.py):
packed training sequences with every gradient, packed serving batches with
cache-slot states, token ranges that split sequences, ragged and odd sizes,
strides, rows outside every sequence, CUDA graphs and streams."""
import numpy as np
import pytest
import torch

import ssm_reference as R
from gpu_helpers import DEV, rand, ragged_cu

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
NAMES = ("u", "delta", "A", "B", "C", "skip", "gate", "delta_bias")


def make(T, D, N, F, dtype, seed, options=("skip", "gate", "delta_bias"), ld=0, rate=1.0):
    """Operands with |dt A| up to about 3."""
    g = torch.Generator().manual_seed(seed)
    wide = lambda: rand(g, T, ld or D, dtype=dtype).to(DEV)[:, :D]  # noqa: E731
    bc = rand(g, T, 2 * F * N + (5 if ld else 0), dtype=dtype).to(DEV)
    s = {"u": wide(), "delta": wide() * 0.5 if not ld else wide(),
         "A": -(torch.rand(D, N, generator=g) * 2 * rate + 0.05).to(DEV),
         "B": bc[:, :F * N].unflatten(1, (F, N)) if ld else bc[:, :F * N].reshape(T, F, N),
         "C": bc[:, F * N:2 * F * N].unflatten(1, (F, N)) if ld else bc[:, F * N:2 * F * N].reshape(T, F, N),
         "skip": rand(g, D, dtype=torch.float32).to(DEV), "gate": wide(),
         "delta_bias": (rand(g, D, dtype=torch.float32) - 2).to(DEV)}
    for k in ("skip", "gate", "delta_bias"):
        if k not in options:
            s[k] = None
    return s, rand(g, T, D, dtype=dtype).to(DEV)


def run_train(s, dout, cu, softplus=True):
    from greta_plugin_b200 import selective_scan

    leaf = {k: None if v is None else v.detach().requires_grad_() for k, v in s.items()}
    a = dict(leaf)
    for k in ("u", "delta", "gate"):
        a[k] = None if a[k] is None else a[k][None]
    out = selective_scan(**a, delta_softplus=softplus, cu_seqlens=cu)
    out.backward(dout[None])
    return {"out": out[0].detach(), **{"d" + k: v.grad for k, v in leaf.items() if v is not None}}


def compare(got, val, mag, dtype, longest, tokens, D, F):
    base = 32 * longest + 64
    for k, v in got.items():
        if k in ("dA", "dskip", "ddelta_bias"):
            R.assert_within(v, val[k], mag[k], torch.float32, 2 * base + tokens, k)
        else:
            # a sum over the channels of a group has that many terms
            n = base if k == "out" else 2 * base + (D // F if k in ("dB", "dC") else 0)
            R.assert_within(v, val[k], mag[k], dtype, n, k)


def check_train(lens, D, N, F=1, dtype=torch.float32, seed=0, ranges=0, head=0, tail=0, no_cu=False, softplus=True, **kw):
    from greta_plugin_b200 import _capi

    T = sum(lens) + head + tail
    s, dout = make(T, D, N, F, dtype, seed, **kw)
    if not softplus:
        s["delta"] = (s["delta"].abs() * 0.3).to(dtype)
        if s["delta_bias"] is not None:
            s["delta_bias"] = s["delta_bias"].abs() * 0.01
    cu = None if no_cu else (ragged_cu(lens) + head).to(DEV)
    with _capi.launch_options(rows_ranges=ranges):
        got = run_train(s, dout, cu, softplus)
    val, mag = R.scan(**s, softplus=softplus, cu=None if no_cu else cu.tolist(), dout=dout)
    compare(got, val, mag, dtype, max(lens), T, D, F)
    return got


@pytest.mark.parametrize("N", [1, 3, 4, 5, 8, 12, 16, 17, 32, 33, 64, 100, 128])
def test_train_states(N):
    check_train([20, 1, 35], 48, N, seed=N)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D, F", [(1, 1), (7, 1), (31, 1), (32, 1), (100, 1), (130, 2), (264, 1), (96, 3), (40, 8)])
def test_train_channels_and_groups(dtype, D, F):
    check_train([33, 2, 18], D, 16, F, dtype, seed=D)


@pytest.mark.parametrize("N, D, F", [(64, 40, 1), (64, 96, 2), (128, 24, 2), (20, 72, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_train_wide_states(dtype, N, D, F):
    check_train([33, 2, 18], D, N, F, dtype, seed=N)


@pytest.mark.parametrize("options", [(), ("skip",), ("gate",), ("delta_bias",), ("skip", "gate")])
@pytest.mark.parametrize("softplus", [True, False])
def test_train_options(options, softplus):
    check_train([17, 16, 15], 64, 16, dtype=torch.bfloat16, options=options, softplus=softplus)


@pytest.mark.parametrize("ranges", [1, 2, 3, 5, 16, 40])
@pytest.mark.parametrize("lens", [[200], [90, 1, 109], [1] * 30 + [150, 3], [16, 32, 48, 64], [15, 17, 1, 160]])
def test_train_split_ranges(ranges, lens):
    """Ranges that begin inside sequences carry states and adjoints on."""
    check_train(lens, 40, 16, seed=ranges, ranges=ranges)


@pytest.mark.parametrize("lens", [[24] * 20, [5, 0, 40, 1, 1, 33, 17, 8, 64, 2, 0, 30] * 2, [16] * 31, [9] * 40])
@pytest.mark.parametrize("head, tail", [(0, 0), (13, 21)])
def test_train_whole_sequences(lens, head, tail):
    """Many short sequences and enough channels: ranges of whole sequences, which
    begin inside tiles (up to 31; 40 are cut by position)."""
    check_train(lens, 2048, 16, dtype=torch.bfloat16, head=head, tail=tail)


@pytest.mark.parametrize("ranges", [0, 1, 4])
def test_train_slow_decay_long(ranges):
    """Decay rates of 0.05 to 0.1 a unit step: states that remember hundreds of
    tokens across the ranges."""
    check_train([400, 112], 32, 16, seed=3, ranges=ranges, rate=0.03)


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [31, 0, 1], [0, 0, 5, 0]])
def test_train_short(lens):
    check_train(lens, 32, 16, dtype=torch.bfloat16)


def test_train_no_offsets():
    check_train([77], 32, 16, no_cu=True)


@pytest.mark.parametrize("ranges", [0, 3])
def test_train_rows_outside_give_zeros(ranges):
    head, tail = 21, 40
    got = check_train([30, 9], 32, 16, dtype=torch.bfloat16, head=head, tail=tail, ranges=ranges)
    for k in ("out", "du", "ddelta", "dgate", "dB", "dC"):
        assert not got[k][:head].any() and not got[k][-tail:].any(), k


def test_train_strided():
    check_train([30, 41], 64, 16, dtype=torch.bfloat16, ld=200)
    check_train([30, 41], 61, 9, dtype=torch.float16, ld=131)


@pytest.mark.parametrize("ranges", [1, 3])
def test_train_sequences_do_not_mix(ranges):
    """NaN and inf in a sequence, and in the rows outside, stay there: nothing
    else changes by a bit (dA and the other sums over tokens apart)."""
    from greta_plugin_b200 import _capi

    lens, tail = [25, 14, 50], 9
    s, dout = make(sum(lens) + tail, 32, 16, 1, torch.bfloat16, 5)
    cu = ragged_cu(lens).to(DEV)
    with _capi.launch_options(rows_ranges=ranges):
        clean = run_train(s, dout, cu)
        for k in ("u", "delta", "B", "C", "gate"):
            s[k] = s[k].clone()
            s[k][25:39] = float("nan")
            s[k][-tail:] = float("nan")
        s["u"][30] = float("inf")
        got = run_train(s, dout, cu)
    for k in ("out", "du", "ddelta", "dgate", "dB", "dC"):
        assert torch.equal(got[k][:25], clean[k][:25]) and torch.equal(got[k][39:], clean[k][39:]), k


def test_train_same_call_same_bits_and_int64_offsets():
    s, dout = make(300, 96, 16, 2, torch.bfloat16, 6)
    cu = ragged_cu([100, 1, 199]).to(DEV)
    a = run_train(s, dout, cu)
    for other in (run_train(s, dout, cu), run_train(s, dout, cu.long())):
        assert all(torch.equal(a[k], other[k]) for k in a)


def test_train_masked_steps():
    """Steps of -inf before the softplus are steps of 0: the state stays, and
    the token's own input does not enter."""
    from greta_plugin_b200 import selective_scan

    s, dout = make(40, 32, 16, 1, torch.float32, 7)
    s["delta"][10:20] = float("-inf")
    got = run_train(s, dout, None)
    assert all(torch.isfinite(v).all() for v in got.values())
    assert not got["ddelta"][10:20].any()
    keep = [t for t in range(40) if not 10 <= t < 20]
    cut = {k: v if v is None or v.shape[0] != 40 else v[keep] for k, v in s.items()}
    for k in ("u", "delta", "gate"):
        cut[k] = cut[k][None]
    want = selective_scan(**cut, delta_softplus=True)[0]
    torch.testing.assert_close(got["out"][keep], want, rtol=1e-6, atol=1e-6)


def test_train_large_steps():
    """Steps beyond softplus' linear range and decays that underflow."""
    s, dout = make(40, 32, 16, 1, torch.float32, 8)
    s["delta"] = s["delta"] * 40
    got = run_train(s, dout, None)
    val, mag = R.scan(**s, softplus=True, dout=dout)
    # |dt A| reaches 200: where a decay is above 2^-126 its argument is below
    # 88, of which the step's own error is 88 * 8 roundings a token
    for k in got:
        R.assert_within(got[k], val[k], mag[k], torch.float32, 2 * (40 * 720 + 64), k)


def test_broadcast_operands():
    """A shared by all channels, steps shared by a head: expanded views work and
    their gradients are the sums over what they are shared by."""
    from greta_plugin_b200 import selective_scan

    s, dout = make(50, 64, 16, 1, torch.float32, 9, options=())
    rate = s["A"][:1].clone().requires_grad_()
    step = s["delta"][:, :4].clone().requires_grad_()
    out = selective_scan(s["u"][None], step.repeat_interleave(16, 1)[None], rate.expand(64, 16), s["B"], s["C"],
                         delta_softplus=True)
    out.backward(dout[None])
    s["A"], s["delta"] = rate.detach().expand(64, 16).contiguous(), step.detach().repeat_interleave(16, 1)
    full = run_train(s, dout, None)
    torch.testing.assert_close(rate.grad, full["dA"].sum(0, keepdim=True), rtol=1e-6, atol=1e-5)
    torch.testing.assert_close(step.grad, full["ddelta"].view(50, 4, 16).sum(2), rtol=1e-5, atol=1e-5)


def test_gradients_equal_differences():
    """Directional differences of the kernel's own forward (fp32)."""
    s, dout = make(37, 16, 8, 2, torch.float32, 10)
    cu = ragged_cu([20, 17]).to(DEV)
    got = run_train(s, dout, cu)
    g = torch.Generator().manual_seed(1)
    for name in NAMES:
        v = torch.randn(s[name].shape, generator=g).to(DEV)
        step = 1e-2 / v.norm() * s[name].norm().clamp(min=1)
        side = []
        for sign in (1, -1):
            o = run_train({**s, name: s[name] + sign * step * v}, dout, cu)["out"]
            side.append((o.double() * dout.double()).sum())
        diff = float((side[0] - side[1]) / (2 * step))
        want = float((got["d" + name].double() * v.double()).sum())
        # the third derivative's part is of the order of step^2, the forward's
        # rounding 37 * 16 values of 1e-6 over the step
        assert abs(diff - want) <= 2e-3 * max(abs(want), float(got["d" + name].norm() * v.norm()) * 0.05) + 1e-2, name


def test_train_empty():
    from greta_plugin_b200 import selective_scan

    s, _ = make(0, 32, 16, 1, torch.bfloat16, 0)
    leaf = {k: v.requires_grad_() for k, v in s.items()}
    out = selective_scan(leaf["u"][None], leaf["delta"][None], leaf["A"], leaf["B"], leaf["C"], leaf["skip"],
                         leaf["gate"][None], leaf["delta_bias"], True)
    out.sum().backward()
    assert out.shape == (1, 0, 32) and not leaf["A"].grad.any() and not leaf["skip"].grad.any()


def test_no_gradient_keeps_no_states():
    from greta_plugin_b200 import selective_scan

    s, _ = make(4096, 64, 16, 1, torch.bfloat16, 1)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = selective_scan(s["u"][None], s["delta"][None], s["A"], s["B"], s["C"])
    assert torch.cuda.memory_allocated() - before <= 2 * out.numel() * 2
    assert not out.requires_grad


def test_no_grad_block_makes_no_states():
    """Parameters that take gradients, under no_grad: the states (2 MB) are not
    even made."""
    from greta_plugin_b200 import selective_scan

    s, _ = make(4096, 64, 16, 1, torch.bfloat16, 1)
    A = s["A"].clone().requires_grad_(True)
    selective_scan(s["u"][None], s["delta"][None], s["A"], s["B"], s["C"])
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        out = selective_scan(s["u"][None], s["delta"][None], A, s["B"], s["C"])
    assert torch.cuda.max_memory_allocated() - before < out.numel() * 2 + 513 * 64 * 16 * 4
    assert not out.requires_grad


def test_train_captured():
    """Forward and backward in one captured graph, replayed on new inputs."""
    s, dout = make(150, 64, 16, 1, torch.bfloat16, 11)
    s2, dout2 = make(150, 64, 16, 1, torch.bfloat16, 12)
    cu = ragged_cu([70, 80]).to(DEV)
    want = run_train(s2, dout2, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_train(s, dout, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_train(s, dout, cu)
    for k, v in s2.items():
        s[k].copy_(v)
    dout.copy_(dout2)
    graph.replay()
    assert all(torch.equal(got[k], want[k]) for k in want)


# ---------------------------------------------------------------------------
# packed serving batches
# ---------------------------------------------------------------------------
def make_state(logical, layout):
    n, D, N = logical.shape
    if layout == "rows":
        return logical.to(DEV).contiguous()
    if layout == "transposed":
        return logical.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    big = torch.zeros(n, D * N + 3)
    big[:, :D * N] = logical.reshape(n, -1)
    return big.to(DEV).as_strided((n, D, N), (D * N + 3, N, 1))


def check_packed(lens, slots, init, D, N, F=1, dtype=torch.bfloat16, layout="rows", ranges=0, tail=0, given_out=True,
                 seed=0, softplus=True, **kw):
    from greta_plugin_b200 import _capi, packed_selective_scan

    T = sum(lens) + tail
    s, _ = make(T, D, N, F, dtype, seed, **kw)
    n_slots = max(list(slots) + [0]) + 3
    logical = torch.randn(n_slots, D, N, generator=torch.Generator().manual_seed(seed))
    state = make_state(logical, layout)
    starts = ragged_cu(lens)
    out = torch.full((T, D), 7.0, dtype=dtype, device=DEV) if given_out else None
    with _capi.launch_options(rows_ranges=ranges):
        got = packed_selective_scan(**s, state=state, starts=starts.to(DEV),
                                    slots=torch.tensor(slots, dtype=torch.int32, device=DEV),
                                    has_initial=torch.tensor(init, dtype=torch.int8, device=DEV),
                                    delta_softplus=softplus, out=out)
    before = {i: logical[k].to(DEV) for i, k in enumerate(slots) if k >= 0 and init[i]}
    val, mag = R.scan(**s, softplus=softplus, cu=starts.tolist(), before=before)
    live, base = sum(lens), 32 * max(lens) + 64
    R.assert_within(got[:live], val["out"][:live], mag["out"][:live], dtype, base, "out")
    assert (got[live:] == (7.0 if given_out else 0.0)).all(), "rows behind the last request"
    named = set()
    for i, k in enumerate(slots):
        if k >= 0 and lens[i] > 0:
            named.add(k)
            R.assert_within(state[k], val["last"][i], mag["last"][i], torch.float32, base, f"state of request {i}")
    for k in range(n_slots):
        if k not in named:
            assert torch.equal(state[k].cpu(), logical[k]), f"slot {k} is not of this batch"


LENS, SLOTS, INIT = [1, 1, 1, 2, 40, 0, 3, 129], [3, -1, 7, 0, 5, 8, 2, 9], [1, 1, 0, 1, 0, 1, 1, 1]


@pytest.mark.parametrize("layout", ["rows", "transposed", "generic"])
@pytest.mark.parametrize("N", [5, 16, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_mixed(layout, N, dtype):
    check_packed(LENS, SLOTS, INIT, 72, N, 1, dtype, layout, tail=6, seed=N)


@pytest.mark.parametrize("ranges", [1, 2, 4, 11])
def test_packed_split_ranges(ranges):
    """A request over several ranges starts from its slot although the last
    range writes it; many requests in one range."""
    check_packed(LENS, SLOTS, INIT, 48, 16, 3, torch.float32, ranges=ranges, tail=20)
    check_packed([177], [1], [1], 48, 16, 1, torch.float32, ranges=ranges)
    check_packed([50, 60, 67], [1, 0, 2], [1, 1, 1], 48, 16, 1, torch.float32, ranges=ranges, given_out=False, tail=3)


@pytest.mark.parametrize("n, D, N, F", [(1, 2048, 16, 1), (5, 72, 16, 2), (33, 100, 7, 1), (9, 64, 128, 2), (300, 1024, 16, 1),
                                        (17, 40, 64, 1)])
@pytest.mark.parametrize("layout", ["rows", "transposed"])
def test_packed_decode(n, D, N, F, layout):
    slots = [int(v) for v in np.random.RandomState(n).permutation(n + 2)[:n]]
    init = [1] * n
    if n > 2:
        slots[1], init[2] = -1, 0
    check_packed([1] * n, slots, init, D, N, F, torch.bfloat16, layout)


def test_packed_whole_sequences():
    lens = [33, 2, 40, 0, 17, 64, 1, 50, 50, 8, 31, 60]
    check_packed(lens, list(range(12)), [1, 0] * 6, 2048, 16, tail=9)


def test_packed_decode_uneven():
    """Batches of about a token per request, some of none and of several, rows
    behind the last."""
    check_packed([1, 0, 4, 1, 0, 1], [0, 1, 2, 3, 4, 5], [1] * 6, 64, 16, tail=4)
    check_packed([1, 0, 4, 1, 0, 1], [0, 1, 2, 3, 4, 5], [1] * 6, 64, 16, tail=2, given_out=False)
    check_packed([0, 9], [0, 1], [1, 1], 64, 16)


def test_packed_options_and_strides():
    check_packed(LENS, SLOTS, INIT, 64, 16, options=(), softplus=True)
    check_packed(LENS, SLOTS, INIT, 64, 16, 2, ld=333)
    check_packed([1] * 8, SLOTS, INIT, 64, 16, 2, ld=333)


def test_packed_slot_out_of_range_and_empty():
    from greta_plugin_b200 import packed_selective_scan, packed_selective_scan_checked

    s, _ = make(3, 32, 16, 1, torch.bfloat16, 0)
    state = torch.ones(2, 32, 16, device=DEV)
    for lens in ([1, 2], [3, 0]):
        meta = [torch.tensor(v, dtype=t, device=DEV) for v, t in
                ((np.cumsum([0] + lens).tolist(), torch.int32), ([5, 0], torch.int32), ([1, 1], torch.int8))]
        with pytest.raises(IndexError, match="cache slot"):
            packed_selective_scan_checked(**s, state=state, starts=meta[0], slots=meta[1], has_initial=meta[2])
        assert (state[1] == 1).all()
    none = [torch.zeros(n, dtype=t, device=DEV) for n, t in ((1, torch.int32), (0, torch.int32), (0, torch.int8))]
    out = packed_selective_scan(**s, state=state, starts=none[0], slots=none[1], has_initial=none[2])
    assert not out.any()


def test_packed_continues_like_one_call():
    """A prompt in chunks, then token by token, leaves what one call leaves."""
    from greta_plugin_b200 import packed_selective_scan

    s, _ = make(60, 64, 16, 1, torch.float32, 13)
    one = torch.zeros(1, 64, 16, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    i8 = lambda *v: torch.tensor(v, dtype=torch.int8, device=DEV)  # noqa: E731
    rest = {k: s[k] for k in ("A", "skip", "delta_bias")}
    rows = ("u", "delta", "B", "C", "gate")
    want = packed_selective_scan(**s, state=one, starts=i32(0, 60), slots=i32(0), has_initial=i8(0),
                                 delta_softplus=True)
    state = torch.full((1, 64, 16), 9.0, device=DEV)
    got, at = [], 0
    for n in [20, 33] + [1] * 7:
        part = {k: s[k][at:at + n] for k in rows}
        got.append(packed_selective_scan(**part, **rest, state=state, starts=i32(0, n), slots=i32(0),
                                         has_initial=i8(int(at > 0)), delta_softplus=True))
        at += n
    torch.testing.assert_close(torch.cat(got), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, one, rtol=1e-5, atol=1e-6)


def test_two_captured_graphs_and_streams():
    """Two captured steps (each with its own workspace) and an eager call on a
    third stream, all at once, give what they give alone."""
    from greta_plugin_b200 import _capi, packed_selective_scan

    jobs = []
    for k in range(2):
        s, _ = make(500, 64, 16, 1, torch.bfloat16, 20 + k)
        state = torch.randn(2, 64, 16, device=DEV)
        meta = [torch.tensor(v, dtype=t, device=DEV) for v, t in
                (([0, 230, 500], torch.int32), ([1, 0], torch.int32), ([1, 1], torch.int8))]
        jobs.append((s, state, meta, torch.empty(500, 64, dtype=torch.bfloat16, device=DEV)))

    def call(s, state, meta, out):
        with _capi.launch_options(rows_ranges=6):
            return packed_selective_scan(**s, state=state, starts=meta[0], slots=meta[1], has_initial=meta[2],
                                         delta_softplus=True, out=out)

    want, graphs = [], []
    for s, state, meta, out in jobs:
        keep = state.clone()
        want.append((call(s, keep, meta, torch.empty_like(out)), keep))
    for s, state, meta, out in jobs:
        first = state.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(s, state, meta, out)
        state.copy_(first)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for g, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    with torch.cuda.stream(streams[2]):
        s, dout = make(300, 64, 16, 1, torch.bfloat16, 30)
        streams[2].synchronize()
        eager = run_train(s, dout, None)
    torch.cuda.synchronize()
    for (_, state, _, out), (o, st) in zip(jobs, want):
        assert torch.equal(out, o) and torch.equal(state, st)
    again = run_train(*make(300, 64, 16, 1, torch.bfloat16, 30), None)
    assert all(torch.equal(eager[k], again[k]) for k in again)


def test_far_rows_and_slots():
    """Rows and slots more than 2^31 elements apart give the near ones' bits."""
    from greta_plugin_b200 import packed_selective_scan

    lens, D, N = [9, 1, 1, 6], 64, 16
    s, _ = make(sum(lens), D, N, 1, torch.bfloat16, 21)
    starts, ld = ragged_cu(lens).to(DEV), 2 ** 28 + 8
    slots = torch.tensor([1, 0, -1, 2], dtype=torch.int32, device=DEV)
    init = torch.ones(4, dtype=torch.int8, device=DEV)
    state = torch.randn(3, D, N, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    far = torch.empty(2 * (2 ** 30 + 64) + D * N, device=DEV).as_strided((3, D, N), (2 ** 30 + 64, N, 1))
    far.copy_(state)
    rows = torch.empty(16 * ld + D, dtype=torch.bfloat16, device=DEV).as_strided((17, D), (ld, 1))
    rows.copy_(s["u"])
    for single in (False, True):  # the prompts' kernels, then the single tokens'
        if single:
            starts, slots, init = starts[:0].new_tensor([0, 1, 2, 3]), slots[[0, 1, 3]].contiguous(), init[:3]
            rows = rows[13:16]
            s = {k: v[13:16] if v.shape[0] == 17 else v for k, v in s.items()}
        want = packed_selective_scan(**s, state=state, starts=starts, slots=slots, has_initial=init)
        got = packed_selective_scan(**{**s, "u": rows}, state=far, starts=starts, slots=slots, has_initial=init)
        # (bits: without softplus some of these steps grow past what the type holds)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
        assert torch.equal(far.contiguous().view(torch.int32), state.view(torch.int32))
