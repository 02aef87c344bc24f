"""Short causal convolution on the GPU against its plain 64-bit form
(ssm_reference.py): packed training sequences with gradients, packed serving
batches with cache-slot state (bit-exact), ragged and odd sizes, strides, rows
outside every sequence, CUDA graphs."""
import numpy as np
import pytest
import torch

import ssm_reference as R
from gpu_helpers import DEV, rand, ragged_cu

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _train(x, w, b, cu, silu, dout):
    from greta_plugin_b200 import causal_conv1d

    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    lb = None if b is None else b.detach().requires_grad_()
    out = causal_conv1d(lx[None], lw, lb, cu, "silu" if silu else None)
    out.backward(dout[None])
    return out[0], lx.grad, lw.grad, None if b is None else lb.grad


def check_train(lens, D, W, dtype, silu=True, bias=True, seed=0, head=0, tail=0, transposed=False, ld=0, no_cu=False):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + head + tail
    x = rand(g, T, ld or D, dtype=dtype).to(DEV)[:, :D]
    w = rand(g, W, D, scale=W ** -0.5, dtype=dtype).to(DEV)
    if transposed:
        w = w.t().contiguous().t()
    b = rand(g, D, dtype=dtype).to(DEV) if bias else None
    dout = rand(g, T, D, dtype=dtype).to(DEV)
    cu = None if no_cu else (ragged_cu(lens) + head).to(DEV)
    got = _train(x, w, b, cu, silu, dout)
    val, mag = R.conv(x, w, b, silu, cu=None if no_cu else cu.tolist(), dout=dout)
    n = W + 8
    R.assert_within(got[0], val["out"], mag["out"], dtype, n, "out")
    # the sigmoid's few ulp and dpre's products again, then the taps
    R.assert_within(got[1], val["dx"], mag["dx"], dtype, 2 * n, "dx")
    R.assert_within(got[2], val["dw"], mag["dw"], dtype, 2 * n + T, "dw")
    if bias:
        R.assert_within(got[3], val["dbias"], mag["dbias"], dtype, 2 * n + T, "dbias")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 9, 16])
def test_train_widths(dtype, W):
    check_train([1, 2, W, 40, 3, 129], 256, W, dtype, seed=W)


@pytest.mark.parametrize("D", [1, 7, 8, 20, 100, 264, 1000])
@pytest.mark.parametrize("dtype", TYPES)
def test_train_channels(dtype, D):
    check_train([65, 1, 30], D, 4, dtype, seed=D)


@pytest.mark.parametrize("silu, bias", [(False, False), (False, True), (True, False)])
def test_train_options(silu, bias):
    check_train([5, 0, 17, 0, 0, 1], 64, 4, torch.bfloat16, silu, bias)


def test_train_one_sequence_and_one_token():
    check_train([300], 512, 4, torch.bfloat16, no_cu=True)
    check_train([1], 64, 4, torch.float32, no_cu=True)


def test_train_many_short_sequences():
    check_train([1] * 300 + [2] * 100 + [0] * 70 + [3] * 50, 128, 4, torch.float16)


def test_train_strided_rows_and_transposed_weight():
    check_train([40, 3, 61], 256, 4, torch.bfloat16, ld=512, transposed=True)
    check_train([40, 3, 61], 99, 3, torch.bfloat16, ld=201, transposed=True)
    check_train([40, 3, 61], 256, 4, torch.float32, ld=264)


@pytest.mark.parametrize("D", [64, 63])
def test_train_rows_outside_give_zeros(D):
    head, tail = 5, 21
    out, dx, _, _ = check_train([9, 30], D, 4, torch.bfloat16, head=head, tail=tail)
    for t in (out, dx):
        assert not t[:head].any() and not t[-tail:].any()


def test_train_large_runs():
    """Long enough for several blocks of long runs, and the partial sums of dw."""
    check_train([1500, 1, 2596], 2048, 4, torch.bfloat16, seed=9)


def test_train_empty():
    from greta_plugin_b200 import causal_conv1d

    x = torch.zeros(1, 0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(4, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out = causal_conv1d(x, w, b, torch.zeros(3, dtype=torch.int32, device=DEV), "silu")
    out.sum().backward()
    assert out.shape == (1, 0, 64) and not w.grad.any() and not b.grad.any()


def test_train_sequences_do_not_mix():
    """NaN and inf in one sequence reach no other sequence's outputs or dx."""
    g = torch.Generator().manual_seed(4)
    lens = [20, 7, 33]
    x, w, b, dout = (rand(g, *s).to(DEV) for s in ((60, 64), (4, 64), (64,), (60, 64)))
    cu = ragged_cu(lens).to(DEV)
    clean = _train(x, w, b, cu, True, dout)
    bad = x.clone()
    bad[20:27] = float("nan")
    bad[22] = float("inf")
    got = _train(bad, w, b, cu, True, dout)
    for i in (0, 1):
        assert torch.equal(got[i][:20], clean[i][:20]) and torch.equal(got[i][27:], clean[i][27:])


def test_train_same_call_same_bits_and_int64_offsets():
    g = torch.Generator().manual_seed(5)
    x, w, b, dout = (rand(g, *s).to(DEV) for s in ((700, 320), (4, 320), (320,), (700, 320)))
    cu = ragged_cu([300, 1, 399]).to(DEV)
    a = _train(x, w, b, cu, True, dout)
    for other in (_train(x, w, b, cu, True, dout), _train(x, w, b, cu.long(), True, dout)):
        assert all(torch.equal(p, q) for p, q in zip(a, other))


def test_train_mixed_parameter_types():
    """fp32 weights beside bf16 activations: used in bf16, gradients in fp32."""
    from greta_plugin_b200 import causal_conv1d

    g = torch.Generator().manual_seed(6)
    x = rand(g, 1, 50, 64).to(DEV)
    w = rand(g, 4, 64).to(DEV).float().requires_grad_()
    causal_conv1d(x, w).sum().backward()
    assert w.grad.dtype == torch.float32


# ---------------------------------------------------------------------------
# packed serving batches
# ---------------------------------------------------------------------------
def make_state(logical, layout):
    n, D, H = logical.shape
    if layout == "DS":
        return logical.to(DEV).contiguous()
    if layout == "SD":
        return logical.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    big = torch.zeros(n, D * H + 5, dtype=logical.dtype)
    big[:, :D * H] = logical.reshape(n, -1)
    return big.to(DEV).as_strided((n, D, H), (D * H + 5, H, 1))


def check_packed(lens, slots, init, D, W, dtype, layout="DS", tail=0, given_out=True, ld=0, silu=True, seed=0):
    from greta_plugin_b200 import packed_causal_conv1d

    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    n_slots = max([s for s in slots] + [0]) + 3
    x = rand(g, T, ld or D, dtype=dtype).to(DEV)[:, :D]
    w, b = rand(g, W, D, scale=W ** -0.5, dtype=dtype).to(DEV), rand(g, D, dtype=dtype).to(DEV)
    logical = rand(g, n_slots, D, W - 1, dtype=dtype)
    state = make_state(logical, layout)
    starts = ragged_cu(lens)
    out = torch.full((T, D), 7.0, dtype=dtype, device=DEV) if given_out else None
    got = packed_causal_conv1d(x, w, b, state, starts.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV),
                               torch.tensor(init, dtype=torch.int8, device=DEV), "silu" if silu else None, out)
    hist = {i: logical[s].t().to(DEV) for i, s in enumerate(slots) if s >= 0 and init[i]}
    val, mag = R.conv(x, w, b, silu, cu=starts.tolist(), history=hist)
    live = sum(lens)
    R.assert_within(got[:live], val["out"][:live], mag["out"][:live], dtype, W + 8, "out")
    assert (got[live:] == (7.0 if given_out else 0.0)).all(), "rows behind the last request"
    want = logical.clone()
    for i, s in enumerate(slots):
        if s >= 0 and lens[i] > 0 and W > 1:
            past = logical[s] if init[i] else torch.zeros_like(logical[s])
            rows = x[int(starts[i]):int(starts[i + 1])].t().cpu()
            want[s] = torch.cat([past, rows], 1)[:, 1 - W:]
    assert torch.equal(state.cpu(), want), "state must be bit-exact"


@pytest.mark.parametrize("layout", ["DS", "SD", "generic"])
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 7, 16])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_mixed(layout, W, dtype):
    check_packed([1, 1, 1, 2, W, 40, 0, 3, 129], [3, -1, 7, 0, 11, 5, 8, 2, 9], [1, 1, 0, 1, 1, 0, 1, 1, 1], 256, W,
                 dtype, layout, tail=6, seed=W)


@pytest.mark.parametrize("D", [1, 9, 24, 100, 520])
@pytest.mark.parametrize("layout", ["DS", "SD"])
def test_packed_channels(D, layout):
    check_packed([1, 30, 2, 1], [2, 0, 1, -1], [1, 1, 0, 1], D, 4, torch.bfloat16, layout, given_out=False, tail=3)


@pytest.mark.parametrize("n, D", [(1, 2048), (256, 512), (3, 64)])
def test_packed_decode(n, D):
    slots = list(np.random.RandomState(n).permutation(n + 2)[:n])
    check_packed([1] * n, [int(s) for s in slots], [1] * n, D, 4, torch.bfloat16)


def test_packed_decode_uneven():
    """Batches of about a token per request, some of none and of several, rows
    behind the last."""
    for kw in (dict(tail=4), dict(tail=2, given_out=False), dict(tail=0)):
        check_packed([1, 0, 4, 1, 0, 1], [0, 1, 2, 3, 4, 5], [1, 1, 1, 0, 1, 1], 64, 4, torch.bfloat16, **kw)
    check_packed([0, 9], [0, 1], [1, 1], 65, 3, torch.float32)
    check_packed([3, 1, 1], [2, 0, -1], [1, 1, 1], 64, 7, torch.float16, layout="SD")


@pytest.mark.parametrize("extra", [0, 1, 2, 3, 5])
def test_packed_borders_of_runs(extra):
    """Sequence starts at every offset from where one run of tokens ends and the
    next begins: the first W-1 tokens of a request stay with one run."""
    for D in (8, 512):
        check_packed([13 + extra, 3, 2, 1, 60, 1, 1, 47, 2, 300], list(range(10)), [1] * 10, D, 4, torch.float32)


def test_packed_long_and_strided():
    check_packed([2000, 1, 700], [1, 0, 2], [1, 1, 0], 1024, 4, torch.bfloat16, ld=2056)
    check_packed([50, 1, 70], [1, 0, 2], [1, 1, 0], 101, 3, torch.float16, ld=203, silu=False)


@pytest.mark.parametrize("W", [4, 7])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_state_keeps_bits(W, dtype):
    """Every 16-bit pattern, NaN payloads among them, goes into the slots as it
    is: from short requests, ones inside a run and ones over several."""
    from greta_plugin_b200 import packed_causal_conv1d

    lens, D = [1, 2, 5, 200, 1], 512
    g = torch.Generator().manual_seed(W)
    bits = lambda *s: torch.randint(-2 ** 15, 2 ** 15, s, generator=g).to(torch.int16).to(DEV).view(dtype)  # noqa: E731
    x, state = bits(sum(lens), D), bits(6, D, W - 1)
    want, starts = state.clone().view(torch.int16), ragged_cu(lens)
    slots, init = [3, 0, 5, 1, 2], [1, 1, 0, 1, 0]
    for i, k in enumerate(slots):
        past = want[k] if init[i] else torch.zeros_like(want[k])
        rows = x[int(starts[i]):int(starts[i + 1])].view(torch.int16).t()
        want[k] = torch.cat([past, rows], 1)[:, 1 - W:]
    packed_causal_conv1d(x, torch.zeros(W, D, dtype=dtype, device=DEV), None, state, starts.to(DEV),
                         torch.tensor(slots, dtype=torch.int32, device=DEV),
                         torch.tensor(init, dtype=torch.int8, device=DEV))
    assert torch.equal(state.view(torch.int16), want)


def test_packed_slot_out_of_range():
    from greta_plugin_b200 import packed_causal_conv1d_checked

    x = torch.ones(3, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(4, 64, device=DEV, dtype=torch.bfloat16)
    state = torch.ones(2, 64, 3, device=DEV, dtype=torch.bfloat16)
    meta = [torch.tensor(v, dtype=t, device=DEV) for v, t in
            (([0, 1, 3], torch.int32), ([0, 5], torch.int32), ([1, 1], torch.int8))]
    with pytest.raises(IndexError, match="cache slot"):
        packed_causal_conv1d_checked(x, w, None, state, *meta)
    assert (state[1] == 1).all()


def test_packed_no_requests_and_no_tokens():
    from greta_plugin_b200 import packed_causal_conv1d

    x = torch.ones(3, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(4, 64, device=DEV, dtype=torch.bfloat16)
    state = torch.ones(2, 64, 3, device=DEV, dtype=torch.bfloat16)
    none = [torch.zeros(n, dtype=t, device=DEV) for n, t in ((1, torch.int32), (0, torch.int32), (0, torch.int8))]
    assert not packed_causal_conv1d(x, w, None, state, *none).any()
    assert packed_causal_conv1d(x[:0], w, None, state, *none).shape == (0, 64)
    assert (state == 1).all()


def test_packed_captured():
    """A captured decode step, replayed on new inputs, equals eager calls."""
    from greta_plugin_b200 import packed_causal_conv1d

    g = torch.Generator().manual_seed(8)
    n, D = 16, 256
    xs = [rand(g, n, D).to(DEV) for _ in range(4)]
    w, b = rand(g, 4, D).to(DEV), rand(g, D).to(DEV)
    start = rand(g, n, D, 3).to(DEV)
    meta = (torch.arange(n + 1, dtype=torch.int32, device=DEV), torch.randperm(n, generator=g).to(torch.int32).to(DEV),
            torch.ones(n, dtype=torch.int8, device=DEV))
    state = start.clone()
    want = [packed_causal_conv1d(x, w, b, state, *meta, "silu").clone() for x in xs]
    ref = state.clone()
    state.copy_(start)
    x, out = xs[0].clone(), torch.empty(n, D, dtype=torch.bfloat16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed_causal_conv1d(x, w, b, state, *meta, "silu", out)
    for k, v in enumerate(xs):
        x.copy_(v)
        graph.replay()
        assert torch.equal(out, want[k])
    assert torch.equal(state, ref)


def test_far_rows_and_slots():
    """Rows and slots more than 2^31 elements apart give the near ones' bits."""
    from greta_plugin_b200 import causal_conv1d, packed_causal_conv1d

    lens, D, W = [9, 1, 1, 6], 64, 4
    g = torch.Generator().manual_seed(22)
    T, ld = sum(lens), 2 ** 28 + 8
    x = rand(g, T, D, dtype=torch.bfloat16).to(DEV)
    w, b = rand(g, W, D, dtype=torch.bfloat16).to(DEV), rand(g, D, dtype=torch.bfloat16).to(DEV)
    far_x = torch.empty((T - 1) * ld + D, dtype=torch.bfloat16, device=DEV).as_strided((T, D), (ld, 1))
    far_x.copy_(x)
    state = rand(g, 3, D, W - 1, dtype=torch.bfloat16).to(DEV)
    far = torch.empty(2 * (2 ** 30 + 64) + D * 3, dtype=torch.bfloat16, device=DEV).as_strided(
        (3, D, W - 1), (2 ** 30 + 64, W - 1, 1))
    far.copy_(state)
    starts = ragged_cu(lens).to(DEV)
    slots = torch.tensor([1, 0, -1, 2], dtype=torch.int32, device=DEV)
    init = torch.ones(4, dtype=torch.int8, device=DEV)
    cu, dout = starts, rand(g, 1, T, D, dtype=torch.bfloat16).to(DEV)
    near = [t.detach().requires_grad_() for t in (x, w, b)]
    wide = [t.detach().requires_grad_() for t in (far_x, w, b)]
    outs = [causal_conv1d(t[0][None], t[1], t[2], cu, "silu") for t in (near, wide)]
    assert torch.equal(*outs)
    grads = [torch.autograd.grad(o, t[1:], dout) for o, t in zip(outs, (near, wide))]
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    for single in (False, True):  # the prompts' kernel, then the single tokens'
        if single:
            starts, slots, init = starts[:0].new_tensor([0, 1, 2, 3]), slots[[0, 1, 3]].contiguous(), init[:3]
            x, far_x = x[13:16], far_x[13:16]
        want = packed_causal_conv1d(x, w, b, state, starts, slots, init, "silu")
        got = packed_causal_conv1d(far_x, w, b, far, starts, slots, init, "silu")
        assert torch.equal(got, want) and torch.equal(far, state)
