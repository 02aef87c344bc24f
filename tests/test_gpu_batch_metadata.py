"""packed_batch_metadata on the GPU against a request-by-request host form, and
the serving operators run together from it: metadata, convolution, scan, for
prompts in chunks and single tokens, against one training call."""
import numpy as np
import pytest
import torch

import ssm_reference as R
from gpu_helpers import DEV, rand

pytestmark = pytest.mark.gpu


def host_metadata(query, context, T, tables=None, bs=0, free=None):
    """Request by request, in Python integers."""
    starts, init, seq, pos, slot, used = [0], [], [-1] * T, [0] * T, [-1] * T, 0
    tables = None if tables is None else [list(r) for r in tables]
    at = 0
    for i, (q, c) in enumerate(zip(query, context)):
        q, c = max(q, 0), max(c, 0)
        init.append(int(c > 0))
        if tables is not None:
            for b in range(-(-c // bs), -(-(c + q) // bs)):
                first_token = at + b * bs - c
                if b < len(tables[i]) and first_token < T:
                    tables[i][b] = free[used] if used < len(free) else -1
                used += 1
        for k in range(q):
            if at < T:
                seq[at], pos[at] = i, c + k
                if tables is not None and (c + k) // bs < len(tables[i]):
                    blk = tables[i][(c + k) // bs]
                    slot[at] = blk * bs + (c + k) % bs if blk >= 0 else -1
            at += 1
        starts.append(min(at, T))
    return starts, init, seq, pos, slot, used, tables


def check(query, context, T, bs=0, width=0, nfree=0, seed=0, pad_rows=0):
    from greta_plugin_b200 import packed_batch_metadata

    rng = np.random.RandomState(seed)
    N = len(query)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    if not bs:
        m = packed_batch_metadata(i32(query), i32(context), T)
        want = host_metadata(query, context, T)
        assert m.slot_map is None and m.blocks_used is None
    else:
        ids = rng.permutation(N * width + nfree).astype(np.int32)
        table = ids[:N * width].reshape(N, width)
        free = ids[N * width:].tolist()
        big = torch.full((N, width + pad_rows), -7, dtype=torch.int32, device=DEV)
        big[:, :width] = torch.from_numpy(table).to(DEV)
        m = packed_batch_metadata(i32(query), i32(context), T, big[:, :width], bs, i32(free))
        want = host_metadata(query, context, T, table.tolist(), bs, free)
        assert m.slot_map.tolist() == want[4]
        assert m.blocks_used.tolist() == [want[5]]
        assert big[:, :width].tolist() == want[6]
        assert (big[:, width:] == -7).all()
    assert m.starts.tolist() == want[0] and m.starts.dtype == torch.int32
    assert m.has_initial.tolist() == want[1] and m.has_initial.dtype == torch.int8
    assert m.seq_idx.tolist() == want[2] and m.seq_idx.dtype == torch.int32
    assert m.positions.tolist() == want[3] and m.positions.dtype == torch.int64
    return m


@pytest.mark.parametrize("bs", [0, 1, 16, 100])
def test_small_batches(bs):
    check([1], [0], 1, bs, 8, 4)
    check([0], [5], 3, bs, 8, 4)
    check([3, 0, 0, 5, 1], [0, 7, 0, 31, 2], 12, bs, 40, 50, pad_rows=3)
    check([0, 0], [0, 0], 0, bs, 4, 4)
    check([-3, 4], [2, -9], 6, bs, 40, 50)


@pytest.mark.parametrize("N", [31, 32, 33, 511, 512, 513, 1500])
def test_many_requests(N):
    rng = np.random.RandomState(N)
    query = rng.randint(0, 4, N).tolist()
    context = rng.randint(0, 300, N).tolist()
    check(query, context, sum(query) + 9, 16, 20, sum(query) + N, seed=N)


def test_largest_batch():
    check([1] * 16384, list(range(16384)), 16384, 64, 257, 16384)


def test_list_runs_out_and_table_too_narrow():
    check([40, 40, 40], [10, 0, 3], 120, 16, 8, 4)  # 8 blocks asked for, 4 there
    check([40, 40, 40], [10, 0, 3], 120, 16, 2, 12)  # tables of two blocks
    check([40, 40], [10, 0], 80, 16, 8, 0)  # an empty list
    check([40, 40], [10, 0], 80, 16, 0, 9)  # tables of no block


def test_more_tokens_than_rows():
    m = check([10, 20, 30], [5, 0, 100], 25, 16, 20, 30)
    assert m.starts.tolist() == [0, 10, 25, 25]


def test_far_positions():
    """Slots past 2^31: a large pool of large blocks."""
    from greta_plugin_b200 import packed_batch_metadata

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    table = i32(2 ** 31 - 1, 5).view(1, 2)
    m = packed_batch_metadata(i32(3), i32(4094), 3, table, 4096, i32(2 ** 31 - 2))
    base = (2 ** 31 - 1) * 4096
    assert m.slot_map.tolist() == [base + 4094, base + 4095, (2 ** 31 - 2) * 4096]
    assert table.tolist() == [[2 ** 31 - 1, 2 ** 31 - 2]]


def test_captured_with_changing_lengths():
    from greta_plugin_b200 import packed_batch_metadata

    q = torch.ones(8, dtype=torch.int32, device=DEV)
    c = torch.arange(8, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = packed_batch_metadata(q, c, 16)
    for query in ([1] * 8, [0, 3, 0, 2, 1, 0, 0, 10], [2] * 8):
        q.copy_(torch.tensor(query))
        graph.replay()
        want = host_metadata(query, list(range(8)), 16)
        assert m.starts.tolist() == want[0] and m.seq_idx.tolist() == want[2] and m.positions.tolist() == want[3]


def test_serving_steps_equal_one_training_call():
    """Three requests served in steps of mixed prompts chunks and single tokens,
    from lengths on the device (metadata -> convolution -> scan, cache slots
    between the steps), give what the training operators give on the whole
    sequences at once."""
    import greta_plugin_b200 as greta

    D, N, W, total = 64, 16, 4, [70, 23, 41]
    g = torch.Generator().manual_seed(0)
    f32 = torch.float32
    seqs = [{k: rand(g, n, *s, dtype=f32).to(DEV) for k, s in
             (("x", (D,)), ("delta", (D,)), ("gate", (D,)), ("B", (1, N)), ("C", (1, N)))} for n in total]
    w, b = rand(g, W, D, scale=0.5, dtype=f32).to(DEV), rand(g, D, dtype=f32).to(DEV)
    A = -(torch.rand(D, N, generator=g) * 2 + 0.05).to(DEV)
    skip, bias = rand(g, D, dtype=f32).to(DEV), (rand(g, D, dtype=f32) - 2).to(DEV)

    cu = torch.tensor(np.cumsum([0] + total), dtype=torch.int32, device=DEV)
    whole = {k: torch.cat([s[k] for s in seqs]) for k in seqs[0]}
    u = greta.causal_conv1d(whole["x"][None], w, b, cu, "silu")
    want = greta.selective_scan(u, whole["delta"][None], A, whole["B"], whole["C"], skip, whole["gate"][None], bias,
                                True, cu)[0]

    conv_state = torch.full((5, D, W - 1), 3.0, device=DEV)
    scan_state = torch.full((5, D, N), 3.0, device=DEV)
    tables = torch.full((3, 8), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(40, 70, dtype=torch.int32, device=DEV)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
    context, got, taken, seen = [0, 0, 0], [[], [], []], 0, set()
    for step in ([20, 0, 9], [30, 1, 1], [1, 20, 1], [18, 1, 0], [1, 1, 30]):
        step = [min(n, total[i] - context[i]) for i, n in enumerate(step)]
        T = sum(step) + 3  # three rows of padding
        rows = {k: torch.cat([s[k][c:c + n] for s, c, n in zip(seqs, context, step)] + [whole[k][:3] * float("nan")])
                for k in whole}
        m = greta.packed_batch_metadata(torch.tensor(step, dtype=torch.int32, device=DEV),
                                        torch.tensor(context, dtype=torch.int32, device=DEV), T, tables, 16,
                                        free[taken:])
        taken += int(m.blocks_used)
        live = m.slot_map[m.slot_map >= 0].tolist()
        assert len(live) == sum(step) and not seen & set(live)  # every token its own place
        seen |= set(live)
        xc = greta.packed_causal_conv1d(rows["x"], w, b, conv_state, m.starts, slots, m.has_initial, "silu")
        y = greta.packed_selective_scan(xc, rows["delta"], A, rows["B"], rows["C"], skip, rows["gate"], bias,
                                        scan_state, m.starts, slots, m.has_initial, True)
        assert not y[sum(step):].any()
        at = 0
        for i, n in enumerate(step):
            got[i].append(y[at:at + n])
            at += n
            context[i] += n
    assert context == total
    got = torch.cat([torch.cat(v) for v in got])
    # both are within 32 roundings a token of the same sums
    val, mag = R.scan(u[0], whole["delta"], A, whole["B"], whole["C"], skip, whole["gate"], bias, True, cu.tolist())
    n = 32 * max(total) + 64
    R.assert_within(want, val["out"], mag["out"], f32, n, "training")
    # u itself differs by its own few roundings between the two
    R.assert_within(got, val["out"], mag["out"], f32, n + W + 8, "serving")
