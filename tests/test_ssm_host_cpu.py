"""Host side of the state-space operators without a GPU: what a call sets, asks
for and passes on. Kernels do not run: launches go to a stand-in for the CUDA
runtime's functions in a child process, or the C call is recorded."""
import importlib
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent

# What the library asks the CUDA runtime for, printed: attribute changes and
# launches (dynamic shared memory, blocks).
RUNTIME = r"""
#include <stdio.h>
#include <stddef.h>
typedef struct { unsigned gx, gy, gz, bx, by, bz; size_t smem; } Config;
int cudaFuncSetAttribute(const void* f, int attr, int value) {
  printf("set %d %d\n", attr, value);
  fflush(stdout);
  return 0;
}
int cudaLaunchKernelExC(const Config* c, const void* f, void** args) {
  printf("launch %zu %u %u\n", c->smem, c->gx, c->gy);
  fflush(stdout);
  return 0;
}
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    d = tmp_path_factory.mktemp("runtime")
    (d / "runtime.c").write_text(RUNTIME)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", d / "runtime.so", d / "runtime.c"], check=True)
    return d / "runtime.so"


def recorded(runtime, code):
    """Lines that the stand-in printed while `code` ran with the library as L."""
    setup = "import ctypes; from greta_plugin_b200 import _capi; L = _capi.lib(); F = ctypes.c_void_p(0x1000)\n"
    env = {**os.environ, "LD_PRELOAD": str(runtime), "PYTHONPATH": str(ROOT)}
    out = subprocess.run([sys.executable, "-c", setup + code], env=env, capture_output=True, text=True, check=True)
    return [line.split() for line in out.stdout.splitlines()]


def test_metadata_calls_do_not_lower_each_others_limit(runtime):
    """Two host threads with batches of different sizes: the shared memory that
    one allows its launch may not be taken back by the other's call."""
    lines = recorded(runtime, "for n in (16384, 8000, 100, 16384, 7000):\n"
                     "    assert L.greta_ssm_batch_metadata(F, F, n, 8, F, F, F, F, None, 0, 0, 0, None, 0, None, None,\n"
                     "                                      None) == 0")
    limits = {int(v[2]) for v in lines if v[0] == "set"}
    launches = [int(v[1]) for v in lines if v[0] == "launch"]
    assert len(launches) == 5
    assert len(limits) == 1 and limits.pop() >= max(launches)


def test_token_ranges_of_a_training_call_reach_its_backward(monkeypatch):
    """launch_options holds for the calls that are made inside its block; the
    backward of such a call runs on autograd's thread, and maybe behind it."""
    from greta_plugin_b200 import _capi

    module = importlib.import_module("greta_plugin_b200.selective_scan")  # (the package has the function's name)
    seen = []
    monkeypatch.setattr(module, "_workspace", lambda kind, dev, nseq, T, D, N, F, ranges: (None, 0))
    monkeypatch.setattr(_capi, "call", lambda name, t, *a: seen.append((name, a[-3])))  # ranges, workspace, bytes
    u = torch.zeros(1, 20, 8, requires_grad=True)
    B = torch.zeros(20, 1, 4)
    with _capi.launch_options(rows_ranges=5):
        out = module.SelectiveScanFunction.apply(u, u, -torch.ones(8, 4), B, B, None, None, None, None, True, True)
    out.backward(torch.ones_like(out))
    assert seen == [("greta_ssm_scan_fwd", 5), ("greta_ssm_scan_bwd", 5)]


def test_request_tensors_of_other_types_keep_their_meaning():
    """A count as has_initial, and offsets and slots past 32 bits: not the numbers
    that their low bits make."""
    from greta_plugin_b200.causal_conv import packed_metadata

    x, state = torch.zeros(5, 8), torch.zeros(4, 8, 3)
    starts = torch.tensor([0, 2, 2 ** 32 + 1], dtype=torch.int64)
    slots = torch.tensor([2 ** 32 + 3, -(2 ** 32) + 1], dtype=torch.int64)
    for init in (torch.tensor([256, 0]), torch.tensor([512, 0], dtype=torch.int32), torch.tensor([True, False]),
                 torch.tensor([0.5, 0.0])):
        st, sl, has = packed_metadata(x, state, starts, slots, init)
        assert has.dtype == torch.int8 and (has != 0).tolist() == [True, False]
    assert st.dtype == sl.dtype == torch.int32
    assert st.tolist() == [0, 2, 2 ** 31 - 1]
    assert sl[0] >= 4 and sl[1] < 0  # out of range, and none
    st, sl, _ = packed_metadata(x, state, starts.new_tensor([0, 2, 5]), slots.new_tensor([3, -1]), init)
    assert st.tolist() == [0, 2, 5] and sl.tolist() == [3, -1]


def test_complex_parameters_are_refused():
    """Their imaginary parts would be dropped. (Where they are converted, so that
    no other call pays for the test.)"""
    from greta_plugin_b200.causal_conv import _as_type, _bias
    from greta_plugin_b200.selective_scan import _fp32

    z = torch.zeros(8, dtype=torch.complex64)
    for convert in (_fp32, lambda t: _as_type(t, torch.bfloat16), lambda t: _bias(t, torch.float32)):
        with pytest.raises(ValueError, match="must be real"):
            convert(z)
        assert convert(torch.ones(8, dtype=torch.float64)).tolist() == [1.0] * 8


def test_conv_backward_workspace_holds_the_launch_and_little_more(runtime):
    """The workspace is what the launch's blocks write: a row of partial sums for
    every block of runs, not for the shortest runs that there could be."""
    shapes = [(T, D, W, dt) for T, D in ((1, 64), (9, 1), (300, 1000), (1531, 1001), (16288, 4096), (131072, 8192))
              for W in (1, 2, 4, 8, 16) for dt in (0, 1, 2)]
    lines = recorded(runtime, f"for T, D, W, dt in {shapes}:\n"
                     "    n = L.greta_ssm_conv_bwd_workspace(T, D, W)\n"
                     "    print('bytes', n, flush=True)\n"
                     "    assert L.greta_ssm_conv_bwd(dt, F, D, F, D, 1, None, F, F, F, None, None, 0, 0, T, D, W, 0, F, n,\n"
                     "                                None) == 0")
    lines = [v for v in lines if v[0] != "set"]
    assert len(lines) == 3 * len(shapes)  # (the second launch adds the rows up)
    for (T, D, W, dt), (_, n), (_, _, blocks, _) in zip(shapes, lines[::3], lines[1::3]):
        whole = 4 if dt and 2 <= W <= 4 else 2 if dt or W <= 8 else 1  # channels of a vector
        vec = whole if D % whole == 0 else 1
        rows = int(blocks) // -(-(-(-D // vec)) // 32)
        wrote = rows * (W + 1) * D * 4
        # (a grid of as many blocks has up to four times the rows with vectors of four
        # channels that it has with one, and a row more by rounding)
        assert wrote <= int(n) <= 5 * wrote, (T, D, W, dt)


def test_a_long_request_beside_empty_ones_is_no_decode_step(runtime):
    """A table of 256 requests with one prompt has the rows of 256 single tokens;
    where the host knows the longest request, the choice of the kernels goes by it."""
    lines = recorded(runtime, """
for T, n, most in ((256, 256, 0), (256, 256, 1), (256, 256, 256), (300, 256, 1), (10, 4, 7), (10, 4, 40)):
    flag = most << 8
    need = L.greta_ssm_scan_workspace(1 | flag, n, T, 4096, 16, 1, 0)
    print("bytes", need, flush=True)
    assert L.greta_ssm_scan_packed(2, F, 4096, F, 4096, None, 0, F, 16, F, 16, F, None, None, F, F, n, 65536, 16, 1, F,
                                   F, F, n, T, 4096, 16, 1, 0, 1 | flag, 0, None, F, need, None) == 0
    assert L.greta_ssm_conv_packed(2, F, 4096, F, 4096, 1, None, F, F, n, 12288, 3, 1, F, F, F, n, T, 4096, 4, 0,
                                   1 | flag, None, None) == 0
    print("end", flush=True)
""")
    lines = [v for v in lines if v[0] != "set"]
    calls, at = [], 0
    for _ in range(6):
        end = lines.index(["end"], at)
        calls.append(lines[at:end])
        at = end + 1
    # decode: a scan launch of its own, without a workspace; else carries and outputs
    launches = [len(c) - 1 for c in calls]
    assert launches == [2, 2, 3, 3, 2, 2]
    assert [int(c[0][1]) > 0 for c in calls] == [False, False, True, True, False, False]
    # the convolution's decode kernel has 16 blocks of channels for four requests each
    conv = [int(c[-1][2]) for c in calls]
    assert conv[0] == conv[1] == 64 * 16 and conv[2] != conv[0]


def test_max_query_len_reaches_the_calls(monkeypatch):
    from greta_plugin_b200 import _capi
    from greta_plugin_b200.causal_conv import longest

    assert longest(0) == 1 << 8 and longest(33) == 33 << 8
    assert longest(10 ** 9) == (2 ** 22 - 1) << 8 < 2 ** 31
    with pytest.raises(ValueError, match="max_query_len"):
        longest(-1)
    assert _capi.lib().greta_ssm_scan_workspace(1, 64, 70, 64, 16, 1, 0) == 0
    assert _capi.lib().greta_ssm_scan_workspace(1 | longest(64), 64, 70, 64, 16, 1, 0) > 0


def test_scan_backward_parts_are_bounded(runtime):
    """A row of sums of dB and dC for every token and block of channels is as much as
    the inputs times the states: 8.6 GB in one launch of 16384 x 4096 x 128. Launches
    of some of the blocks after one another, whole waves of CTAs, keep it to 2 GB,
    or to what one wave leaves."""
    shapes = [(16384, 4096, 128, 1), (16384, 4096, 128, 3), (16384, 4096, 16, 1), (131072, 4096, 128, 1),
              (16384, 4096, 128, 512), (65536, 8192, 64, 8)]
    shapes = [(T, D // F * F, N, F) for T, D, N, F in shapes]
    lines = recorded(runtime, f"""
for T, D, N, F_ in {shapes}:
    n = L.greta_ssm_scan_bwd_workspace(1, T, D, N, F_, 0)
    print("bytes", n, flush=True)
    assert L.greta_ssm_scan_bwd(2, F, D, F, D, None, 0, F, F_ * N, F, F_ * N, F, None, None, F, F, F, F, None, F, F, F,
                                None, None, None, 0, 0, T, D, N, F_, 0, 0, F, n, None) == 0
    print("end", flush=True)
""")
    lines = [v for v in lines if v[0] != "set"]
    at = 0
    for T, D, N, F in shapes:
        end = lines.index(["end"], at)
        need, launches = int(lines[at][1]), [(int(v[2]), int(v[3])) for v in lines[at + 1:end]]
        at = end + 1
        lanes = 4 if N <= 16 else 8 if N <= 32 else 16 if N <= 64 else 32
        blocks = F * -(-(-(-(D // F) // (32 // lanes * 2))) // 4)
        R = launches[0][1]  # (the carries first)
        main = [x for x, y in launches[1:-1] if y == R and x <= blocks]
        sums = [x for x, y in launches[1:-1] if x == -(-T * 2 * N // 256)]
        assert sum(main) == blocks and len(sums) == len(main) and len(launches) == 2 + 2 * len(main)
        row, wave = T * 2 * N * 4, 148 * 3 // R
        most = max(main) * row
        assert most <= max(2 << 30, wave * row)
        assert len(main) == 1 or max(main) % wave == 0
        # what else there is: the carries and parts of the ranges, and the sums between the launches
        assert need <= most + R * D * N * 4 * 3 + 3 * R * D * 4 + F * row + 4096
