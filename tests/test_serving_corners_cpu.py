"""The serving operators' checks that need no GPU, beyond those of test_serving_cpu.py."""
import pathlib
import shutil
import subprocess
import sys

import pytest

import titan_rs_b200 as tb
from titan_rs_b200 import _native as N
from titan_rs_b200.kernel_abi import DType

from test_serving_cpu import execute, paged, tensor, varlen


class UnlaunchedRuntime(tb.Runtime):
    def __init__(self):
        self.session, self.stream, self.autotuner = object(), None, None


@pytest.mark.parametrize("operator,dtype,shape", [("kv_cache.append", DType.BF16, (6, 16, 2, 64)),
                                                  ("attention.varlen", DType.BF16, (6, 16, 64))])
def test_an_output_has_to_be_its_spec(operator, dtype, shape):
    rt = UnlaunchedRuntime()
    handle = lambda dtype, shape, strides=None: tb.TensorHandle(  # noqa: E731
        rt.session, None, dtype, shape, strides or tb.runtime.contiguous_strides(shape))
    count = 2 if operator == "kv_cache.append" else 1
    inputs = [handle(dtype, (4, 2, 64))] * (3 if count == 2 else 4)

    def outputs(spec, tensor):
        return rt._checked(tb.OpRequest(operator, inputs, [spec] * count), [tensor] * count)

    plain = tb.runtime.contiguous_strides(shape)
    turned = tuple(2 * x for x in plain[:-1]) + (1,)
    # A spec without strides takes the tensor's; equal ones and those of an extent of one pass.
    request, _ = outputs(tb.TensorSpec(dtype, shape), handle(dtype, shape, turned))
    assert [s.resolved_strides() for s in request.outputs] == [turned] * count
    outputs(tb.TensorSpec(dtype, shape, turned), handle(dtype, shape, turned))
    single = (1,) + shape[1:]
    outputs(tb.TensorSpec(dtype, single, (7,) + plain[1:]), handle(dtype, single))
    for spec, tensor in [(tb.TensorSpec(dtype, shape, plain), handle(dtype, shape, turned)),
                         (tb.TensorSpec(dtype, shape), handle(DType.F16, shape)),
                         (tb.TensorSpec(dtype, shape), handle(dtype, (5,) + shape[1:])),
                         (tb.TensorSpec(dtype, shape), handle(dtype, shape[1:]))]:
        with pytest.raises(tb.ExecutionError, match="their specs' dtype, shape and strides"):
            outputs(spec, tensor)


BANKS = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "attn_params.cuh"
using namespace tb;
int main() {
  std::vector<int> work(kWorkFront / 4, 0);  // as a workspace begins
  const int grids[] = {148, 3, 148, 1, 1, 148, 512, 2, 148, 148};
  for (int n = 0; n < 200; ++n) {
    const int grid = grids[n % 10], threads = grid * 32, turn = work[kTileTurn];
    for (int slot = 0; slot < 2 * kTileMaxCtas; ++slot)
      for (int x = 0; x < 2; ++x)
        if (work[tile_parts_at(turn, slot, x)] != 0) return std::printf("launch %d, slot %d\n", n, slot), 1;
    for (int id = 0; id < threads; ++id) clear_next_bank(work.data(), turn, id, threads);
    // Finished parts of all of the launch's slots: whatever a wait that ran out leaves.
    for (int slot = 0; slot < 2 * grid; ++slot)
      for (int x = 0; x < 2; ++x) work[tile_parts_at(turn, slot, x)] = std::rand() % 33;
    work[kTileTurn] = turn ^ 1;
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler on this machine")
def test_no_launch_counts_parts_of_an_earlier_one(tmp_path):
    """The counters of finished parts, as a row of launches of different grids uses and clears them:
    each finds its own at zero, whatever the ones before left."""
    kernels = pathlib.Path(__file__).resolve().parents[1] / "titan_rs_b200" / "csrc" / "kernels"
    (tmp_path / "banks.cpp").write_text(BANKS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-I", str(kernels),
                    str(tmp_path / "banks.cpp"), "-o", str(tmp_path / "banks")], check=True, capture_output=True,
                   text=True)
    done = subprocess.run([str(tmp_path / "banks")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("call", [varlen, paged])
def test_a_scale_that_is_no_float_is_refused(call):
    for scale in ("1e-46", "1e-300", "2.4e38", "1e39", "1e300", "inf", "0", "1e-500"):
        status, detail = call(attrs={"scale": scale})
        assert status == N.TB_ERR_INVALID and "positive finite" in detail, (scale, detail)
    for scale in ("1e-45", "1e-40", "2.3e38"):
        assert call(attrs={"scale": scale}) == (N.TB_ERR_INVALID, "null session"), scale


def test_append_refuses_rows_of_more_chunks_than_it_counts():
    """A token's K and V rows in chunks of 16, 4 or 2 bytes: below 2^31 of them."""
    def append(h, d, dtype, steps=None):
        row = tensor(dtype, (1, h, d), steps)
        cache = tensor(dtype, (1, 1, h, d), steps and (1,) + steps)
        return execute("kv_cache.append", [row, row, tensor(N.TB_I32, (1,))], [cache, cache])

    for h, d, dtype, steps in [(65535, 65535, N.TB_F32, None), (65535, 65535, N.TB_BF16, None),
                               (65535, 32767, N.TB_BF16, None), (65535, 16385, N.TB_F32, None),
                               (65535, 65528, N.TB_BF16, (1, 65529, 1))]:
        status, detail = append(h, d, dtype, steps)
        assert status == N.TB_ERR_INVALID and "i32 ABI" in detail, (h, d, detail)
    for h, d, dtype in [(65535, 65532, N.TB_F32), (65535, 65528, N.TB_BF16), (65535, 16383, N.TB_BF16)]:
        assert append(h, d, dtype) == (N.TB_ERR_INVALID, "null session"), (h, d)


NO_MEMORY = """
import ctypes, resource
from titan_rs_b200 import _native as N
lib, handle = N.lib(), ctypes.c_void_p(0)
t = N.Tensor()
name = ctypes.create_string_buffer(b"x" * (1 << 28))
# No room for another copy of the name.
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (1 << 26), resource.RLIM_INFINITY))
print(lib.tb_execute_outputs(None, None, name, ctypes.byref(t), 1, ctypes.byref(t), 1, None, 0, None))
print(lib.tb_execute(None, None, name, ctypes.byref(t), 1, ctypes.byref(t), None, 0, None))
"""


def test_the_router_returns_when_host_memory_runs_out():
    """A C++ exception does not leave the C entries: they return a status."""
    done = subprocess.run([sys.executable, "-c", NO_MEMORY], capture_output=True, text=True,
                          cwd=pathlib.Path(__file__).resolve().parents[1])
    assert done.returncode == 0, (done.returncode, done.stderr)
    assert done.stdout.split() == [str(N.TB_ERR_OUT_OF_MEMORY)] * 2
