"""The serving operators on a machine without a GPU: the refusals that need no session, the
index arithmetic that the kernels share (compiled for the host), the Python side's checks,
and the restated planner's own properties."""
import ctypes
import pathlib
import shutil
import subprocess

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200 import _native as N
from titan_rs_b200.kernel_abi import DType

from serving_util import plan_reference

ROOT = pathlib.Path(__file__).resolve().parents[1]


def tensor(dtype, shape, strides=None):
    t = N.Tensor()
    t.dtype, t.rank = dtype, len(shape)
    steps = strides or tb.runtime.contiguous_strides(shape)
    for i, (n, st) in enumerate(zip(shape, steps)):
        t.shape[i], t.strides[i] = n, st
    return t


def execute(op, inputs, outputs, attrs=None):
    """The status and the detail of a call without a session: metadata is checked before it."""
    from titan_rs_b200.runtime import _attrs
    arr, n, _keep = _attrs(attrs or {})
    status = N.lib().tb_execute_outputs(None, None, op.encode(), (N.Tensor * len(inputs))(*inputs), len(inputs),
                                        (N.Tensor * len(outputs))(*outputs), len(outputs), arr, n, None)
    operation, detail = N.last_error()
    assert operation == "contract"
    return status, detail


BF, I32, F32 = N.TB_BF16, N.TB_I32, N.TB_F32


def varlen(**change):
    a = dict(q=(BF, (10, 4, 64)), k=(BF, (10, 2, 64)), v=(BF, (10, 2, 64)), cq=(I32, (4,)), ck=(I32, (4,)),
             o=(BF, (10, 4, 64)), attrs={})
    a.update(change)
    ins = [tensor(*a[n]) for n in ("q", "k", "v", "cq", "ck") if a[n]]
    return execute("attention.varlen", ins, [tensor(*a["o"])], a["attrs"])


def test_varlen_metadata_reaches_the_session_check():
    assert varlen() == (N.TB_ERR_INVALID, "null session")
    assert varlen(ck=None) == (N.TB_ERR_INVALID, "null session")
    assert varlen(attrs={"causal": True, "scale": 0.5}) == (N.TB_ERR_INVALID, "null session")


@pytest.mark.parametrize("change,keyword", [
    (dict(q=(F32, (10, 4, 64)), o=(F32, (10, 4, 64))), "BF16 or F16"),
    (dict(o=(N.TB_F16, (10, 4, 64))), "one dtype"),
    (dict(k=(N.TB_F16, (10, 2, 64))), "one dtype"),
    (dict(q=(BF, (10, 4)), o=(BF, (10, 4))), "rank-3"),
    (dict(o=(BF, (9, 4, 64))), "output shape"),
    (dict(q=(BF, (0, 4, 64)), o=(BF, (0, 4, 64))), "non-zero"),
    (dict(k=(BF, (0, 2, 64)), v=(BF, (0, 2, 64))), "non-zero"),
    (dict(v=(BF, (10, 1, 64))), "one shape"),
    (dict(k=(BF, (10, 2, 32)), v=(BF, (10, 2, 32))), "head dimension"),
    (dict(k=(BF, (10, 3, 64)), v=(BF, (10, 3, 64))), "multiple of the key heads"),
    (dict(k=(BF, (10, 8, 64)), v=(BF, (10, 8, 64))), "multiple of the key heads"),
    (dict(k=(BF, (9, 2, 64)), v=(BF, (9, 2, 64)), ck=None), "cu_seqlens_k"),
    (dict(cq=(N.TB_I64, (4,))), "I32 cu_seqlens"),
    (dict(cq=(I32, (1,)), ck=(I32, (1,))), "I32 cu_seqlens"),
    (dict(ck=(I32, (5,))), "I32 cu_seqlens"),
    (dict(cq=(I32, (4,), (2,))), "I32 cu_seqlens"),
    (dict(o=(BF, (10, 4, 64), (64, 64, 1))), "do not overlap"),
    (dict(attrs={"scale": "-1"}), "positive finite"),
    (dict(attrs={"scale": "nan"}), "positive finite"),
])
def test_varlen_refusals(change, keyword):
    status, detail = varlen(**change)
    assert status == N.TB_ERR_INVALID and keyword in detail, detail


def test_varlen_unsupported():
    for change in (dict(attrs={"mask": 1}), dict(attrs={"causal": 2}), dict(attrs={"max_query_len": 4}),
                   dict(q=(BF, (10, 4, 257)), o=(BF, (10, 4, 257)), k=(BF, (10, 2, 257)), v=(BF, (10, 2, 257)))):
        status, detail = varlen(**change)
        assert status == N.TB_ERR_UNSUPPORTED and "does not implement" in detail


def paged(**change):
    a = dict(q=(BF, (10, 4, 64)), k=(BF, (6, 16, 2, 64)), v=(BF, (6, 16, 2, 64)), table=(I32, (3, 5)),
             lens=(I32, (3,)), cq=(I32, (4,)), o=(BF, (10, 4, 64)), attrs={})
    a.update(change)
    return execute("attention.paged", [tensor(*a[n]) for n in ("q", "k", "v", "table", "lens", "cq")],
                   [tensor(*a["o"])], a["attrs"])


def test_paged_refusals():
    assert paged() == (N.TB_ERR_INVALID, "null session")
    assert paged(table=(I32, (3, 5), (9, 1))) == (N.TB_ERR_INVALID, "null session")
    for change, keyword in [
        (dict(k=(BF, (6, 16, 128)), v=(BF, (6, 16, 128))), "rank-4"),
        (dict(v=(BF, (6, 8, 2, 64))), "one shape"),
        (dict(k=(BF, (6, 0, 2, 64)), v=(BF, (6, 0, 2, 64))), "non-zero"),
        (dict(k=(BF, (6, 16, 2, 32)), v=(BF, (6, 16, 2, 32))), "head dimension"),
        (dict(k=(N.TB_F16, (6, 16, 2, 64)), v=(N.TB_F16, (6, 16, 2, 64))), "one dtype"),
        (dict(lens=(I32, (2,))), "seq_lens [batch]"),
        (dict(lens=(BF, (3,))), "seq_lens [batch]"),
        (dict(table=(I32, (2, 5))), "block_table"),
        (dict(table=(I32, (3, 0))), "block_table"),
        (dict(table=(I32, (3, 5), (1, 3))), "block_table"),
        (dict(attrs={"max_query_len": 0}), "positive integer"),
        (dict(attrs={"max_query_len": "2"}), "positive integer"),
    ]:
        status, detail = paged(**change)
        assert status == N.TB_ERR_INVALID and keyword in detail, (change, detail)


def test_append_and_plan_refusals():
    def append(k=(BF, (4, 2, 64)), v=(BF, (4, 2, 64)), slots=(I32, (4,)), kc=(BF, (6, 16, 2, 64)),
               vc=(BF, (6, 16, 2, 64)), attrs=None):
        return execute("kv_cache.append", [tensor(*k), tensor(*v), tensor(*slots)], [tensor(*kc), tensor(*vc)], attrs)

    def plan(ctx=(I32, (3,)), new=(I32, (3,)), free=(I32, (8,)), table=(I32, (3, 5)), lens=(I32, (3,)),
             cu=(I32, (4,)), slots=(I32, (20,)), status=(I32, (2,)), attrs={"page_size": 16}):
        return execute("kv_cache.plan", [tensor(*t) for t in (ctx, new, free)],
                       [tensor(*t) for t in (table, lens, cu, slots, status)], attrs)

    assert append() == plan() == (N.TB_ERR_INVALID, "null session")
    for got, keyword in [
        (append(k=(I32, (4, 2, 64))), "one dtype"), (append(kc=(F32, (6, 16, 2, 64))), "one dtype"),
        (append(v=(BF, (5, 2, 64))), "one shape"), (append(k=(BF, (4, 3, 64))), "one H and D"),
        (append(slots=(I32, (5,))), "slot_map [T]"), (append(slots=(N.TB_I64, (4,))), "slot_map [T]"),
        (append(vc=(BF, (5, 16, 2, 64))), "one shape"),
        (append(kc=(BF, (6, 16, 2, 64), (64, 64, 64, 1))), "do not overlap"),
        (append(k=(BF, (0, 2, 64)), v=(BF, (0, 2, 64)), slots=(I32, (0,))), "non-zero"),
        (append(kc=(BF, (1 << 30, 4, 2, 64)), vc=(BF, (1 << 30, 4, 2, 64))), "i32 ABI"),
        (plan(attrs={}), "page_size"), (plan(attrs={"page_size": 0}), "page_size"),
        (plan(new=(I32, (4,))), "[batch]"), (plan(cu=(I32, (3,))), "[batch]"), (plan(table=(I32, (2, 5))), "[batch]"),
        (plan(status=(I32, (1,))), "two words"), (plan(slots=(I32, (0,))), "non-zero"),
        (plan(ctx=(N.TB_I64, (3,))), "I32"), (plan(table=(I32, (3, 5), (2, 1))), "do not overlap"),
    ]:
        assert got[0] == N.TB_ERR_INVALID and keyword in got[1], got
    assert append(attrs={"page_size": 1})[0] == plan(attrs={"page_size": 4, "x": 1})[0] == N.TB_ERR_UNSUPPORTED
    many = 16385
    assert plan(ctx=(I32, (many,)), new=(I32, (many,)), table=(I32, (many, 1)), lens=(I32, (many,)),
                cu=(I32, (many + 1,)))[0] == N.TB_ERR_UNSUPPORTED


def test_routes_count_inputs_and_outputs():
    t = tensor(BF, (2, 2, 2))
    for op, n_in, n_out in [("attention.varlen", 3, 1), ("attention.varlen", 6, 1), ("attention.paged", 5, 1),
                            ("attention.paged", 6, 2), ("kv_cache.append", 3, 1), ("kv_cache.plan", 3, 4),
                            ("softmax", 1, 2)]:
        status, detail = execute(op, [t] * n_in, [t] * n_out)
        assert status == N.TB_ERR_INVALID and "requires" in detail, (op, detail)
    ev = ctypes.c_void_p(0)
    ins = (N.Tensor * 3)(t, t, t)
    assert N.lib().tb_execute(None, None, b"kv_cache.append", ins, 3, ctypes.byref(t), None, 0,
                              ctypes.byref(ev)) == N.TB_ERR_INVALID


def test_python_requests_name_their_outputs():
    class FakeRuntime(tb.Runtime):
        def __init__(self):
            self.session, self.stream, self.autotuner = object(), None, None

    rt = FakeRuntime()
    spec = tb.TensorSpec(DType.BF16, (6, 16, 2, 64))
    handle = tb.TensorHandle(rt.session, None, DType.BF16, (4, 2, 64), (128, 64, 1))
    request = tb.OpRequest("kv_cache.append", [handle] * 3, [spec, spec])
    for output in (None, handle, [handle], [handle] * 3):
        with pytest.raises(tb.ExecutionError, match="writes into existing tensors"):
            rt.execute(request, output=output)
    with pytest.raises(tb.ExecutionError, match="requires K, V and slot_map"):
        rt.execute(tb.OpRequest("kv_cache.append", [handle] * 3, [spec]))
    with pytest.raises(tb.ExecutionError, match="requires K, V and slot_map"):
        rt.bind(tb.OpRequest("kv_cache.append", [handle] * 2, [spec, spec]))


def test_request_creation_checks_its_arguments():
    L, t, handle = N.lib(), tensor(BF, (2, 2, 2)), ctypes.c_void_p(0)
    ins = (N.Tensor * 1)(t)
    for op, place, keyword in ((None, ctypes.byref(handle), "operator name"), (b"softmax", None, "handle"),
                               (b"softmax", ctypes.byref(handle), "null session")):
        assert L.tb_request_create(None, None, op, ins, 1, ins, 1, None, 0, place) == N.TB_ERR_INVALID
        assert keyword in N.last_error()[1]
    assert L.tb_request_create(None, None, b"softmax", None, 1, ins, 1, None, 0, ctypes.byref(handle)) == N.TB_ERR_INVALID
    assert L.tb_request_enqueue(None, None) == N.TB_ERR_INVALID and N.last_error()[1] == "null request"
    L.tb_request_release(None)


HARNESS = r"""
#include <cstdio>
#include "attn_params.cuh"
using namespace tb;
int main() {
  const int cu_q[] = {-5, 3, 2, 9, 2147483647}, lens[] = {-1, 40, 2147483647, 7};
  const int cu_k[] = {0, -2147483647 - 1, 6, 4, 30}, table[] = {0, 5, 6, -1, 2147483647, -2147483647 - 1, 1, 2};
  AttnParams p{};
  p.cu_q = (uint64_t)cu_q; p.cu_k = (uint64_t)cu_k; p.lens = (uint64_t)lens;
  p.tq = 8; p.tk = 10; p.batch = 4; p.page = 16; p.pages = 6; p.width = 2; p.table_row = 2; p.causal = 1;
  for (int paged = 0; paged < 2; ++paged) {
    p.table = paged ? (uint64_t)table : 0;
    for (int b = 0; b < 4; ++b) {
      const AttnRequest r = request_of(p, b);
      std::printf("%d %d %d %d %d %d\n", r.q0, r.lq, r.k0, r.lk, visible_keys(p, r, 0), visible_keys(p, r, 100));
    }
  }
  for (int b = 0; b < 4; ++b) std::printf("%d %d\n", page_of(p, b, 0), page_of(p, b, 1));
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler on this machine")
def test_index_arithmetic_clamps_what_the_device_holds(tmp_path):
    """request_of, visible_keys and page_of on broken index tensors: every row, key and page they
    give lies inside the extents the host checked."""
    (tmp_path / "harness.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-I",
                    str(ROOT / "titan_rs_b200" / "csrc" / "kernels"), str(tmp_path / "harness.cpp"), "-o",
                    str(tmp_path / "harness")], check=True, capture_output=True, text=True)
    text = subprocess.run([str(tmp_path / "harness")], check=True, capture_output=True, text=True).stdout
    lines = [[int(x) for x in line.split()] for line in text.splitlines()]
    for q0, lq, k0, lk, first, far in lines[:8]:
        assert 0 <= q0 and lq >= 0 and q0 + lq <= 8 and k0 >= 0 and lk >= 0
        assert 0 <= first <= lk and far == lk
    assert all(k0 + lk <= 10 for _, _, k0, lk, _, _ in lines[:4])
    assert [row[3] for row in lines[4:8]] == [0, 32, 32, 7]
    assert lines[8:] == [[0, 5], [-1, -1], [-1, -1], [1, 2]]


def test_planner_restatement_gives_each_token_a_slot_of_its_own():
    rng = np.random.default_rng(5)
    ctx, new = rng.integers(0, 70, 12), rng.integers(0, 40, 12)
    page, width = 16, 8
    table = np.full((12, width), -1, np.int32)
    used = 0
    for b in range(12):
        n = -(-int(ctx[b]) // page)
        table[b, :n] = np.arange(used, used + n)
        used += n
    free = np.arange(used, used + 100, dtype=np.int32)
    out, lens, cu, slots, status = plan_reference(ctx, new, free, table, int(new.sum()), page)
    assert status[1] == 0 and len(set(slots.tolist())) == slots.size and slots.min() >= 0
    assert (lens == ctx + new).all() and cu[-1] == new.sum()
    assert sorted(out[out >= used].tolist()) == free[:status[0]].tolist()
