"""The serving operators at sizes, bounds and arguments between those of the other tests."""
import math

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import as_f64, assert_attention, paged_reference, plan_reference, rows
from test_attention_serving_gpu import check_varlen, ints, make_cache, prefix, run_paged, view
from test_kv_cache_gpu import assert_plan, random_plan, spec_of

pytestmark = pytest.mark.gpu


@pytest.fixture()
def session():
    s = tb.Session(0)
    yield s
    s.close()


@pytest.fixture()
def rt(session):
    return tb.Runtime(session)


def test_plan_of_every_batch_launches(session, rt):
    """Batches whose shared memory is 48 KB with the kernel's static bytes, the smaller ones first."""
    for batch in (6109, 6110, 6143, 6144, 16384, 6120):
        rng = np.random.default_rng(batch)
        ctx, new, free, table = random_plan(rng, batch, 9, 2, 4)
        got = assert_plan(session, rt, ctx, new, free, table, int(new.sum()) + 1, 4)
        assert got[4][1] == 0


def test_outputs_are_written_where_their_tensors_lie(session, rt):
    """Specs without strides beside strided outputs: a cache with heads before rows, an attention
    output inside a wider tensor, a block table with wider rows."""
    hk, h, d, page, pages, t, dtype = 2, 4, 64, 8, 4, 5, DType.BF16
    host = rows((t, hk, d), dtype, 1)
    k = upload(session, rt.stream, host, dtype)
    base = upload(session, rt.stream, np.zeros((2, pages, hk, page, d), np.uint16), dtype)
    caches = [view(session, base, i * pages * hk * page * d, (pages, page, hk, d), (hk * page * d, d, page * d, 1))
              for i in range(2)]
    slots = [0, 9, 17, 3, 30]
    rt.execute(tb.OpRequest("kv_cache.append", [k, k, ints(session, rt, slots)],
                            [tb.TensorSpec(dtype, c.shape) for c in caches]), output=caches).wait()
    want = np.zeros((2, pages, hk, page, d), np.uint16)
    for n, slot in enumerate(slots):
        want[:, slot // page, :, slot % page] = host[n]
    np.testing.assert_array_equal(base.to_numpy(rt.stream), want)

    q = upload(session, rt.stream, rows((t, h, d), dtype, 2), dtype)
    wide = upload(session, rt.stream, np.zeros((t, h, d + 24), np.uint16), dtype)
    o = view(session, wide, 0, (t, h, d), (h * (d + 24), d + 24, 1))
    inputs = [q, k, k, ints(session, rt, [0, 2, 5])]
    plain = rt.execute(tb.OpRequest("attention.varlen", inputs, [tb.TensorSpec(dtype, (t, h, d))])).wait()
    got = rt.execute(tb.OpRequest("attention.varlen", inputs, [tb.TensorSpec(dtype, (t, h, d))]), output=o).wait()
    assert got.outputs[0].strides == o.strides
    after = wide.to_numpy(rt.stream)
    np.testing.assert_array_equal(after[:, :, :d], plain.outputs[0].to_numpy(rt.stream))
    np.testing.assert_array_equal(after[:, :, d:], 0)

    table = ints(session, rt, np.full((2, 5), -3))
    outs = [tb.TensorHandle(session, table.buffer, DType.I32, (2, 2), (5, 1)), ints(session, rt, [0, 0]),
            ints(session, rt, [0, 0, 0]), ints(session, rt, [0] * 9), ints(session, rt, [0, 0])]
    rt.bind(tb.OpRequest("kv_cache.plan", [ints(session, rt, x) for x in ([0, 0], [9, 3], [5, 6, 7])],
                         [tb.TensorSpec(DType.I32, x.shape) for x in outs], {"page_size": 8}), outs).enqueue()
    # (The second request's tokens, 9 to 11, pass the end of the slot map: it is refused.)
    np.testing.assert_array_equal(table.to_numpy(rt.stream), [[5, 6, -3, -3, -3], [-3, -3, -3, -3, -3]])


def test_cut_requests_one_behind_another(session):
    """Requests whose keys are cut into parts, of different sizes and grids, launched in turn on one
    stream: every launch gives the same result."""
    page, dtype, d = 16, DType.BF16, 64
    runtime = tb.Runtime(session)
    bound = []
    for lens, new, h, hk in (([6000], [70], 4, 1), ([3000, 70, 1100], [20, 20, 20], 8, 2), ([700], [40], 2, 1)):
        cu = prefix(new)
        k, v, table = make_cache(lens, page, hk, d, dtype, 40 + h)
        q = upload(session, runtime.stream, rows((int(cu[-1]), h, d), dtype, 50 + h), dtype)
        ins = [q] + [upload(session, runtime.stream, x, dtype) for x in (k, v)]
        ins += [ints(session, runtime, x) for x in (table, lens, cu)]
        request = tb.OpRequest("attention.paged", ins, [spec_of(q)], {"candidate": "attention_tiles"})
        bound.append(runtime.bind(request, tb.TensorHandle.allocate(session, dtype, q.shape)))
    want = []
    for b in bound:
        b.enqueue()
        want.append(b.outputs[0].to_numpy(runtime.stream))
    for n in range(60):
        bound[(n * n) % 3].enqueue()
        bound[n % 3].enqueue()
        if n % 7 == 0:
            for b, w in zip(bound, want):
                np.testing.assert_array_equal(b.outputs[0].to_numpy(runtime.stream), w)
    for b, w in zip(bound, want):
        np.testing.assert_array_equal(b.outputs[0].to_numpy(runtime.stream), w)


@pytest.mark.parametrize("candidate", ["attention_tiles", "attention_rows", "attention_tokens"])
def test_the_smallest_scales_give_means(session, rt, candidate):
    """With a scale below the normal floats every visible key weighs the same, and a hidden one nothing."""
    h, hk, d, page, dtype, lens, new = 4, 2, 64, 16, DType.BF16, [70, 5], [4, 3]
    cu = prefix(new)
    q, out = rows((7, h, d), dtype, 60), np.zeros((7, h, d), np.uint16)
    k, v, table = make_cache(lens, page, hk, d, dtype, 61)
    for scale in (1e-40, 1.4e-45):
        name, got = run_paged(session, rt, q, k, v, table, lens, cu, out, dtype,
                              {"scale": scale, "candidate": candidate, "max_query_len": 4})
        assert name.startswith(candidate)
        ref, mag = paged_reference(q, k, v, table, lens, cu, True, scale, as_f64(out))
        assert_attention(got, ref, mag, dtype, 70, np.nanmax(np.abs(as_f64(v))))


def test_a_request_past_max_query_len_takes_nothing_from_the_others(session, rt):
    """max_query_len says too little for one request: its rows may be left, the others' may not."""
    h, hk, d, page, dtype, bound = 32, 8, 128, 16, DType.BF16, 40
    lens, new = [4000, 50, 300], [4000, bound, 33]
    cu = prefix(new)
    q = rows((int(cu[-1]), h, d), dtype, 70)
    out = np.zeros((int(cu[-1]), h, d), np.uint16)
    k, v, table = make_cache(lens, page, hk, d, dtype, 71)
    name, got = run_paged(session, rt, q, k, v, table, lens, cu, out, dtype, {"max_query_len": bound})
    assert name.startswith("attention_tiles")
    at = cu[1]
    ref, mag = paged_reference(q[at:], k, v, table[1:], lens[1:], cu[1:] - at, True, 1 / math.sqrt(d),
                               as_f64(out[at:]))
    assert_attention(got[at:], ref, mag, dtype, 300, np.nanmax(np.abs(as_f64(v))))


def test_rows_of_no_request_in_an_omitted_output_are_zeros(session, rt):
    n, dtype = 500, DType.BF16
    x = upload(session, rt.stream, rows((n, 4, 64), dtype, 80), dtype)
    cu = ints(session, rt, [0, 40])
    for _ in range(8):  # memory that another tensor was in
        upload(session, rt.stream, np.full((n, 4, 64), 0x7FC1, np.uint16), dtype).buffer.release()
        got = rt.execute(tb.OpRequest("attention.varlen", [x, x, x, cu], [spec_of(x)])).wait()
        host = got.outputs[0].to_numpy(rt.stream)
        assert host[:40].any() and not host[40:].any()


def halves_of_a_row(session, rt, op, candidate, group, n, gap, d=64):
    """O of `group` heads over n f16 keys, of which the first scores `gap` above the others; v = 0 for it and
    1 for them, so O is what the others weigh."""
    dtype, page = DType.F16, 16
    q = np.zeros((1, group, d), np.float16)
    k, v = np.zeros((n, 1, d), np.float16), np.ones((n, 1, d), np.float16)
    q[..., 0], k[0, 0, 0], v[0] = 1.0, gap, 0.0
    attrs = {"scale": 1.0, "causal": False, "candidate": candidate}
    spec = [tb.TensorSpec(dtype, q.shape)]
    if op == "attention.varlen":
        ins = [upload(session, rt.stream, x, dtype) for x in (q, k, v)] + [ints(session, rt, x) for x in ([0, 1], [0, n])]
    else:
        pages = -(-n // page)
        caches = [np.zeros((pages * page, 1, d), np.float16) for _ in range(2)]
        caches[0][:n], caches[1][:n] = k, v
        ins = [upload(session, rt.stream, q, dtype)]
        ins += [upload(session, rt.stream, c.reshape(pages, page, 1, d), dtype) for c in caches]
        ins += [ints(session, rt, x) for x in (np.arange(pages)[None], [n], [0, 1])]
        attrs["max_query_len"] = 1
    got = rt.execute(tb.OpRequest(op, ins, spec, attrs)).wait()
    assert got.candidate.startswith(candidate)
    return got.outputs[0].to_numpy(rt.stream).astype(np.float64)


@pytest.mark.parametrize("op,candidate,group", [("attention.varlen", "attention_tiles", 4),
                                                ("attention.paged", "attention_tiles", 40),
                                                ("attention.paged", "attention_tokens", 4),
                                                ("attention.paged", "attention_tokens", 32),
                                                ("attention.paged", "attention_rows", 4)])
@pytest.mark.parametrize("n,gap", [(100000, 17.75), (131072, 14.0), (3000, 17.5)])
def test_f16_keys_of_little_weight_count_together(session, rt, op, candidate, group, n, gap):
    """Many keys that each weigh less than f16 holds next to 1: the weights are held 2^7 times as large,
    so each is off by at most 2^-25 / 2^7 (or half a step, 2^-11 of it), and O by n times that. The
    fp32 sums and ex2.approx are within 2^-11 of O, and O is rounded once (2^-11)."""
    got = halves_of_a_row(session, rt, op, candidate, group, n, gap)
    weight = math.exp(-gap)
    want = (n - 1) * weight / (1 + (n - 1) * weight)
    assert np.abs(got - want).max() <= 3 * 2.0 ** -11 * want + n * 2.0 ** -32 + 2.0 ** -25
