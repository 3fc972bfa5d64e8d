"""Attention over packed and paged sequences on the GPU against a 64-bit restatement: types,
head groupings, ragged, empty and single-row requests, strides, foreign page ids, and bits
that no row may see."""
import math

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import assert_attention, as_f64, paged_reference, quiet_nan, rows, varlen_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def session():
    s = tb.Session(0)
    yield s
    s.close()


@pytest.fixture(scope="module")
def rt(session):
    return tb.Runtime(session)


def ints(session, rt, values):
    return upload(session, rt.stream, np.asarray(values, np.int32), DType.I32)


def prefix(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def view(session, base: tb.TensorHandle, offset: int, shape, strides):
    """A strided tensor inside another one's memory, `offset` elements from its start."""
    size = 2
    extent = 1 + sum((n - 1) * st for n, st in zip(shape, strides))
    buf = session.wrap(base.buffer.device_ptr + offset * size, extent * size)
    buf.base = base  # keeps the memory alive
    return tb.TensorHandle(session, buf, base.dtype, tuple(shape), tuple(strides))


def run_varlen(session, rt, q, k, v, cu_q, cu_k, out, dtype, attrs, handles=None):
    ins = handles or [upload(session, rt.stream, t, dtype) for t in (q, k, v)]
    ins = ins + [ints(session, rt, cu_q)] + ([] if cu_k is None else [ints(session, rt, cu_k)])
    o = upload(session, rt.stream, out, dtype)
    h = rt.execute(tb.OpRequest("attention.varlen", ins, [tb.TensorSpec(dtype, out.shape)], attrs), output=o)
    h.wait()
    return h.candidate, h.outputs[0].to_numpy(rt.stream)


def check_varlen(session, rt, lq, lk, h, hk, d, dtype, causal, pad=0, scale=None, candidate=None, seed=1, std=1.0):
    cross = lk is not None
    cu_q, cu_k = prefix(lq), prefix(lk if cross else lq)
    tq, tk = int(cu_q[-1]) + pad, int(cu_k[-1]) + (3 if cross else pad)
    q = rows((tq, h, d), dtype, seed, std)
    k, v = rows((tk, hk, d), dtype, seed + 1, std), rows((tk, hk, d), dtype, seed + 2)
    out = rows((tq, h, d), dtype, seed + 3)
    k[cu_k[-1]:] = v[cu_k[-1]:] = quiet_nan(dtype)
    attrs = {"causal": causal}
    if scale:
        attrs["scale"] = scale
    if candidate:
        attrs["candidate"] = candidate
    name, got = run_varlen(session, rt, q, k, v, cu_q, cu_k if cross else None, out, dtype, attrs)
    ref, mag = varlen_reference(q, k, v, cu_q, cu_k, causal, scale or 1 / math.sqrt(d), as_f64(out))
    assert_attention(got, ref, mag, dtype, max(max(lk if cross else lq), 1), np.abs(as_f64(v[:cu_k[-1]])).max(initial=0))
    np.testing.assert_array_equal(got[cu_q[-1]:], out[cu_q[-1]:])
    return name


LENGTHS = [[1], [5, 1, 0, 7], [64, 63, 65], [130, 2, 127, 128, 129], [300, 0, 0, 33]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [DType.BF16, DType.F16])
@pytest.mark.parametrize("h,hk", [(1, 1), (4, 4), (8, 2), (6, 2), (8, 1)])
@pytest.mark.parametrize("lq", LENGTHS, ids=str)
def test_varlen_causal(session, rt, lq, h, hk, d, dtype):
    check_varlen(session, rt, lq, None, h, hk, d, dtype, True, pad=2, seed=len(lq) * 10 + h)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([3, 0, 200], [0, 50, 70]), ([1, 1, 1, 1], [500, 1, 128, 129]),
                                   ([257, 20], [100, 300]), ([128, 256], [256, 128])], ids=str)
@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.F16, 64)])
def test_varlen_key_lengths_of_their_own(session, rt, lq, lk, causal, dtype, d):
    """Rows that see no key (no keys at all; more causal rows than keys) give zeros."""
    check_varlen(session, rt, lq, lk, 8, 2, d, dtype, causal, pad=1, seed=50 + sum(lq))


@pytest.mark.parametrize("d", [1, 7, 80, 96, 136, 256])
def test_varlen_other_head_dimensions(session, rt, d):
    check_varlen(session, rt, [17, 1, 40], None, 4, 2, d, DType.BF16, True, pad=1, seed=60 + d)


def test_varlen_groups_that_do_not_divide_a_tile(session, rt):
    for h, hk in [(5, 1), (7, 1), (12, 1), (24, 2), (40, 1)]:
        check_varlen(session, rt, [90, 31], None, h, hk, 128, DType.BF16, True, seed=80 + h)


def test_varlen_many_requests(session, rt):
    lq = [int(x) for x in np.random.default_rng(7).integers(0, 20, 700)]
    check_varlen(session, rt, lq, None, 4, 2, 64, DType.BF16, True, pad=5, seed=90)


def test_varlen_scale_and_large_scores(session, rt):
    check_varlen(session, rt, [200, 70], None, 4, 2, 128, DType.BF16, True, scale=0.03, seed=100)
    # Scores of some hundreds: all but a few probabilities vanish, the running maximum moves.
    d, std, dtype = 128, 4.0, DType.F16
    q, k, v = (rows((260, 2, d), dtype, 110 + i, std if i < 2 else 1.0) for i in range(3))
    cu = prefix([260])
    _, got = run_varlen(session, rt, q, k, v, cu, None, np.zeros((260, 2, d), np.float16), dtype, {"causal": True})
    ref, mag = varlen_reference(q, k, v, cu, cu, True, 1 / math.sqrt(d), np.zeros((260, 2, d)))
    # fp32 scores of size 16 x 11: |ds| <= 2^-23 x 128 x sum|q k| scale, sum|q k| scale <= 16 x 0.64 x 128 / 11.3 = 116.
    ds = 2.0 ** -23 * 128 * 120
    excess = np.abs(as_f64(got) - ref) - (2.0 ** -11 * np.abs(ref) + (2.0 ** -11 + 2 * ds + 2.0 ** -11) * mag + 1e-4)
    assert excess.max() <= 0


def test_varlen_strided_projection_and_output(session, rt):
    """Q, K and V as slices of one projection, the output inside a wider tensor with heads outermost."""
    h, hk, d, lq, dtype = 8, 2, 128, [70, 1, 129], DType.BF16
    cu = prefix(lq)
    t, width = int(cu[-1]), (8 + 4) * 128
    qkv = rows((t, h + 2 * hk, d), dtype, 120)
    base = upload(session, rt.stream, qkv, dtype)
    q = view(session, base, 0, (t, h, d), (width, d, 1))
    k = view(session, base, h * d, (t, hk, d), (width, d, 1))
    v = view(session, base, (h + hk) * d, (t, hk, d), (width, d, 1))
    wide = upload(session, rt.stream, rows((h, t + 2, d + 8), dtype, 121), dtype)
    before = wide.to_numpy(rt.stream)
    strides = (d + 8, (t + 2) * (d + 8), 1)
    o = view(session, wide, 0, (t, h, d), strides)
    rt.execute(tb.OpRequest("attention.varlen", [q, k, v, ints(session, rt, cu)],
                            [tb.TensorSpec(dtype, (t, h, d), strides)], {"causal": True}), output=o).wait()
    after = wide.to_numpy(rt.stream)
    ref, mag = varlen_reference(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], cu, cu, True, 1 / math.sqrt(d),
                                np.zeros((t, h, d)))
    assert_attention(after[:, :t, :d].transpose(1, 0, 2), ref, mag, dtype, 129, np.abs(as_f64(qkv)).max())
    after[:, :t, :d] = before[:, :t, :d]
    np.testing.assert_array_equal(after, before)


def test_varlen_odd_strides_and_offsets(session, rt):
    """Rows that start at odd elements: no 16-byte load fits."""
    h, hk, d, dtype = 4, 2, 64, DType.BF16
    cu = prefix([33, 70])
    t, step = 103, 6 * 67 + 1
    flat = rows((t * step + 1,), dtype, 130)
    base = upload(session, rt.stream, flat, dtype)
    handles = [view(session, base, 1, (t, h, d), (step, 67, 1)),
               view(session, base, 1 + 4 * 67, (t, hk, d), (step, 67, 1)),
               view(session, base, 1 + 2 * 67, (t, hk, d), (step, 67, 1))]
    host = [np.lib.stride_tricks.as_strided(flat[at:], (t, n, d), (2 * step, 134, 2)).copy()
            for at, n in ((1, h), (1 + 4 * 67, hk), (1 + 2 * 67, hk))]
    out = np.zeros((t, h, d), np.uint16)
    _, got = run_varlen(session, rt, None, None, None, cu, None, out, dtype, {"causal": True}, handles)
    ref, mag = varlen_reference(*host, cu, cu, True, 1 / math.sqrt(d), as_f64(out))
    assert_attention(got, ref, mag, dtype, 70, np.abs(as_f64(host[2])).max())


def test_varlen_infinite_scores_weigh_nothing_or_everything(session, rt):
    """-inf scores have weight 0, in a row with other keys and in one with none; +inf gives NaN, as
    inf - inf does in the definition."""
    h, d, dtype = 1, 64, DType.F16
    q, k, v = np.zeros((6, h, d), np.float16), np.zeros((6, h, d), np.float16), rows((6, h, d), dtype, 140)
    q[:, 0, 0] = 1.0
    k[1, 0, 0] = -np.inf  # key 1 of request 0
    k[3, 0, 0] = -np.inf  # the only key of request 1
    k[5, 0, 0] = np.inf   # the last key of request 2
    cu = np.array([0, 3, 4, 6], np.int32)
    _, got = run_varlen(session, rt, q, k, v, cu, None, np.ones((6, h, d), np.float16), dtype, {"causal": False})
    got = got.astype(np.float64)
    want = (as_f64(v[0]) + as_f64(v[2])) / 2
    np.testing.assert_allclose(got[0], want, rtol=2.0 ** -9, atol=2.0 ** -12)
    np.testing.assert_array_equal(got[3], 0.0)
    assert np.isnan(got[4]).all() and np.isnan(got[5]).all()


def test_varlen_broken_index_tensors_stay_inside(session, rt):
    """cu_seqlens that run backwards or past the tensors: nothing outside is read or written, and
    requests with a sound range are computed."""
    h, d, dtype, t = 2, 64, DType.BF16, 40
    q, k, v = (rows((t, h, d), dtype, 150 + i) for i in range(3))
    guard = rows((3 * t, h, d), dtype, 154)
    base = upload(session, rt.stream, guard, dtype)
    o = view(session, base, t * h * d, (t, h, d), (h * d, d, 1))
    cu = np.array([-7, 10, 5, 30, 2 ** 31 - 1], np.int32)
    ins = [upload(session, rt.stream, x, dtype) for x in (q, k, v)] + [ints(session, rt, cu)]
    rt.execute(tb.OpRequest("attention.varlen", ins, [tb.TensorSpec(dtype, (t, h, d))], {}), output=o).wait()
    after = base.to_numpy(rt.stream)
    np.testing.assert_array_equal(after[:t], guard[:t])
    np.testing.assert_array_equal(after[2 * t:], guard[2 * t:])
    ref, mag = varlen_reference(q, k, v, [30, t], [30, t], False, 1 / math.sqrt(d), np.zeros((t, h, d)))
    assert_attention(after[t + 30:2 * t], ref[30:], mag[30:], dtype, t, np.abs(as_f64(v)).max())


# ---------------------------------------------------------------- paged
def make_cache(lengths, page, hk, d, dtype, seed, spare=4, width=None):
    """Caches whose unused rows and pages hold NaNs, a shuffled table whose unused entries hold
    page ids of no page."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    width = width or max(max(need), 1) + 1
    table = np.full((len(lengths), width), np.int32(2 ** 31 - 1))
    k, v = (np.full((pages, page, hk, d), quiet_nan(dtype)) for _ in range(2))
    at = 0
    for b, n in enumerate(lengths):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for c, cache in ((0, k), (1, v)):
            data = rows((n, hk, d), dtype, seed * 7 + 2 * b + c) if n else None
            for i in range(need[b]):
                part = data[i * page:(i + 1) * page]
                cache[table[b, i], :len(part)] = part
    return k, v, table


def run_paged(session, rt, q, k, v, table, lens, cu_q, out, dtype, attrs):
    ins = [upload(session, rt.stream, t, dtype) for t in (q, k, v)]
    ins += [ints(session, rt, table), ints(session, rt, lens), ints(session, rt, cu_q)]
    o = upload(session, rt.stream, out, dtype)
    h = rt.execute(tb.OpRequest("attention.paged", ins, [tb.TensorSpec(dtype, out.shape)], attrs), output=o)
    h.wait()
    return h.candidate, h.outputs[0].to_numpy(rt.stream)


def check_paged(session, rt, lens, new, h, hk, d, page, dtype, pad=0, causal=True, attrs=None, seed=1):
    cu_q = prefix(new)
    tq = int(cu_q[-1]) + pad
    q, out = rows((tq, h, d), dtype, seed), rows((tq, h, d), dtype, seed + 3)
    k, v, table = make_cache(lens, page, hk, d, dtype, seed)
    attrs = {**({} if causal else {"causal": False}), **(attrs or {})}
    name, got = run_paged(session, rt, q, k, v, table, lens, cu_q, out, dtype, attrs)
    ref, mag = paged_reference(q, k, v, table, lens, cu_q, causal, 1 / math.sqrt(d), as_f64(out))
    v_max = np.nanmax(np.abs(as_f64(v)), initial=0.0)
    assert_attention(got, ref, mag, dtype, max(lens), v_max)
    np.testing.assert_array_equal(got[cu_q[-1]:], out[cu_q[-1]:])
    return name


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [DType.BF16, DType.F16])
@pytest.mark.parametrize("h,hk", [(1, 1), (8, 8), (8, 2), (6, 2), (16, 1), (40, 1)])
@pytest.mark.parametrize("bound", [False, True])
def test_paged_single_tokens(session, rt, h, hk, d, dtype, bound):
    lens = [1, 16, 17, 63, 64, 65, 700, 0, 129]
    check_paged(session, rt, lens, [1] * 9, h, hk, d, 16, dtype, pad=2, seed=200 + h,
                attrs={"max_query_len": 1} if bound else None)


@pytest.mark.parametrize("page", [1, 8, 16, 24, 64, 128, 256])
def test_paged_page_sizes(session, rt, page):
    check_paged(session, rt, [300, 5, 257], [1, 1, 1], 8, 2, 128, page, DType.BF16, seed=300 + page)
    check_paged(session, rt, [300, 5, 257], [150, 5, 1], 8, 2, 128, page, DType.BF16, seed=310 + page)


@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.F16, 128), (DType.BF16, 64), (DType.F16, 64)])
@pytest.mark.parametrize("h,hk", [(2, 2), (8, 2), (5, 1), (8, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_chunks(session, rt, dtype, d, h, hk, causal):
    """New tokens of every kind in one call: a whole prompt, a chunk behind a context, one token, none,
    a few (as in speculation), and more rows than keys."""
    lens, new = [200, 333, 512, 40, 90, 20], [200, 130, 1, 0, 5, 30]
    check_paged(session, rt, lens, new, h, hk, d, 16, dtype, pad=3, causal=causal, seed=400 + h)


@pytest.mark.parametrize("bound", [2, 3, 4, 9, 40])
def test_paged_bounded_chunks(session, rt, bound):
    new = [bound, 1, max(1, bound - 1), 0]
    check_paged(session, rt, [300, 77, 128, 64], new, 8, 2, 128, 32, DType.BF16, seed=450 + bound,
                attrs={"max_query_len": bound})


def test_paged_long_context_is_split_and_joined(session, rt):
    check_paged(session, rt, [20011, 3, 9000], [1, 1, 1], 8, 2, 128, 16, DType.F16, seed=500)
    check_paged(session, rt, [6007], [70], 4, 1, 64, 64, DType.F16, seed=510)


def test_paged_many_requests(session, rt):
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(1, 60, 600)]
    new = [int(min(n, x)) for n, x in zip(lens, rng.integers(0, 4, 600))]
    check_paged(session, rt, lens, new, 4, 2, 64, 8, DType.BF16, seed=520)


def test_paged_table_entries_without_a_page_read_as_zeros(session, rt):
    h, hk, d, page, dtype = 8, 2, 128, 16, DType.BF16
    lens, new = [100, 60, 300], [1, 1, 200]
    k, v, table = make_cache(lens, page, hk, d, dtype, 530)
    table[0, 2], table[1, 3], table[2, 7] = -1, 10 ** 9, k.shape[0]
    cu = prefix(new)
    q, out = rows((202, h, d), dtype, 531), np.zeros((202, h, d), np.uint16)
    _, got = run_paged(session, rt, q, k, v, table, lens, cu, out, dtype, {})
    ref, mag = paged_reference(q, k, v, table, lens, cu, True, 1 / math.sqrt(d), as_f64(out))
    assert_attention(got, ref, mag, dtype, 300, np.nanmax(np.abs(as_f64(v))))


def test_paged_lengths_past_the_table_are_clamped(session, rt):
    h, hk, d, page, dtype = 4, 1, 64, 16, DType.BF16
    k, v, table = make_cache([32, 32], page, hk, d, dtype, 540, width=2)
    q, out = rows((2, h, d), dtype, 541), np.zeros((2, h, d), np.uint16)
    _, got = run_paged(session, rt, q, k, v, table, [2 ** 31 - 1, -5], [0, 1, 2], out, dtype, {})
    ref, mag = paged_reference(q, k, v, table, [32, 0], [0, 1, 2], True, 1 / math.sqrt(d), as_f64(out))
    assert_attention(got, ref, mag, dtype, 32, np.nanmax(np.abs(as_f64(v))))


def test_paged_cache_with_heads_before_rows(session, rt):
    """A cache stored [pages, Hkv, page, D], K and V interleaved in one tensor."""
    h, hk, d, page, dtype = 8, 2, 128, 16, DType.BF16
    lens, new = [70, 333], [1, 40]
    k, v, table = make_cache(lens, page, hk, d, dtype, 550)
    pages = k.shape[0]
    both = np.stack([k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)], 1).copy()  # [pages, 2, Hkv, page, D]
    base = upload(session, rt.stream, both, dtype)
    strides = (2 * hk * page * d, d, page * d, 1)
    caches = [view(session, base, i * hk * page * d, (pages, page, hk, d), strides) for i in range(2)]
    cu = prefix(new)
    q = rows((41, h, d), dtype, 551)
    ins = [upload(session, rt.stream, q, dtype), *caches, ints(session, rt, table), ints(session, rt, lens),
           ints(session, rt, cu)]
    got = rt.execute(tb.OpRequest("attention.paged", ins, [tb.TensorSpec(dtype, q.shape)], {})).wait()
    ref, mag = paged_reference(q, k, v, table, lens, cu, True, 1 / math.sqrt(d), np.zeros(q.shape))
    assert_attention(got.outputs[0].to_numpy(rt.stream), ref, mag, dtype, 333, np.nanmax(np.abs(as_f64(v))))


@pytest.mark.parametrize("candidate", ["attention_rows", "attention_tiles"])
@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.F16, 64)])
def test_each_candidate_takes_chunks(session, rt, candidate, dtype, d):
    name = check_varlen(session, rt, [130, 0, 1, 300], [64, 9, 500, 333], 8, 2, d, dtype, True, pad=2, seed=560,
                        candidate=candidate)
    assert name.startswith(candidate)
    name = check_paged(session, rt, [200, 333, 1200, 40], [200, 130, 1, 0], 8, 2, d, 16, dtype, pad=3, seed=570,
                       attrs={"candidate": candidate})
    assert name.startswith(candidate)


@pytest.mark.parametrize("candidate", ["attention_rows", "attention_tiles", "attention_tokens"])
def test_each_candidate_takes_single_tokens(session, rt, candidate):
    name = check_paged(session, rt, [700, 1, 65, 0], [1, 1, 1, 1], 8, 2, 128, 32, DType.BF16, pad=1, seed=580,
                       attrs={"candidate": candidate, "max_query_len": 1})
    assert name.startswith(candidate)


def test_the_default_kernel_follows_shapes_and_bounds(session, rt):
    one = dict(lens=[300, 20], new=[1, 1], h=8, hk=2, d=128, dtype=DType.BF16)
    assert check_paged(session, rt, page=16, attrs={"max_query_len": 1}, **one) == "attention_tokens_bf16_d128_r8"
    assert check_paged(session, rt, page=24, attrs={"max_query_len": 8}, **one) == "attention_tokens_bf16_d128_r8"
    few = {**one, "new": [4, 1]}
    assert check_paged(session, rt, page=24, attrs={"max_query_len": 4}, **few) == "attention_tokens_bf16_d128_r16"
    few = {**one, "new": [8, 3]}
    assert check_paged(session, rt, page=16, attrs={"max_query_len": 8}, **few) == "attention_tokens_bf16_d128_r32"
    long = dict(lens=[300, 60], new=[1, 40], h=8, hk=2, d=64, dtype=DType.F16)
    assert check_paged(session, rt, page=16, **long) == "attention_tiles_f16_d64"
    assert check_paged(session, rt, page=24, **long) == "attention_rows_f16"
    assert check_varlen(session, rt, [30], None, 4, 4, 128, DType.BF16, True) == "attention_tiles_bf16_d128"
    assert check_varlen(session, rt, [30], None, 4, 4, 96, DType.BF16, True) == "attention_rows_bf16"
    for attrs in ({"candidate": "attention_tokens"}, {"candidate": "attention_tiles"}):
        with pytest.raises(tb.ExecutionError, match="does not take"):
            check_paged(session, rt, page=24, attrs=attrs, **long)


def test_unknown_candidate_foreign_session_and_small_buffers(session, rt):
    q = upload(session, rt.stream, rows((4, 2, 64), DType.BF16, 1), DType.BF16)
    cu = ints(session, rt, [0, 4])
    spec = [tb.TensorSpec(DType.BF16, (4, 2, 64))]
    with pytest.raises(tb.ExecutionError, match="unknown attention.varlen candidate"):
        rt.execute(tb.OpRequest("attention.varlen", [q, q, q, cu], spec, {"candidate": "no_such_kernel"}))
    short = tb.TensorHandle(session, session.allocate(4 * 2 * 64 * 2 - 2), DType.BF16, (4, 2, 64), (128, 64, 1))
    with pytest.raises(tb.ExecutionError, match="does not hold"):
        rt.execute(tb.OpRequest("attention.varlen", [q, short, q, cu], spec))
    with pytest.raises(tb.ExecutionError, match="does not hold"):
        rt.execute(tb.OpRequest("attention.varlen", [q, q, q, cu], spec), output=short)
    wide = tb.TensorHandle(session, q.buffer, DType.BF16, (4, 2, 64), (2 ** 62, 64, 1))
    with pytest.raises(tb.ExecutionError, match="does not hold"):
        rt.execute(tb.OpRequest("attention.varlen", [wide, q, q, cu], spec))
    other = tb.Session(0)
    foreign = upload(other, other.create_stream(), rows((4, 2, 64), DType.BF16, 1), DType.BF16)
    foreign.session = session
    with pytest.raises(tb.ExecutionError, match="foreign buffer"):
        rt.execute(tb.OpRequest("attention.varlen", [q, foreign, q, cu], spec))
