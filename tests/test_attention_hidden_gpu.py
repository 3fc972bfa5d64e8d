"""Bits behind the causal mask: infinities and NaNs in K and V rows that a query row may not see
leave its result as it was, bit for bit, and reach the rows that see them."""
import math

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import as_f64, rows
from test_attention_serving_gpu import ints, make_cache, prefix, run_paged, run_varlen

pytestmark = pytest.mark.gpu

SPECIAL = {DType.BF16: [np.uint16(x) for x in (0x7FC1, 0x7F80, 0xFF80)],
           DType.F16: [np.float16(x) for x in (np.nan, np.inf, -np.inf)]}


@pytest.fixture(scope="module")
def session():
    s = tb.Session(0)
    yield s
    s.close()


@pytest.fixture(scope="module")
def rt(session):
    return tb.Runtime(session)


def poison(v, dtype, seed, keys):
    """V [n, Hkv, D] with a NaN, +inf or -inf in some dimensions of these keys, and what they add to a
    row that sees its first s keys: added[s] [Hkv, D] (0 where nothing is added)."""
    rng = np.random.default_rng(seed)
    v = v.copy()
    added = np.zeros((v.shape[0] + 1,) + v.shape[1:])
    step = np.zeros(v.shape)
    for key in keys:
        hit = rng.random(v.shape[1:]) < 0.2
        kind = rng.integers(0, 3, v.shape[1:])
        for i, x in enumerate((np.nan, np.inf, -np.inf)):
            v[key][hit & (kind == i)] = SPECIAL[dtype][i]
            step[key][hit & (kind == i)] = x
    with np.errstate(invalid="ignore"):
        np.cumsum(step, axis=0, out=added[1:])
    return v, added


def check(base, got, added, seen, group):
    """`got` [lq, H, D] against the run without poison: special values where a row sees some, else its bits."""
    for i, s in enumerate(seen):
        want = np.repeat(added[s], group, axis=0)
        same = want == 0
        np.testing.assert_array_equal(got[i][same], base[i][same], err_msg=f"row {i}")
        np.testing.assert_array_equal(as_f64(got[i])[~same], want[~same], err_msg=f"row {i}")


def poisoned_keys(n, lq, rng):
    """Keys that some rows see and others do not, and one or two that all see."""
    late = [n - 1 - int(x) for x in rng.integers(0, max(1, min(lq, n)), 6)] if n else []
    return sorted(set(late + [int(x) for x in rng.integers(0, n, 1)])) if n else []


@pytest.mark.parametrize("candidate", ["attention_tiles", "attention_rows"])
@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.BF16, 64), (DType.F16, 128), (DType.F16, 64)])
@pytest.mark.parametrize("h,hk", [(2, 2), (8, 2), (5, 1), (40, 1)])
@pytest.mark.parametrize("lq,lk", [([300, 1, 128, 0, 77], None), ([40, 256, 3], [200, 256, 700]),
                                   ([300, 70], [130, 64]), ([1, 1, 2], [64, 129, 128])], ids=str)
def test_packed_rows_do_not_see_behind_the_mask(session, rt, lq, lk, h, hk, dtype, d, candidate):
    lk = lk or lq
    cu_q, cu_k = prefix(lq), prefix(lk)
    rng = np.random.default_rng(sum(lq) + h + d)
    q = rows((int(cu_q[-1]), h, d), dtype, 1)
    k, v = rows((int(cu_k[-1]), hk, d), dtype, 2), rows((int(cu_k[-1]), hk, d), dtype, 3)
    out = np.zeros(q.shape, q.dtype)
    attrs = {"causal": True, "candidate": candidate}
    bad, added = v.copy(), []
    for b in range(len(lk)):
        sl = slice(cu_k[b], cu_k[b + 1])
        bad[sl], more = poison(v[sl], dtype, 7 + b, poisoned_keys(lk[b], lq[b], rng))
        added.append(more)
    _, base = run_varlen(session, rt, q, k, v, cu_q, cu_k, out, dtype, attrs)
    name, got = run_varlen(session, rt, q, k, bad, cu_q, cu_k, out, dtype, attrs)
    assert name.startswith(candidate)
    for b in range(len(lk)):
        seen = np.clip(lk[b] - lq[b] + np.arange(lq[b]) + 1, 0, lk[b])
        sl = slice(cu_q[b], cu_q[b + 1])
        check(base[sl], got[sl], added[b], seen, h // hk)


@pytest.mark.parametrize("candidate,lens,new,h,hk", [
    ("attention_tiles", [300, 5, 140], [200, 5, 60], 8, 2), ("attention_tiles", [5000, 64], [70, 40], 4, 1),
    ("attention_tiles", [700, 129, 20], [8, 2, 30], 8, 1), ("attention_tokens", [300, 5, 64, 200], [8, 5, 2, 1], 4, 4),
    ("attention_tokens", [300, 5, 70, 3000], [4, 2, 3, 4], 8, 2), ("attention_tokens", [129, 20, 3000], [8, 30, 5], 1, 1),
    ("attention_tokens", [129, 2, 3000], [8, 8, 5], 8, 2), ("attention_rows", [129, 2, 300], [8, 8, 5], 8, 2)])
@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.F16, 64)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_new_tokens_do_not_see_behind_the_mask(session, rt, candidate, lens, new, h, hk, dtype, d, page):
    cu = prefix(new)
    rng = np.random.default_rng(sum(lens) + h + d + page)
    q = rows((int(cu[-1]), h, d), dtype, 11)
    k, v, table = make_cache(lens, page, hk, d, dtype, 12)
    out = np.zeros(q.shape, q.dtype)
    attrs = {"candidate": candidate, "max_query_len": max(new)}
    bad, added = v.copy(), []
    for b, n in enumerate(lens):
        at = table[b, np.arange(n) // page], np.arange(n) % page
        bad[at], more = poison(v[at], dtype, 17 + b, poisoned_keys(n, new[b], rng))
        added.append(more)
    _, base = run_paged(session, rt, q, k, v, table, lens, cu, out, dtype, attrs)
    name, got = run_paged(session, rt, q, k, bad, table, lens, cu, out, dtype, attrs)
    assert name.startswith(candidate)
    for b, n in enumerate(lens):
        seen = np.clip(n - new[b] + np.arange(new[b]) + 1, 0, n)
        sl = slice(cu[b], cu[b + 1])
        check(base[sl], got[sl], added[b], seen, h // hk)


@pytest.mark.parametrize("candidate", ["attention_tiles", "attention_tokens", "attention_rows"])
def test_keys_behind_the_mask_may_hold_anything(session, rt, candidate):
    """NaNs and infinities in K rows: the rows that do not see them keep their bits, the others are NaN."""
    h, hk, d, page, dtype, lens, new = 4, 2, 128, 16, DType.BF16, [130, 40], [6, 4]
    cu = prefix(new)
    q = rows((10, h, d), dtype, 21)
    k, v, table = make_cache(lens, page, hk, d, dtype, 22)
    out = np.zeros(q.shape, q.dtype)
    attrs = {"candidate": candidate, "max_query_len": 6}
    _, base = run_paged(session, rt, q, k, v, table, lens, cu, out, dtype, attrs)
    for b, key in ((0, 127), (0, 128), (1, 38)):
        for x in SPECIAL[dtype]:
            bad = k.copy()
            bad[table[b, key // page], key % page, :, ::3] = x
            _, got = run_paged(session, rt, q, bad, v, table, lens, cu, out, dtype, attrs)
            for i in range(cu[-1]):
                own = int(i >= cu[1])
                sees = own == b and key < lens[b] - new[b] + (i - cu[b]) + 1
                if sees and x == SPECIAL[dtype][0]:
                    assert np.isnan(as_f64(got[i])).all()
                elif not sees:
                    np.testing.assert_array_equal(got[i], base[i])
