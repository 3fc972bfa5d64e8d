"""Helpers of the serving-operator tests: attention and step planning restated in 64 bits with
numpy, and the tolerance of the 16-bit kernels (no test functions here)."""
from __future__ import annotations

import numpy as np

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

# Half a unit in the last place, relative to the value.
HALF_STEP = {DType.BF16: 2.0 ** -8, DType.F16: 2.0 ** -11}


def rows(shape, dtype: DType, seed: int, std: float = 1.0) -> np.ndarray:
    """Normal values in the dtype's storage form (uint16 bits for BF16, float16 for F16)."""
    x = tb.fill_normal(int(np.prod(shape)), seed=seed, std=std).reshape(shape)
    return tb.f32_to_bf16_bits(x) if dtype == DType.BF16 else x.astype(np.float16)


def as_f64(a: np.ndarray) -> np.ndarray:
    return (tb.bf16_bits_to_f32(a).reshape(a.shape) if a.dtype == np.uint16 else a).astype(np.float64)


def quiet_nan(dtype: DType):
    return np.uint16(0x7FC1) if dtype == DType.BF16 else np.float16(np.nan)


def one_request(q, k, v, causal, scale):
    """(O, A) of one request in 64 bits: q [Lq, H, D], k, v [Lk, Hkv, D]; A = sum_j p_j |v_j| is
    what the rounding of the probabilities is relative to."""
    lq, h, d = q.shape
    lk, hk = k.shape[0], k.shape[1]
    out, mag = np.zeros((lq, h, d)), np.zeros((lq, h, d))
    if lk == 0:
        return out, mag
    seen = np.arange(lk)[None, :] <= (np.arange(lq) + lk - lq)[:, None] if causal else np.ones((lq, lk), bool)
    for head in range(h):
        g = head // (h // hk)
        s = np.where(seen, scale * (q[:, head] @ k[:, g].T), -np.inf)
        top = np.max(s, axis=1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        total = p.sum(axis=1, keepdims=True)
        p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
        out[:, head], mag[:, head] = p @ v[:, g], p @ np.abs(v[:, g])
    return out, mag


def attention_tolerance(ref, mag, dtype, longest, v_max):
    """|error| allowed, from the arithmetic of the kernels (u = half a step of the type):
      u |O|                 the output's rounding;
      u A                   each probability is rounded to the type once;
      2^-11 A               fp32 scores: D <= 128 products of unit normals, |ds| <= 2^-23 D sum|q k| scale
                            = 1.1e-4, which moves p by at most 2 |ds|; fp32 sums over up to 4096 keys,
                            4096 x 2^-24 = 2.4e-4; ex2.approx 2^-22; together below 4.9e-4;
      longest 2^-25 max|v|  f16 probabilities below 2^-14 are rounded to multiples of 2^-24 (the row's
                            largest is at least 1).
    """
    u = HALF_STEP[dtype]
    return u * np.abs(ref) + (u + 2.0 ** -11) * mag + longest * 2.0 ** -25 * v_max + 1e-12


def assert_attention(got, ref, mag, dtype, longest, v_max):
    got = as_f64(got)
    assert np.isfinite(got).all()
    excess = np.abs(got - ref) - attention_tolerance(ref, mag, dtype, longest, v_max)
    at = np.unravel_index(np.argmax(excess), excess.shape)
    assert excess[at] <= 0, (at, got[at], ref[at], mag[at])


def varlen_reference(q, k, v, cu_q, cu_k, causal, scale, out):
    """`out` (64 bits, the buffer's contents before) with every request's rows written, and A."""
    q, k, v = as_f64(q), as_f64(k), as_f64(v)
    out, mag = out.copy(), np.zeros_like(out)
    for b in range(len(cu_q) - 1):
        sl, kl = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        out[sl], mag[sl] = one_request(q[sl], k[kl], v[kl], causal, scale)
    return out, mag


def gather(cache, table_row, length):
    """The first `length` rows of one request in a [pages, page, Hkv, D] cache; a page id that
    names no page reads as zeros."""
    pages, page = cache.shape[:2]
    got = np.zeros((length,) + cache.shape[2:])
    for j in range(length):
        i = table_row[j // page]
        if 0 <= i < pages:
            got[j] = as_f64(cache[i, j % page])
    return got


def paged_reference(q, k_cache, v_cache, table, lens, cu_q, causal, scale, out):
    q = as_f64(q)
    out, mag = out.copy(), np.zeros_like(out)
    for b in range(len(lens)):
        sl = slice(cu_q[b], cu_q[b + 1])
        out[sl], mag[sl] = one_request(q[sl], gather(k_cache, table[b], lens[b]), gather(v_cache, table[b], lens[b]),
                                       causal, scale)
    return out, mag


def plan_reference(ctx, new, free, table, tokens, page):
    """The step's tables as the operator documents them, request by request."""
    table = table.copy()
    batch, width = table.shape
    lens, cu, slots = np.zeros(batch, np.int64), np.zeros(batch + 1, np.int64), np.full(tokens, -1, np.int64)
    at = taken = given = refused = 0
    for b in range(batch):
        c, n = max(int(ctx[b]), 0), max(int(new[b]), 0)
        held, wanted = -(-c // page), -(-(c + n) // page)
        cu[b] = min(at, tokens)
        fits = ctx[b] >= 0 and new[b] >= 0 and c + n < 2 ** 31 and wanted <= width and at + n <= tokens
        need = wanted - held if fits else 0
        if fits and taken + need <= len(free):
            table[b, held:wanted] = free[taken:taken + need]
            lens[b] = c + n
            given += need
            for i in range(n):
                x = c + i
                slot = int(table[b, x // page]) * page + x % page
                slots[at + i] = slot if 0 <= slot <= 0x7FFFFFFF and table[b, x // page] >= 0 else -1
        else:
            refused += 1
            lens[b] = c
        taken += need
        at += n
    cu[batch] = min(at, tokens)
    return [a.astype(np.int32) for a in (table, lens, cu, slots, np.array([given, refused]))]
