// Attention over packed or paged sequences on the tensor cores: whole prompts and chunks of
// new tokens, head dimension 64 or 128, bf16 or f16, grouped heads.
//
//   O = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  s_j = q . k_j,  c = scale log2(e)
//
// A tile has 128 rows of M = (query row, head of the group) pairs: with G query heads to a
// key head, floor(128 / G) consecutive query rows times their G heads, which all read the
// same K and V. One CTA takes two such tiles, A and B, of one request and key head
// and walks the keys in tiles of 128 with the two-tile pipeline of the square attention kernel
// (sdpa_pair_common.cuh): while the tensor core runs one tile's products, the other's
// warpgroup exponentiates. Per CTA, three warpgroups:
//   warp 0       producer: Q once, then K_j and V_{j-1} into stage j & 1 of a 2-stage ring. A
//                packed key tile is one box; a paged one is 128 / page boxes, each lane copying
//                the page whose id it looked up one tile ahead. A page id that names no page, and
//                pages past the request's end, are given a coordinate outside the map, which
//                the copy fills with zeros.
//   warp 1       owns the tensor memory S_A | S_B | O_A | O_B; one lane issues the MMAs.
//   warp 2       clears the rows of the last V tile that lie past the request's end (another
//                request's, or whatever an unfinished page holds) between its copy and its
//                use: their probabilities are 0, but 0 x NaN is not. Scores of such keys are
//                replaced before use.
//   warps 4..11  softmax, one row a thread, warps 4-7 tile A, 8-11 tile B.
// When the calls' items cannot fill the SMs, each item's keys are cut into `parts`, whose
// unfinished (O, maximum, sum) go to the workspace; attention_tiles_join adds them up.
// Bound by the softmax and the single issuing lane beside the tensor core, as the square kernel.
// Every wait is bounded; on a timeout the kernel records a code, drains and returns.
#include <cuda_fp16.h>

#include "attn_params.cuh"
#include "sdpa_pair_common.cuh"

namespace {

using namespace tb;
using sdpa2::BM;
using sdpa2::BN;
using sdpa2::desc_add;
using sdpa2::mask_max_chunk;
using sdpa2::reg_fence;

constexpr float kLowest = -3.402823466e38f;
constexpr uint32_t kFailProducer = 0x56010000u;
constexpr uint32_t kFailMma = 0x56020000u;
constexpr uint32_t kFailSoftmax = 0x56030000u;
constexpr uint32_t kFailClear = 0x56040000u;
constexpr uint32_t kControlRegs = 56, kSoftmaxRegs = 216;
static_assert(128 * kControlRegs + 256 * kSoftmaxRegs <= kTileThreads * kTileLaunchRegs,
              "the warpgroups' registers exceed the launch allocation");

struct Barriers {
  uint64_t q_full;
  uint64_t kv_full[2], kv_empty[2];  // stage j & 1 holds K_j and V_{j-1}
  uint64_t s_full[2];                // per query tile (A, B)
  uint64_t p_half[2];                // per query tile: P of keys [0, 64) is in TMEM
  uint64_t p_full[2];                // per query tile: P of keys [64, 128) is in TMEM
  uint64_t v_raw;                    // the last V tile, before its rows past the end are cleared
  uint64_t o_final;
  uint64_t drain;
  uint32_t tmem_base;
};
static_assert(sizeof(Barriers) <= kTileBarrierBytes, "barrier block overflows its reservation");

struct Scratch {
  long long scan[kTileThreads / 32];
  long long found_before;
  int found;
};
static_assert(sizeof(Scratch) <= kTileScratchBytes, "scratch block overflows its reservation");

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  return pack_bf16x2(x, y);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;            // 64-dimension boxes of a row
  static constexpr int kHalfBytes = 128 * 128;       // 128 rows of one box
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr uint32_t kF16 = sizeof(T) == 2 && !__is_same(T, __nv_bfloat16);
  // The operand type fields of the instruction descriptor: 1 = bf16, 0 = f16.
  static constexpr uint32_t kTypes = kF16 ? (1u << 7) | (1u << 10) : 0u;
  static constexpr uint32_t kIdescS = idesc_bf16_f32(BM, BN, false) & ~kTypes;
  static constexpr uint32_t kIdescO = idesc_bf16_f32(BM, HD, true) & ~kTypes;
};

// Pairs of tiles of one request (0 where the token kernel takes it).
__device__ __forceinline__ int pairs_of(const AttnParams& p, const AttnRequest& r) {
  return is_token_request(p, r) ? 0 : (r.lq + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
}

// One 32-column chunk of S to probabilities in the values' type, and its part of the row sum.
template <typename T>
__device__ __forceinline__ void exp_chunk(const uint32_t (&cur)[32], float2 scale2, float2 neg_m2, float2 (&rs)[4],
                                          uint32_t p_tmem) {
  uint32_t packed[16];
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(cur[i]), __uint_as_float(cur[i + 1])), scale2, neg_m2);
    const float2 e = make_float2(exp2_mufu(x.x), exp2_mufu(x.y));
    rs[(i >> 1) & 3] = __fadd2_rn(rs[(i >> 1) & 3], e);
    packed[i / 2] = pack2<T>(e.x, e.y);
  }
  tmem_st_x16(p_tmem, packed);
}

template <int HD>
__device__ __forceinline__ void scale_o(uint32_t o_tmem, float alpha) {
#pragma unroll 1
  for (int c = 0; c < HD; c += 16) {
    uint32_t o[16];
    tmem_ld_x16(o_tmem + c, o);
    tmem_ld_wait();
    reg_fence(o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st_x16(o_tmem + c, o);
  }
}

// One key tile of one row's online softmax, as softmax_tile of the square kernel: the
// reference maximum m moves only when the row's maximum grows by more than 2^8, so P stays
// at or below 256. It starts at the lowest finite value, so a row (or a tile of it) without
// a visible key adds exp2(-inf) = 0.
template <typename T, int HD>
__device__ __forceinline__ void softmax_step(uint32_t s_tmem, uint32_t o_tmem, int valid, bool rescale, float scale2,
                                             float& m, float& l, uint64_t* p_half, uint64_t* p_full) {
  const int lane = lane_id();
  const bool need_mask = valid < BN;
  uint32_t c0[32], c1[32], c2[32], c3[32];
  tmem_ld_x32(s_tmem, c0);
  tmem_ld_x32(s_tmem + 32, c1);
  tmem_ld_x32(s_tmem + 64, c2);
  tmem_ld_x32(s_tmem + 96, c3);
  tmem_ld_wait();
  reg_fence(c0);
  reg_fence(c1);
  reg_fence(c2);
  reg_fence(c3);
  float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  mask_max_chunk(c0, valid, need_mask, mx4);
  mask_max_chunk(c1, valid - 32, need_mask, mx4);
  mask_max_chunk(c2, valid - 64, need_mask, mx4);
  mask_max_chunk(c3, valid - 96, need_mask, mx4);
  const float mx = fmaxf(fmax3f(mx4[0], mx4[1], mx4[2]), mx4[3]) * scale2;
  const bool grow = mx > m + sdpa2::kLazyRescaleLog2;
  if (__any_sync(0xffffffffu, grow)) {
    const float m_new = grow ? mx : m;
    const float alpha = exp2_mufu(m - m_new);
    l *= alpha;
    if (rescale) scale_o<HD>(o_tmem, alpha);
    m = m_new;
  }
  const float2 sc = make_float2(scale2, scale2), neg_m = make_float2(-m, -m);
  float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  exp_chunk<T>(c0, sc, neg_m, rs, s_tmem);
  exp_chunk<T>(c1, sc, neg_m, rs, s_tmem + 16);
  tmem_st_wait();
  tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) mbar_arrive(p_half);
  exp_chunk<T>(c2, sc, neg_m, rs, s_tmem + 32);
  exp_chunk<T>(c3, sc, neg_m, rs, s_tmem + 48);
  const float2 sum = __fadd2_rn(__fadd2_rn(rs[0], rs[1]), __fadd2_rn(rs[2], rs[3]));
  l += sum.x + sum.y;
  tmem_st_wait();
  tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) mbar_arrive(p_full);
}

template <typename T, int HD>
__device__ __forceinline__ void attention_tiles(const AttnParams& p, const CUtensorMap& tmap_q,
                                                const CUtensorMap& tmap_k, const CUtensorMap& tmap_v,
                                                uint32_t* status) {
  using S = Shape<T, HD>;
  constexpr int OFF_Q = 0, OFF_K = OFF_Q + 2 * S::kTileBytes, OFF_V = OFF_K + 2 * S::kTileBytes,
                OFF_BAR = OFF_V + 2 * S::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + OFF_BAR);
  Scratch* scratch = reinterpret_cast<Scratch*>(smem + OFF_BAR + kTileBarrierBytes);
  const int warp = warp_id(), lane = lane_id();
  const int group = p.heads / p.kv_heads;

  // ---- this CTA's item: (pair of tiles, key head, part), the longest rows first ----
  const auto units = [&](int b) { return pairs_of(p, request_of(p, b)); };
  const Stretch stretch = count_units<kTileThreads>(p.batch, scratch->scan, units);
  const long long items = stretch.total * p.kv_heads;
  // Parts of an item: as many as fill the SMs, when the caller gave a workspace for them.
  const int parts = p.work && items > 0 ? (int)max(1ll, min((long long)p.splits, gridDim.x / items)) : 1;
  if (p.work && blockIdx.x == 0 && threadIdx.x == 0) {
    int* head = reinterpret_cast<int*>(p.work + 4ull * kTokenCounters);
    head[0] = parts > 1 ? (int)items : 0;
    head[1] = parts;
  }
  const long long item = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  if (item >= items) return;
  const long long unit = stretch.total - 1 - item / p.kv_heads;
  const int hk = (int)(item % p.kv_heads);
  find_unit(stretch, unit, units, &scratch->found, &scratch->found_before);
  const int b = scratch->found;
  const AttnRequest r = request_of(p, b);
  const int tok0 = (int)(unit - scratch->found_before) * 2 * p.tile_tokens;  // tile A's first query row
  const bool has_b = tok0 + p.tile_tokens < r.lq;
  // Key tiles that each tile needs (of its last row), and this part's range of them.
  const int end_a = (visible_keys(p, r, min(tok0 + p.tile_tokens, r.lq) - 1) + BN - 1) / BN;
  const int end_b = has_b ? (visible_keys(p, r, min(tok0 + 2 * p.tile_tokens, r.lq) - 1) + BN - 1) / BN : 0;
  const int all = max(end_a, end_b);
  const int lo = (int)((long long)part * all / parts), hi = (int)((long long)(part + 1) * all / parts);
  const int n_a = max(0, min(hi, end_a) - lo), n_b = max(0, min(hi, end_b) - lo), n = hi - lo;
  // Whether this part's last key tile runs past the request's end.
  const int last_rows = r.lk % BN;
  const bool clear = last_rows && n > 0 && hi == r.lk / BN + 1;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_half[i], 4);
      mbar_init(&bars->p_full[i], 4);
    }
    mbar_init(&bars->v_raw, 1);
    mbar_init(&bars->o_final, 1);
    mbar_init(&bars->drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;

  if (warp < 4) {
    setmaxnreg_dec<kControlRegs>();
    if (warp == 0 && n > 0) {
      // ---------------- producer ----------------
      if (lane == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
        const uint32_t bytes = S::kHalves * p.tile_tokens * group * 128;
        mbar_arrive_expect_tx(&bars->q_full, bytes * (has_b ? 2 : 1));
        for (int x = 0; x < (has_b ? 2 : 1); ++x)
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_3d(smem + OFF_Q + x * S::kTileBytes + h * S::kHalfBytes, &tmap_q, &bars->q_full, 64 * h,
                        hk * group, r.q0 + tok0 + x * p.tile_tokens);
      }
      __syncwarp();
      // Lane i copies box i of a key tile: rows [i box, (i + 1) box) of it.
      const bool paged = p.table != 0;
      const int box = paged ? min(p.page, BN) : BN, boxes = BN / box;
      const bool active = lane < boxes;
      const int held = paged ? (r.lk + p.page - 1) / p.page : 0;  // pages of the request
      // The coordinates of the lane's box of key tile j: (row, page).
      const auto row_of = [&](int j) { return paged ? (p.page > BN ? j * BN % p.page : 0) : r.k0 + j * BN; };
      const auto page_at = [&](int j) {
        if (!paged || !active || j >= hi) return 0;
        const int index = p.page > BN ? (int)((long long)j * BN / p.page) : j * boxes + lane;
        const int id = index < held ? page_of(p, b, index) : -1;
        return id < 0 ? p.pages : id;
      };
      const auto load = [&](int off, const CUtensorMap* map, uint64_t* bar, int j, int w) {
        if (!active) return;
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
          tma_load_4d(smem + off + h * S::kHalfBytes + lane * box * 128, map, bar, 64 * h, hk, row_of(j), w);
      };
      const auto prefetch = [&](int j, int w) {
        if (!active || j >= hi || (paged && w == p.pages)) return;
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
          tma_prefetch_l2_4d(&tmap_k, 64 * h, hk, row_of(j), w);
          tma_prefetch_l2_4d(&tmap_v, 64 * h, hk, row_of(j), w);
        }
      };
      int w_old = 0, w_now = page_at(lo), w_next = page_at(lo + 1);
      uint32_t issued[2] = {0, 0};
      bool ok = true;
      for (int it = 0; it <= n; ++it) {
        const int w_after = page_at(lo + it + 2);
        prefetch(lo + it + 1, w_next);
        const int st = it & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->kv_empty[st], ((it >> 1) & 1) ^ 1));
        if (!ok) {
          if (lane == 0) report_status(status, kFailProducer | 1);
          break;
        }
        const bool has_k = it < n, has_v = it >= 1;
        // The last iteration brings a V tile only; one to be cleared goes to warp 2 first,
        // which arrives on kv_full for it.
        uint64_t* full = clear && it == n ? &bars->v_raw : &bars->kv_full[st];
        if (lane == 0) mbar_arrive_expect_tx(full, (has_k ? S::kTileBytes : 0) + (has_v ? S::kTileBytes : 0));
        __syncwarp();
        if (has_k) load(OFF_K + st * S::kTileBytes, &tmap_k, full, lo + it, w_now);
        if (has_v) load(OFF_V + st * S::kTileBytes, &tmap_v, full, lo + it - 1, w_old);
        ++issued[st];
        w_old = w_now;
        w_now = w_next;
        w_next = w_after;
      }
      if (!ok) {
        if (!mbar_wait(&bars->q_full, 0)) report_status(status, kFailProducer | 3);
        for (int s = 0; s < 2; ++s)
          if (issued[s] && !mbar_wait(&bars->kv_full[s], (issued[s] - 1) & 1))
            report_status(status, kFailProducer | 4);
      }
    } else if (warp == 1) {
      if (lane == 0 && n > 0) {
        // ---------------- MMA issuer ----------------
        bool ok = mbar_wait(&bars->q_full, 0);
        if (!ok) report_status(status, kFailMma | 1);
        const uint64_t qd_a = sdesc_sw128(smem_addr(smem + OFF_Q), 16, 1024);
        const uint64_t qd_b = sdesc_sw128(smem_addr(smem + OFF_Q + S::kTileBytes), 16, 1024);
        const uint64_t kd0 = sdesc_sw128(smem_addr(smem + OFF_K), 16, 1024);
        const uint64_t vd0 = sdesc_sw128(smem_addr(smem + OFF_V), S::kHalfBytes, 1024);
        for (int j = 0; j <= n && ok; ++j) {
          const int st = j & 1;
          const uint64_t kd = desc_add(kd0, st * (S::kTileBytes >> 4));
          const uint64_t vd = desc_add(vd0, st * (S::kTileBytes >> 4));
          if (!mbar_wait(&bars->kv_full[st], (j >> 1) & 1)) {
            report_status(status, kFailMma | 2);
            ok = false;
            break;
          }
          for (int x = 0; x < 2; ++x) {
            const int nx = x ? n_b : n_a;
            const uint32_t s_tmem = tmem + x * BN, o_tmem = tmem + (2 + x) * BN;
            if (j >= 1 && j - 1 < nx) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!mbar_wait(half ? &bars->p_full[x] : &bars->p_half[x], (j - 1) & 1)) {
                  report_status(status, kFailMma | 3);
                  ok = false;
                  break;
                }
                tc_fence_after_sync();
#pragma unroll
                for (int k = 4 * half; k < 4 * half + 4; ++k)
                  umma_bf16_ts(o_tmem, s_tmem + k * 8, desc_add(vd, k * (2048 >> 4)), S::kIdescO,
                               (k > 0 || j > 1) ? 1u : 0u);
              }
              if (!ok) break;
            }
            if (j < nx) {
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t off = (k >> 2) * (S::kHalfBytes >> 4) + (k & 3) * 2;
                umma_bf16_ss(s_tmem, desc_add(x ? qd_b : qd_a, off), desc_add(kd, off), S::kIdescS, k > 0 ? 1u : 0u);
              }
              umma_commit(&bars->s_full[x]);
            }
          }
          if (!ok) break;
          umma_commit(&bars->kv_empty[st]);
        }
        umma_commit(&bars->o_final);
        umma_commit(&bars->drain);
        if (!mbar_wait(&bars->drain, 0)) report_status(status, kFailMma | 5);
      }
    } else if (warp == 2 && clear) {
      // ---------------- rows of the last V tile past the request's end ----------------
      const int st = n & 1;
      const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_raw, 0));
      if (ok) {
        const int words = (BN - last_rows) * 8;  // 16-byte words of one half
        for (int h = 0; h < S::kHalves; ++h) {
          uint4* at = reinterpret_cast<uint4*>(smem + OFF_V + st * S::kTileBytes + h * S::kHalfBytes + last_rows * 128);
          for (int i = lane; i < words; i += 32) at[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->kv_full[st]);
      } else if (lane == 0) {
        report_status(status, kFailClear | 1);
      }
    }
  } else {
    setmaxnreg_inc<kSoftmaxRegs>();
    // ---------------- softmax warpgroups ----------------
    const int x = warp >= 8 ? 1 : 0;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lane_off + x * BN;
    const uint32_t o_tmem = tmem + lane_off + (2 + x) * BN;
    const int i = tok0 + x * p.tile_tokens + row / group;  // the query row in its request
    const bool in = row < p.tile_tokens * group && i < r.lq;
    // Rows of no query compute on whatever is there and are not stored.
    const int seen = in ? visible_keys(p, r, i) : r.lk;
    const int nx = x ? n_b : n_a;
    const float scale2 = p.scale * 1.4426950408889634f;
    float m = kLowest, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nx; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[x], j & 1));
      if (!ok) {
        if (lane == 0) report_status(status, kFailSoftmax | 1);
        break;
      }
      tc_fence_after_sync();
      softmax_step<T, HD>(s_tmem, o_tmem, seen - (lo + j) * BN, j > 0, scale2, m, l, &bars->p_half[x],
                          &bars->p_full[x]);
    }
    if (ok && n > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_final, 0));
      if (!ok && lane == 0) report_status(status, kFailSoftmax | 2);
      tc_fence_after_sync();
    }
    if (ok) {
      const long long place =
          in ? (long long)(r.q0 + i) * p.o_tok + (long long)(hk * group + row % group) * p.o_head : -1;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const long long slot = item * parts + part;
      const int slots = (int)gridDim.x;
      if (parts > 1) {
        if (part == 0) reinterpret_cast<long long*>(p.work + tile_places_at())[item * kTileRows + x * 128 + row] = place;
        reinterpret_cast<float2*>(p.work + tile_stats_at(slots))[slot * kTileRows + x * 128 + row] = make_float2(m, l);
      }
      float* part_row = reinterpret_cast<float*>(p.work + tile_rows_at(slots)) + (slot * kTileRows + x * 128 + row) * HD;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (nx > 0) {
          tmem_ld_x32(o_tmem + c, o);
          tmem_ld_wait();
          reg_fence(o);
        } else {
#pragma unroll
          for (int q = 0; q < 32; ++q) o[q] = 0u;
        }
        if (in && parts > 1) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            reinterpret_cast<uint4*>(part_row + c)[q] = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        } else if (in) {
          uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + place + c);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 w;
            w.x = pack2<T>(__uint_as_float(o[8 * q + 0]) * inv, __uint_as_float(o[8 * q + 1]) * inv);
            w.y = pack2<T>(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv);
            w.z = pack2<T>(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv);
            w.w = pack2<T>(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv);
            to[q] = w;
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts of every row, one warp a row: M = max m_i, O = sum 2^(m_i - M) O_i /
// sum 2^(m_i - M) l_i. Leaves at once when the call was not split.
template <typename T, int HD>
__device__ __forceinline__ void join_tiles(const AttnParams& p, int slots) {
  const int* head = reinterpret_cast<const int*>(p.work + 4ull * kTokenCounters);
  const long long rows = (long long)head[0] * kTileRows;
  const int parts = head[1];
  const int lane = threadIdx.x & 31;
  constexpr int kPer = HD / 32;
  for (long long u = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < rows;
       u += (long long)gridDim.x * (blockDim.x >> 5)) {
    const long long place = reinterpret_cast<const long long*>(p.work + tile_places_at())[u];
    if (place < 0) continue;
    const long long item = u / kTileRows, row = u % kTileRows;
    float m = kLowest, l = 0.f, acc[kPer];
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
    for (int i = 0; i < parts; ++i) {
      const long long at = (item * parts + i) * kTileRows + row;
      const float2 st = reinterpret_cast<const float2*>(p.work + tile_stats_at(slots))[at];
      const float* o = reinterpret_cast<const float*>(p.work + tile_rows_at(slots)) + at * HD + lane * kPer;
      const float big = fmaxf(m, st.x);
      const float f = exp2_mufu(m - big), g = exp2_mufu(st.x - big);
      m = big;
      l = l * f + st.y * g;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] = acc[c] * f + o[c] * g;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint32_t* to = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.o) + place + lane * kPer);
#pragma unroll
    for (int c = 0; c < kPer; c += 2) to[c / 2] = pack2<T>(acc[c] * inv, acc[c + 1] * inv);
  }
}

}  // namespace

// One CTA per SM at 168 registers a thread; the warpgroups re-divide them (56 and 216).
#define TB_TILE_ENTRY(suffix, T, HD)                                                                                \
  extern "C" __global__ void __launch_bounds__(tb::kTileThreads, 1)                                                 \
      attention_tiles_##suffix(const __grid_constant__ tb::AttnParams p, const __grid_constant__ CUtensorMap tmap_q, \
                               const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, \
                               uint32_t* status) {                                                                  \
    attention_tiles<T, HD>(p, tmap_q, tmap_k, tmap_v, status);                                                      \
  }                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(256) attention_tiles_join_##suffix(                                  \
      const __grid_constant__ tb::AttnParams p, int slots) {                                                        \
    join_tiles<T, HD>(p, slots);                                                                                    \
  }

TB_TILE_ENTRY(bf16_d128, __nv_bfloat16, 128)
TB_TILE_ENTRY(bf16_d64, __nv_bfloat16, 64)
TB_TILE_ENTRY(f16_d128, __half, 128)
TB_TILE_ENTRY(f16_d64, __half, 64)
