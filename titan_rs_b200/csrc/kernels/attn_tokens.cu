// Attention of a few query rows per request over a long paged cache: the decode step.
//
//   O = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  s_j = q . k_j,  c = scale log2(e)
//
// Every cached row is read once for the G x Lq (query row, head) pairs of its key head, so at
// 2 G Lq flops a byte the kernel is bound by the HBM, and the design serves the loads:
//   - One list of 64-key tiles over all (request, key head) pairs is cut into equal runs, one
//     per resident CTA, so requests of any lengths load the SMs evenly. A pair that
//     is cut leaves partial results (O, m, sum) in the workspace; the CTA that finishes it
//     last adds them up in the order of the runs, so the result does not depend on who is last.
//   - Tiles arrive in a ring of shared-memory stages by 16-byte cp.async, which takes any
//     page size and cache layout, and fills rows past the sequence's end (and of page ids
//     that name no page) with zeros: their bits never reach a product. Page ids are read
//     one tile ahead of the copies that need them.
//   - The products run as S^T = K Q^T and O^T = V^T P^T on m16n8k16 tensor-core
//     instructions: keys and dimensions fill the 16 rows, the few query rows the 8
//     columns (a tcgen05 tile has 64 or 128 rows, of which a decode step would fill 8). Each
//     warp takes 16 keys of a tile with a maximum and sum of its own, so the warps
//     meet only for the stage hand-over; they are joined when the pair ends.
//   - Three CTAs an SM with two stages each where the query rows are eight or fewer, two with three
//     stages where more rows take the registers. What bounds a tile's step is the latency of its
//     chain (wait, first product, softmax, second product) and not the depth of the ring, so more
//     warps help and fewer do not: 64 requests of 300-8192 keys (544 MB) 97 us against 108
//     with two CTAs of three stages, 131 with three of 32-key tiles and 127 with one of 128-key
//     tiles; four of 110-131 thousand (2.0 GB) 304 us against 330 (launches in a row on one
//     board). With the caches emptied in between, over the boards seen: 95 to 99 us (5.5 to 5.7
//     TB/s) and 304 to 319 (6.3 to 6.6). A kernel that only reads as many bytes takes 79 and 276.
//   - 17 to 32 query rows of dimension 128 take all 255 registers and spill 316 bytes a thread.
// Scores, statistics and O are fp32; P is rounded to the values' type for the second product (at
// most 2^8, in f16 2^15: the reference maximum moves only when a row's maximum grows by more than
// 2^8).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_math.cuh"
#include "attn_params.cuh"

namespace {

using namespace tb;

constexpr int kTile = kTokenTile;  // 16 keys a warp
constexpr int kThreads = kTokenThreads;
constexpr int kWarps = kThreads / 32;
static_assert(kTile == 16 * kWarps && kThreads > kTile, "a warp takes 16 keys of a tile, a thread looks a row up");
constexpr float kLowest = -3.402823466e38f;
// Tiles of a CTA at least, where there are so many (11.4 us for 1018 keys of eight heads; 14.0
// with three, 13.2 with four).
constexpr int kMinRun = 2;

template <int D>
TB_BOTH constexpr int stage_bytes() { return 2 * kTile * D * 2; }

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes to shared memory without a register, or 16 zero bytes.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void load_matrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrix_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Half<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

__device__ __forceinline__ void add_scaled(float4& a, const float4& v, float f) {
  a.x = fmaf(v.x, f, a.x);
  a.y = fmaf(v.y, f, a.y);
  a.z = fmaf(v.z, f, a.z);
  a.w = fmaf(v.w, f, a.w);
}

// Four elements of a finished row, O / sum (zeros where no key was seen).
template <typename T>
__device__ __forceinline__ void store_row4(T* to, const float4& o, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const uint32_t lo = Half<T>::pack(o.x * inv, o.y * inv), hi = Half<T>::pack(o.z * inv, o.w * inv);
  if ((reinterpret_cast<uintptr_t>(to) & 7) == 0) {
    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
  } else {  // a row that starts at an odd element
    reinterpret_cast<uint16_t*>(to)[0] = (uint16_t)lo;
    reinterpret_cast<uint16_t*>(to)[1] = (uint16_t)(lo >> 16);
    reinterpret_cast<uint16_t*>(to)[2] = (uint16_t)hi;
    reinterpret_cast<uint16_t*>(to)[3] = (uint16_t)(hi >> 16);
  }
}

// The warp's 16 rows of V at `vs`, of keys from `key0` on: infinities and NaNs become zeros, and are
// added to O of the query rows that see their keys. All lanes.
template <typename T, int D, int NT>
__device__ __forceinline__ void take_special(uint32_t vs, int key0, const int (&seen)[NT][2],
                                             float (&o)[NT][D / 16][4]) {
  constexpr uint32_t kExponent = __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  constexpr int kChunks = D / 8;
  const int lane = threadIdx.x & 31;
  bool any = false;
#pragma unroll 1
  for (int i = lane; i < 16 * kChunks * 2; i += 32) {
    uint2 x;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(vs + i * 8) : "memory");
    any |= (x.x & kExponent) == kExponent || (x.x >> 16 & kExponent) == kExponent ||
           (x.y & kExponent) == kExponent || (x.y >> 16 & kExponent) == kExponent;
  }
  if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // dimension k * 16 + h * 8 + lane / 4, as o holds them
        uint16_t x;
        asm volatile("ld.shared.u16 %0, [%1];"
                     : "=h"(x) : "r"(vs + r * (D * 2) + (((k * 2 + h) ^ (r & 7)) << 4) + (lane >> 2) * 2) : "memory");
        if ((x & kExponent) != kExponent) continue;
        const float v = (float)*reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (key0 + r < seen[t][i]) o[t][k][2 * h + i] += v;
      }
    }
  }
  __syncwarp();
#pragma unroll 1
  for (int i = lane; i < 16 * kChunks * 4; i += 32) {
    uint32_t x;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(vs + i * 4) : "memory");
    if ((x & kExponent) == kExponent) x &= 0xffff0000u;
    if ((x >> 16 & kExponent) == kExponent) x &= 0xffffu;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(vs + i * 4), "r"(x) : "memory");
  }
  __syncwarp();
}

// Tiles of one (request, key head) pair; 0 for a request that is not this kernel's. A
// request without keys has one empty tile, which writes its zeros.
__device__ __forceinline__ int tiles_of(const AttnParams& p, const AttnRequest& r) {
  return is_token_request(p, r) ? max(1, (r.lk + kTile - 1) / kTile) : 0;
}

// A position in the list of tiles: request-major, then key heads, then tiles.
struct Cursor {
  int b, head, tile, tiles;
  AttnRequest r;

  // To request `from` or the first one behind it that has tiles.
  __device__ __forceinline__ void seek(const AttnParams& p, int from) {
    head = tile = 0;
    tiles = 0;
    for (b = from; b < p.batch; ++b) {
      r = request_of(p, b);
      tiles = tiles_of(p, r);
      if (tiles) break;
    }
  }
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++head < p.kv_heads) return;
    seek(p, b + 1);
  }
};

// What a tile's copies need: where its rows lie, and, in a pair's first tile of the run, which
// query rows come with it.
struct TileRows {
  long long k[kTile], v[kTile];  // element offsets, or -1 for a row of zeros
};
struct PairRows {
  int q_row, rows, head;  // first row of q, (query row, head) pairs (0: not a first tile), key head
};

template <int D, int kRows>
struct Shared {
  static constexpr int kStages = token_stages(kRows);
  alignas(128) uint8_t stage[kStages][stage_bytes<D>()];  // K rows, then V rows; 16-byte chunks swizzled by row
  alignas(16) uint8_t q[kRows <= 16 ? 2 : 0][kRows * D * 2 + (kRows <= 16 ? 0 : 16)];
  TileRows at[kStages];
  float top[kWarps][8], sum[kWarps][8];
  PairRows pair[kStages];
  long long scan[kThreads / 32], found_before;
  int found_b, last;
};

template <typename T, int D, int NT>
__device__ __forceinline__ void attention_tokens(const AttnParams& p) {
  constexpr int kRows = 8 * NT, kStages = token_stages(kRows);
  constexpr bool kQShared = kRows <= 16;  // Q comes through shared memory, else by plain loads
  extern __shared__ uint8_t raw[];
  using Smem = Shared<D, kRows>;
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~uintptr_t(127));
  constexpr int kChunks = D / 8;                    // 16-byte chunks of a row
  constexpr int kRowsAtOnce = kThreads / kChunks;   // rows one pass of the CTA copies
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = p.heads / p.kv_heads;

  begin_after_earlier_grids();
  // ---- this CTA's run of tiles ----
  const auto units = [&](int b) { return tiles_of(p, request_of(p, b)); };
  const Stretch stretch = count_units<kThreads>(p.batch, sm.scan, units);
  const long long total = stretch.total * p.kv_heads;
  const long long ctas = min((long long)gridDim.x, max(1ll, total / kMinRun));
  if (blockIdx.x >= ctas || total == 0) return;
  const long long begin = blockIdx.x * total / ctas, end = (blockIdx.x + 1) * total / ctas;
  // The tiles of a request start at kv_heads x (tiles before it).
  find_unit(stretch, begin / p.kv_heads, units, &sm.found_b, &sm.found_before);
  Cursor cur;
  cur.seek(p, sm.found_b);
  {
    const long long inside = begin - sm.found_before * p.kv_heads;
    cur.head = (int)(inside / cur.tiles);
    cur.tile = (int)(inside % cur.tiles);
  }
  Cursor ahead = cur;  // of the next tile whose rows are looked up
  const int count = (int)(end - begin);

  // Row offsets of tile `ahead`, by the first kTile threads.
  auto look_up = [&](long long& k_off, long long& v_off) {
    const int j = ahead.tile * kTile + tid;
    k_off = v_off = -1;
    if (tid < kTile && j < ahead.r.lk) {
      const int id = page_of(p, ahead.b, j / p.page);
      if (id >= 0) {
        const int row = j % p.page;
        k_off = id * p.k_page + row * p.k_tok + ahead.head * p.k_head;
        v_off = id * p.v_page + row * p.v_tok + ahead.head * p.v_head;
      }
    }
  };
  auto pair_of = [&](int n) {
    return PairRows{ahead.r.q0, n == 0 || ahead.tile == 0 ? ahead.r.lq * group : 0, ahead.head};
  };
  auto publish = [&](int n, long long k_off, long long v_off, const PairRows& pair) {
    if (tid < kTile) {
      sm.at[n % kStages].k[tid] = k_off;
      sm.at[n % kStages].v[tid] = v_off;
    }
    if (tid == kTile) sm.pair[n % kStages] = pair;
  };
  // Copies of tile n (its offsets are in shared memory) into its stage, and of the query rows
  // of a pair that begins with it into the Q block that its number says.
  const int chunk = tid % kChunks, row0 = tid / kChunks;
  int q_next = 0;
  auto copy_tile = [&](int n) {
    const uint32_t base = smem_of(sm.stage[n % kStages]);
    const TileRows& rows = sm.at[n % kStages];
#pragma unroll
    for (int r = row0; r < kTile; r += kRowsAtOnce) {
      const uint32_t at = base + r * (D * 2) + ((chunk ^ (r & 7)) << 4);
      const long long k = rows.k[r], v = rows.v[r];
      copy16(at, reinterpret_cast<const T*>(p.k) + (k < 0 ? 0 : k) + chunk * 8, k >= 0);
      copy16(at + kTile * D * 2, reinterpret_cast<const T*>(p.v) + (v < 0 ? 0 : v) + chunk * 8, v >= 0);
    }
    if constexpr (kQShared) {
      const PairRows pair = sm.pair[n % kStages];
      if (pair.rows) {
        const uint32_t to = smem_of(sm.q[q_next]);
        q_next ^= 1;
#pragma unroll
        for (int r = row0; r < kRows; r += kRowsAtOnce) {
          const bool in = r < pair.rows;
          const T* from = reinterpret_cast<const T*>(p.q) +
                          (in ? (pair.q_row + r / group) * p.q_tok + (pair.head * group + r % group) * p.q_head : 0);
          copy16(to + r * (D * 2) + ((chunk ^ (r & 7)) << 4), from + chunk * 8, in);
        }
      }
    }
  };

  long long k_next[kStages], v_next[kStages];
  {
    PairRows pairs[kStages];
#pragma unroll
    for (int n = 0; n < kStages; ++n) {
      if (n < count) {
        look_up(k_next[n], v_next[n]);
        pairs[n] = pair_of(n);
        ahead.next(p);
      }
    }
#pragma unroll
    for (int n = 0; n < kStages; ++n)
      if (n < count) publish(n, k_next[n], v_next[n], pairs[n]);
  }
  __syncthreads();
  for (int n = 0; n < kStages - 1; ++n) {
    if (n < count) copy_tile(n);
    copies_commit();
  }

  uint32_t qf[NT][D / 16][2];  // Q^T fragments
  float o[NT][D / 16][4];      // O^T: dimensions x query rows
  float top[NT][2], sum[NT][2];
  int seen[NT][2];             // visible keys of the thread's query rows
  const float scale2 = p.scale * 1.4426950408889634f;
  bool fresh = true;
  int q_now = 0;
  for (int n = 0; n < count; ++n) {
    if (!kQShared && fresh) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int row = t * 8 + (lane >> 2);
        const bool in = row < cur.r.lq * group;
        const T* q = reinterpret_cast<const T*>(p.q) + (in ? (cur.r.q0 + row / group) * p.q_tok +
                                                             (cur.head * group + row % group) * p.q_head : 0);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t* at = reinterpret_cast<const uint32_t*>(q + k * 16 + (lane & 3) * 2);
          qf[t][k][0] = in ? at[0] : 0u;
          qf[t][k][1] = in ? at[4] : 0u;
        }
      }
    }
    copies_wait<kStages - 2>();
    __syncthreads();  // tile n is here, and every warp is done with the stage of tile n - 1
    if (fresh) {
      if constexpr (kQShared) {
        const uint32_t from = smem_of(sm.q[q_now]);
        q_now ^= 1;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int r = t * 8 + (lane & 7);
#pragma unroll
          for (int k = 0; k < D / 16; k += 2) {  // two 16-dimension slices at a time
            uint32_t a[4];
            load_matrix(a, from + r * (D * 2) + (((k * 2 + (lane >> 3)) ^ (r & 7)) << 4));
            qf[t][k][0] = a[0];
            qf[t][k][1] = a[1];
            qf[t][k + 1][0] = a[2];
            qf[t][k + 1][1] = a[3];
          }
        }
        // The block is read before the copies of the pair two behind this one, which may
        // begin in this iteration.
        __syncthreads();
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 8 + (lane & 3) * 2 + i;
          seen[t][i] = r < cur.r.lq * group ? visible_keys(p, cur.r, r / group) : 0;
          top[t][i] = kLowest;
          sum[t][i] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][k][i] = 0.f;
      }
      fresh = false;
    }
    if (n + kStages - 1 < count) copy_tile(n + kStages - 1);
    copies_commit();
    const bool more = n + kStages < count;
    PairRows pair{};
    if (more) {
      look_up(k_next[0], v_next[0]);
      pair = pair_of(n + kStages);
    }

    // ---- S^T of the warp's 16 keys ----
    const uint32_t ks = smem_of(sm.stage[n % kStages]) + warp * 16 * D * 2, vs = ks + kTile * D * 2;
    // (With one block of columns, two accumulators: a chain of D / 16 products waits for each.)
    constexpr int kChains = NT == 1 ? 2 : 1;
    float s[NT][4], other[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
    {
      const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t a[4];
        load_matrix(a, ks + r * (D * 2) + (((k * 2 + (lane >> 4)) ^ (r & 7)) << 4));
#pragma unroll
        for (int t = 0; t < NT; ++t) Half<T>::mma(k % kChains ? other : s[t], a, qf[t][k][0], qf[t][k][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][i] += other[i];
    }
    // ---- softmax of the columns (query rows) over the warp's keys ----
    const int key = cur.tile * kTile + warp * 16 + (lane >> 2);
    uint32_t pf[NT][2];
    constexpr float kBelow = __is_same(T, __half) ? kF16WeightLog2 : 0.f;  // of `top` below the maximum
    bool grow = false;
    float mx[NT][2];  // over the thread's own keys: the lanes only meet when a maximum grows
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + (i >> 1) * 8 >= seen[t][i & 1]) s[t][i] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[t][i] = fmaxf(s[t][i], s[t][i + 2]) * scale2;
        grow |= mx[t][i] > top[t][i] + (8.f + kBelow);
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = fmaxf(top[t][i], mx[t][i] - kBelow);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          f[i] = exp2_mufu(top[t][i] - m);
          top[t][i] = m;
          sum[t][i] *= f[i];
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][k][i] *= f[i & 1];
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = exp2_mufu(fmaf(s[t][i], scale2, -top[t][i & 1]));
        sum[t][i & 1] += e[i];
      }
      // S^T has keys in rows; as the second product's B operand P^T wants them along k.
      pf[t][0] = transpose8x8(Half<T>::pack(e[0], e[1]));
      pf[t][1] = transpose8x8(Half<T>::pack(e[2], e[3]));
    }
    // ---- O^T += V^T P^T ----
    // (Where some of the query rows may not see all of the warp's keys, a product of a hidden key's zero
    // and an infinity or a NaN would reach them: such values are added by hand.)
    if (cur.r.lq > 1 && p.causal && cur.tile * kTile + warp * 16 + 16 > cur.r.lk - cur.r.lq + 1)
      take_special<T, D, NT>(vs, cur.tile * kTile + warp * 16, seen, o);
    {
      const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t a[4];
        load_matrix_t(a, vs + r * (D * 2) + (((k * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
#pragma unroll
        for (int t = 0; t < NT; ++t) Half<T>::mma(o[t][k], a, pf[t][0], pf[t][1]);
      }
    }
    if (more) {
      // (Tile n's offsets were used in an earlier iteration.)
      publish(n + kStages, k_next[0], v_next[0], pair);
      ahead.next(p);
    }

    // ---- the pair ends, or the run does ----
    if (cur.tile + 1 == cur.tiles || n + 1 == count) {
      const long long first_tile = begin + n - cur.tile;  // of the pair, in the list
      const long long first = ((first_tile + 1) * ctas - 1) / total;
      const long long last = ((first_tile + cur.tiles) * ctas - 1) / total;
      const int parts = (int)(last - first + 1);
      const int rows = cur.r.lq * group;
      float* slots = reinterpret_cast<float*>(p.work + kWorkFront);
      const uint64_t slot_floats = token_slot_floats(kRows, D);
      T* const out = reinterpret_cast<T*>(p.o) + cur.r.q0 * p.o_tok + cur.head * group * p.o_head;
      const auto place = [&](int row) { return out + (row / group) * p.o_tok + (row % group) * p.o_head; };
      // The tile's stage is free until the next iteration's copies.
      float(*joined)[8][D + 4] = reinterpret_cast<float(*)[8][D + 4]>(sm.stage[n % kStages]);
      static_assert(sizeof(float) * kWarps * 8 * (D + 4) <= stage_bytes<D>(), "joined results fit a stage");
      __syncthreads();
      float* mine_at = slots + (blockIdx.x == first ? 2 * first + 1 : 2 * (long long)blockIdx.x) * slot_floats;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t * 8 >= rows) break;
        // The warps' results of eight query rows, joined through shared memory.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = sum[t][i];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          const int r = (lane & 3) * 2 + i;
          if (lane < 4) {
            sm.top[warp][r] = top[t][i];
            sm.sum[warp][r] = x;
          }
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            joined[warp][r][k * 16 + (lane >> 2)] = o[t][k][i];
            joined[warp][r][k * 16 + 8 + (lane >> 2)] = o[t][k][i + 2];
          }
        }
        __syncthreads();
        const int limit = min(8, rows - t * 8);
        for (int x = tid; x < limit * (D / 4); x += kThreads) {
          const int r = x / (D / 4), d = x % (D / 4) * 4;
          float m = kLowest;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm.top[w][r]);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float l = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = exp2_mufu(sm.top[w][r] - m);
            add_scaled(acc, *reinterpret_cast<const float4*>(&joined[w][r][d]), f);
            l = fmaf(f, sm.sum[w][r], l);
          }
          const int row = t * 8 + r;
          if (parts == 1) {
            store_row4<T>(place(row) + d, acc, l);
          } else {
            float* at = mine_at + row * D + d;
            __stcg(reinterpret_cast<float4*>(at), acc);
            if (d == 0) __stcg(reinterpret_cast<float2*>(mine_at + kRows * D) + row, make_float2(m, l));
          }
        }
        __syncthreads();
      }
      if (parts > 1) {
        int* counter = reinterpret_cast<int*>(p.work) + first;
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const int done = atomicAdd(counter, 1);
          if (done == parts - 1) *counter = 0;  // as the next launch finds it
          sm.last = done == parts - 1;
        }
        __syncthreads();
        if (sm.last) {
          __threadfence();
          for (int x = tid; x < rows * (D / 4); x += kThreads) {
            const int row = x / (D / 4), d = x % (D / 4) * 4;
            float m = kLowest, l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            // (Four parts' loads are in flight at a time.)
#pragma unroll 4
            for (int i = 0; i < parts; ++i) {
              const float* at = slots + (i == 0 ? 2 * first + 1 : 2 * (first + i)) * slot_floats;
              const float2 st = __ldcg(reinterpret_cast<const float2*>(at + kRows * D) + row);
              const float4 v = __ldcg(reinterpret_cast<const float4*>(at + row * D + d));
              const float big = fmaxf(m, st.x);
              const float f = exp2_mufu(m - big), g = exp2_mufu(st.x - big);
              acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
              add_scaled(acc, v, g);
              l = fmaf(l, f, st.y * g);
              m = big;
            }
            store_row4<T>(place(row) + d, acc, l);
          }
        }
      }
      fresh = true;
    }
    cur.next(p);
  }
}

}  // namespace

#define TB_TOKEN_ENTRY(name, T, D, NT)                                                       \
  extern "C" __global__ void __launch_bounds__(kThreads, tb::token_per_sm(8 * NT))           \
      name(const __grid_constant__ tb::AttnParams p) {                                       \
    static_assert(sizeof(Shared<D, 8 * NT>) + 128 <= tb::token_smem_bytes(D, 8 * NT),        \
                  "shared memory reservation");                                              \
    attention_tokens<T, D, NT>(p);                                                           \
  }

TB_TOKEN_ENTRY(attention_tokens_bf16_d128_r8, __nv_bfloat16, 128, 1)
TB_TOKEN_ENTRY(attention_tokens_bf16_d128_r16, __nv_bfloat16, 128, 2)
TB_TOKEN_ENTRY(attention_tokens_bf16_d128_r32, __nv_bfloat16, 128, 4)
TB_TOKEN_ENTRY(attention_tokens_f16_d128_r8, __half, 128, 1)
TB_TOKEN_ENTRY(attention_tokens_f16_d128_r16, __half, 128, 2)
TB_TOKEN_ENTRY(attention_tokens_f16_d128_r32, __half, 128, 4)
TB_TOKEN_ENTRY(attention_tokens_bf16_d64_r8, __nv_bfloat16, 64, 1)
TB_TOKEN_ENTRY(attention_tokens_bf16_d64_r16, __nv_bfloat16, 64, 2)
TB_TOKEN_ENTRY(attention_tokens_bf16_d64_r32, __nv_bfloat16, 64, 4)
TB_TOKEN_ENTRY(attention_tokens_f16_d64_r8, __half, 64, 1)
TB_TOKEN_ENTRY(attention_tokens_f16_d64_r16, __half, 64, 2)
TB_TOKEN_ENTRY(attention_tokens_f16_d64_r32, __half, 64, 4)
