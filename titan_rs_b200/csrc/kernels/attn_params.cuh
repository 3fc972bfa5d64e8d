// What the packed and paged attention kernels are told about one call: pointers, extents
// and strides (in elements). Filled by the host entry (op_attention.cpp), passed by value.
//
// A request b owns query rows cu_q[b] .. cu_q[b+1] of `q` and `o`, and Lk keys:
//   packed (table == 0): rows cu_k[b] .. cu_k[b+1] of `k` and `v`;
//   paged: key j is row j % page of page table[b, j / page], Lk = lens[b].
// The index tensors live on the device and are not known to the host, so every kernel
// clamps what it reads from them to the extents given here (request_of below).
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TB_BOTH __host__ __device__
#else
#define TB_BOTH
#endif

namespace tb {

struct AttnParams {
  uint64_t q, k, v, o;     // 16-bit elements
  uint64_t cu_q, cu_k;     // int32 [batch + 1]; cu_k unused when paged
  uint64_t table, lens;    // int32 [batch, width], [batch]; 0 when packed
  int64_t q_tok, q_head;   // strides; the innermost dimension is contiguous everywhere
  int64_t k_tok, k_head, k_page;
  int64_t v_tok, v_head, v_page;
  int64_t o_tok, o_head;
  int64_t table_row;
  int32_t tq, tk;          // rows of q; rows of k (packed)
  int32_t batch, heads, kv_heads, dim;
  int32_t page, pages, width;
  int32_t causal;
  int32_t token_rows;      // requests of at most this many (query row, head) pairs per key head
                           // belong to the token kernel, the others to the kernel beside it
  float scale;             // factor of q . k
  uint64_t work;           // workspace of the token and tile kernels
  int32_t tile_tokens;     // query rows of a 128-row tile, 128 / (heads / kv_heads)
  int32_t max_items;       // (pair of tiles, key head) items of sound index tensors at most
  int32_t cut;             // whether the tile kernel may cut an item's keys into parts (the
                           // workspace then has two slots for each CTA)
};

// The front of every workspace holds counters, at the same place for every kernel and form. Zero
// between launches are one per CTA of the token kernel, and the tile kernel's next work number
// and its count of finished CTAs: nothing keeps a kernel from bringing them back. The finished
// parts of each of the tile kernel's slots' two tiles stay behind, since a launch that gave up a
// wait may leave any of them at any value. They are held twice: launches that cut items use
// the two banks in turn (kTileTurn says which) and clear the other bank for the next one, so that
// none sees what an earlier one left.
constexpr int kTokenMaxCtas = 1022, kTileNext = 1022, kTileDone = 1023, kTileTurn = 1024, kTileParts = 1056;
constexpr int kTileMaxCtas = 512;
constexpr int kTileBank = 2 * 2 * kTileMaxCtas;
constexpr uint64_t kWorkFront = 4ull * (kTileParts + 2 * kTileBank);
// (Workspace offsets of both kernels are multiples of their widest store, 32 bytes.)
static_assert(kWorkFront % 128 == 0 && kTileParts % 32 == 0 && kTileBank % 4 == 0, "workspace alignment");
TB_BOTH constexpr int tile_bank(int turn) { return kTileParts + turn * kTileBank; }
// The counter of finished parts of a slot's tile x (0 or 1).
TB_BOTH constexpr int tile_parts_at(int turn, int slot, int x) { return tile_bank(turn) + 2 * slot + x; }

// The token kernel's partial results, behind the counters: two a CTA (its first request may
// have begun in an earlier CTA, its last may go on in a later one), each rows x (dim + 2)
// floats: O, then the row's maximum and sum.
TB_BOTH constexpr uint64_t token_slot_floats(int rows, int dim) { return (uint64_t)rows * (dim + 2); }
TB_BOTH constexpr uint64_t token_workspace_bytes(int ctas, int rows, int dim) {
  return kWorkFront + 2ull * ctas * token_slot_floats(rows, dim) * 4;
}

// The token kernel: keys of a tile, and, for eight rows and for more, stages of the ring and CTAs
// of an SM (registers allow three only with eight rows), and its shared memory (the ring, the
// row offsets of each stage, two Q blocks where they fit (16 rows), the joined statistics and
// some words; 128 bytes to align).
constexpr int kTokenTile = 64, kTokenThreads = 128;
TB_BOTH constexpr int token_stages(int rows) { return rows <= 8 ? 2 : 3; }
TB_BOTH constexpr int token_per_sm(int rows) { return rows <= 8 ? 3 : 2; }
TB_BOTH constexpr int token_smem_bytes(int dim, int rows) {
  return token_stages(rows) * (2 * kTokenTile * dim * 2 + kTokenTile * 16) + (rows <= 16 ? 2 * rows * dim * 2 : 0) +
         2 * (kTokenThreads / 32) * 8 * 4 + 256 + 128;
}

// The tile kernel's workspace for the parts of items whose keys are cut, in slots of 256 rows,
// behind the counters at the workspace's front:
//   stats:  float2 {maximum, sum} (slots x 256)
//   rows:   float [dim] (slots x 256)
// A cut is made where a request's key tiles exceed the average work of a CTA, so there are at
// most two slots a CTA.
constexpr int kTileRows = 256;  // two tiles of 128 (query row, head) pairs
TB_BOTH constexpr uint64_t tile_rows_at(int slots) { return kWorkFront + 8ull * kTileRows * slots; }
TB_BOTH constexpr uint64_t tile_workspace_bytes(int slots, int dim) {
  return tile_rows_at(slots) + 4ull * kTileRows * slots * dim;
}
constexpr int kTileMaxParts = 32, kTileMinPart = 4;  // parts of an item; key tiles of a part
constexpr int kTileThreads = 384, kTileLaunchRegs = 168;
constexpr int kTileBarrierBytes = 512, kTileScratchBytes = 512;
// Three Q tiles, two stages of a K and a V tile, barriers and item descriptions.
TB_BOTH constexpr int tile_smem_bytes(int dim) {
  return 7 * 128 * dim * 2 + kTileBarrierBytes + kTileScratchBytes + 1024;
}

// Probabilities are rounded to the values' type for the product with V: 2^(s - m), with a
// reference m that may fall 8 behind the row's maximum. f16 has no more than 2^-24 next to 1, and
// many keys of less would be lost together; so m is the maximum less 7 there. Probabilities and
// their sum are 2^7 times as large (2^15 at most, below f16's 65504), the quotient is the same.
// bf16 has fp32's exponents.
constexpr float kF16WeightLog2 = 7.f;

// The index arithmetic is shared by the kernels and a host test of it.
#ifdef __CUDACC__
// These kernels are launched with programmatic stream serialization (launch_overlapped):
// the next one's blocks are set up while the one before still runs. Every thread calls this
// before its first access to global memory; it returns when the grids before have ended and
// their writes are visible. (To plain loads: what an earlier grid wrote is not read through
// the read-only path, whose data has to be constant for a grid's whole life.)
__device__ __forceinline__ void begin_after_earlier_grids() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
#define TB_INDEX_FN __device__ __forceinline__
TB_INDEX_FN int load_index(const int* p) { return *p; }
#else
#define TB_INDEX_FN inline
TB_INDEX_FN int load_index(const int* p) { return *p; }
#endif

// Rows of one tensor, and keys of one request, at most: sums with a tile's rows stay below 2^31.
constexpr int64_t kMaxRows = 0x7fffff00;

// Request b: its query rows [q0, q0 + lq) and its keys (lk of them, from row k0 when packed).
struct AttnRequest {
  int q0, lq, k0, lk;
};

TB_INDEX_FN int clamp_index(int64_t x, int64_t lo, int64_t hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }

TB_INDEX_FN AttnRequest request_of(const AttnParams& p, int b) {
  const int* cu_q = reinterpret_cast<const int*>(p.cu_q);
  AttnRequest r;
  r.q0 = clamp_index(load_index(cu_q + b), 0, p.tq);
  r.lq = clamp_index(load_index(cu_q + b + 1), r.q0, p.tq) - r.q0;
  if (p.table) {
    const int64_t most = (int64_t)p.width * p.page;
    r.k0 = 0;
    r.lk = clamp_index(load_index(reinterpret_cast<const int*>(p.lens) + b), 0, most < kMaxRows ? most : kMaxRows);
  } else {
    const int* cu_k = reinterpret_cast<const int*>(p.cu_k);
    r.k0 = clamp_index(load_index(cu_k + b), 0, p.tk);
    r.lk = clamp_index(load_index(cu_k + b + 1), r.k0, p.tk) - r.k0;
  }
  return r;
}

// Clears the counters that the next launch counts finished parts in: thread `id` of `threads`
// over the whole grid takes every `threads`-th four of them.
TB_INDEX_FN void clear_next_bank(int* counters, int turn, int id, int threads) {
  for (int i = id; i < kTileBank / 4; i += threads)
    for (int k = 0; k < 4; ++k) counters[tile_bank(turn ^ 1) + 4 * i + k] = 0;
}

// Whether the request is the token kernel's (it has query rows, and few enough).
TB_INDEX_FN bool is_token_request(const AttnParams& p, const AttnRequest& r) {
  return r.lq > 0 && (int64_t)r.lq * (p.heads / p.kv_heads) <= p.token_rows;
}

// Leading keys that query row i of the request sees. The causal mask is aligned at the
// ends: the last query row sees every key.
TB_INDEX_FN int visible_keys(const AttnParams& p, const AttnRequest& r, int i) {
  return p.causal ? clamp_index((int64_t)r.lk - r.lq + i + 1, 0, r.lk) : r.lk;
}

// Page `index` of request b, or -1 when the table names none of the cache's pages (its keys
// read as zeros).
TB_INDEX_FN int page_of(const AttnParams& p, int b, int index) {
  const int id = load_index(reinterpret_cast<const int*>(p.table) + b * p.table_row + index);
  return id >= 0 && id < p.pages ? id : -1;
}

#ifdef __CUDACC__

// A thread's stretch of the requests, and the units (tiles of work) before and in it: every
// thread of the block adds up units(b) over its stretch and a scan joins the sums. `scan`
// holds one word a warp. Ends with a barrier.
struct Stretch {
  int lo, hi;
  long long before, total;
};

template <int kThreads, typename Units>
__device__ __forceinline__ Stretch count_units(int batch, long long* scan, Units units) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Stretch s;
  const int per = (batch + kThreads - 1) / kThreads;
  s.lo = min((int)threadIdx.x * per, batch);
  s.hi = min(s.lo + per, batch);
  long long mine = 0;
  for (int b = s.lo; b < s.hi; ++b) mine += units(b);
  long long upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += x;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  s.before = upto - mine;
  s.total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) s.before += scan[w];
    s.total += scan[w];
  }
  return s;
}

// The thread whose stretch holds unit `target` writes its request and the units before that
// request. Ends with a barrier; `target` lies below the total.
template <typename Units>
__device__ __forceinline__ void find_unit(const Stretch& s, long long target, Units units, int* found,
                                          long long* found_before) {
  long long at = s.before;
  for (int b = s.lo; b < s.hi && at <= target; ++b) {
    const long long n = units(b);
    if (target < at + n) {
      *found = b;
      *found_before = at;
    }
    at += n;
  }
  __syncthreads();
}

#endif

}  // namespace tb
