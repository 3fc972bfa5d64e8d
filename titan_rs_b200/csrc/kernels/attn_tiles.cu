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
//                packed key tile is one box; a paged one is 128 / page boxes, whose page ids
//                the lanes look up two tiles ahead. A page id that names no page, and
//                pages past the request's end, are given a coordinate outside the map, which
//                the copy fills with zeros.
//   warp 1       owns the tensor memory S_A | S_B | O_A | O_B; one lane issues the MMAs.
//   warp 2       keeps what a row may not see out of P V, between a V tile's copy and its use: the
//                probabilities are 0 there, but 0 x NaN is not. It clears the rows of the last tile
//                that lie past the request's end (another request's, or whatever an unfinished page
//                holds) or that none of the item's rows sees, and looks through those that only some see
//                for infinities and NaNs. It clears these too, and the softmax warps add them to the
//                rows that do see their keys when the item ends (sixteen ragged prompts 121.4 us
//                without this, 122.2 with it; eight long ones 911 and 912; four short sequences 11.7
//                and 12.0). Scores of hidden keys are replaced before use.
//   warps 4..11  softmax, one row a thread, warps 4-7 tile A, 8-11 tile B.
//   warp 3       items: persistent CTAs draw them from a counter. Requests with more key tiles than
//                a CTA's share of the whole call are cut along the keys into parts, drawn first;
//                then come requests with more than half of a share, a quarter, and the rest,
//                so that no long item starts when the others are done. The warpgroup that
//                finishes a tile's last part adds the parts up, in their order.
// Bound by the chain of a tile's softmax and products: a step of the steady state takes about
// 3,300 cycles, of which the tensor core works 2,176 and a tile's exponentials 2,048; an item
// adds some 4,000 in which its rows are stored. With the caches emptied in between, eight prompts
// of 2900 to 4096 tokens, 32 heads (837 GFLOP under the mask) take 895 to 908 us over the boards
// seen, 0.92 to 0.94 PFLOP/s; eight of 4096 (1.1 TFLOP) 1,121 us with 32 key heads and 1,074
// with 8, 0.98 and 1.02 PFLOP/s.
// Items of one to four steps are bound by the instruction caches, which the roles' code shares
// and leaves behind: with the items' arithmetic in 32 bits and the mask, the copies of K and V,
// the halves of P V and the rows' stores in loops, sixteen ragged prompts went from 125 to 114 us,
// 24 of dimension 64 over other sequences' keys from 64 to 54, 128 of 256 tokens from 216
// to 190 (launches in a row on one board; with the caches emptied in between, over several, the
// kept form takes 119 to 122, 54.5 to 55 and 223). A thread spills up to 20 bytes. Built and not
// kept: two threads a row (sixteen softmax warps, 1,110 us where one
// took 992: agreeing on the row's maximum costs more than the halves save), S read from tensor
// memory a second time for the exponentials (less code, but 4 to 9% slower from four steps on),
// items drawn earlier where they are short (up to 8% slower: the last ones are spread less
// evenly), K and V asked into L2 a tile ahead (8% slower: the copy engine takes each request
// in turn), the same for the next item's first tiles (7%).
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
constexpr uint32_t kFailSchedule = 0x56050000u;
constexpr uint32_t kControlRegs = 88, kSoftmaxRegs = 208;
static_assert(128 * kControlRegs + 256 * kSoftmaxRegs <= kTileThreads * kTileLaunchRegs,
              "the warpgroups' registers exceed the launch allocation");

constexpr int kSlots = 4;         // item descriptions in flight
constexpr int kItemReaders = 11;  // warps 0, 1, 2 and the eight softmax warps
constexpr int kQ = 3;             // Q tiles in shared memory
constexpr long long kGroupBytes = 32ll << 20;  // K and V worked on at a time (909 us for long prompts; 921 without)

struct Barriers {
  uint64_t q_full[kQ], q_empty[kQ];
  uint64_t kv_full[2], kv_empty[2];  // the stage of step t holds K of its key tile and V of the one before
  uint64_t s_full[2];                // per query tile (A, B)
  uint64_t p_half[2];                // per query tile: P of keys [0, 64) is in TMEM
  uint64_t p_full[2];                // per query tile: P of keys [64, 128) is in TMEM
  uint64_t o_full[2];                // per query tile: an item's last product is done
  uint64_t v_raw[2];                 // per stage: a V tile that warp 2 looks at first
  uint64_t drain;
  uint64_t item_full[kSlots], item_empty[kSlots];
  uint64_t part_stored[2], part_known[2];  // per query tile: a part is in the workspace; whether it was the last one
  uint64_t item_want;                // the producer nears its item's end: draw the next one
  uint32_t tmem_base;
};
static_assert(sizeof(Barriers) <= kTileBarrierBytes, "barrier block overflows its reservation");

// One item: two query tiles of one request and key head, and a range of key tiles.
struct alignas(16) Item {
  int n, n_a, n_b;       // key tiles of the part, and how many of them tiles A and B need; n < 0: no more items
  int lo;                // the first key tile
  int hk, b;             // key head, request
  int row, valid;        // tile A's first row of q, and rows from there to the request's end
  int base;              // local row i sees base + i keys (causal)
  int lk, k0;            // keys of the request, and its first row of k (packed)
  int cut_from;          // the part's first key tile with keys that some row may not see (n: none)
  short last_rows;       // rows of the last key tile if it runs past the request's end, else 0
  bool special[2];       // whether one of the tiles from cut_from on that query tile x needs held an infinity or a
                         // NaN (warp 2 says so before the tile's product, so it is settled when that ends)
  short parts, part;     // parts that the item's keys are cut into, and which this is
  int slot, stride;      // slot of part 0, and the slots from one part to the next
};

constexpr int kClasses = 4;  // of requests, by their number of key tiles: cut, long, middling, short

struct Scratch {
  Item items[kSlots];
  long long sums[kTileThreads / 32];
  unsigned long long works[kClasses];
  int last[2];  // whether a warpgroup finished its tile's last part
};
static_assert(sizeof(Scratch) <= kTileScratchBytes, "scratch block overflows its reservation");

// True in one lane of the warp (the same one each time), all of which call it. The compiler
// knows of an elected lane that it is one: under `lane == 0` every tcgen05.mma was wrapped in
// a loop over the lanes that might be there (eight prompts of 4096 tokens, 32 heads: 1194 us
// against 1028).
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

// Adds to the bytes the current phase waits for, without arriving.
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
               : "memory");
}

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
  if (p.token_rows && is_token_request(p, r)) return 0;
  return (int)((unsigned)(r.lq + 2 * p.tile_tokens - 1) / (unsigned)(2 * p.tile_tokens));
}

__device__ __forceinline__ int key_tiles(const AttnRequest& r) { return (r.lk + BN - 1) / BN; }

// The class of a request: 0 is cut into parts, 1 to 3 are long, middling and short next to
// a CTA's share. A cut costs a CTA about six key tiles' time (the parts' rows go through
// memory), so it has to save more.
__device__ __forceinline__ int class_of(const AttnParams& p, const AttnRequest& r, int share) {
  const int n = key_tiles(r);
  if (p.cut && n > share + share / 8 + 6) return 0;
  return 2 * n > share ? 1 : 4 * n > share ? 2 : 3;
}

__device__ __forceinline__ int parts_of(const AttnRequest& r, int share) {
  return min(kTileMaxParts, (int)((unsigned)(key_tiles(r) + share - 1) / (unsigned)share));
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

// 32 bytes of a row, in one store where the rows are aligned to it. (A lane stores its own
// row. Turning the rows of four lanes by shuffles, so that a store covers whole lines, cost
// more issue slots than it saved: 261 against 243 us for 128 requests of 256 tokens, 32 heads.)
__device__ __forceinline__ void store32(void* to, const uint32_t* r, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(r[0], r[1], r[2], r[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
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
// at or below 2^8 (in f16 2^15, see kF16WeightLog2). It starts at the lowest finite value, so a
// row (or a tile of it) without a visible key adds exp2(-inf) = 0.
template <typename T, int HD>
__device__ __forceinline__ void softmax_step(uint32_t s_tmem, uint32_t o_tmem, int valid, bool rescale, float scale2,
                                             float& m, float& l, uint64_t* p_half, uint64_t* p_full) {
  const int lane = lane_id();
  // Few tiles have keys to mask: they go through a loop of their own over S in tensor memory.
  // (Its code four times over in everyone's way took 130 us where this takes 120; sixteen prompts.)
  if (__any_sync(0xffffffffu, valid < BN)) {
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      if (__all_sync(0xffffffffu, valid >= c + 32)) continue;
      uint32_t s[32];
      tmem_ld_x32(s_tmem + c, s);
      tmem_ld_wait();
      reg_fence(s);
      sdpa2::mask_chunk(s, valid - c);
      tmem_st_x16(s_tmem + c, reinterpret_cast<uint32_t(&)[16]>(s[0]));
      tmem_st_x16(s_tmem + c + 16, reinterpret_cast<uint32_t(&)[16]>(s[16]));
    }
    tmem_st_wait();
  }
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
  mask_max_chunk(c0, BN, false, mx4);
  mask_max_chunk(c1, BN, false, mx4);
  mask_max_chunk(c2, BN, false, mx4);
  mask_max_chunk(c3, BN, false, mx4);
  const float mx = fmaxf(fmax3f(mx4[0], mx4[1], mx4[2]), mx4[3]) * scale2;
  constexpr float kBelow = __is_same(T, __half) ? kF16WeightLog2 : 0.f;  // of m below the maximum
  const bool grow = mx > m + (sdpa2::kLazyRescaleLog2 + kBelow);
  if (__any_sync(0xffffffffu, grow)) {
    const float m_new = grow ? mx - kBelow : m;
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

// Two 16-bit values each times zero, added to `sum`: zeros, or NaN where one is no finite number.
template <typename T>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t x, uint32_t sum) {
  if constexpr (__is_same(T, __half)) {
    const __half2 s = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2(), *reinterpret_cast<const __half2*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&s);
  } else {
    const __nv_bfloat162 s = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __nv_bfloat162(),
                                     *reinterpret_cast<const __nv_bfloat162*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&s);
  }
}

template <typename T>
constexpr uint32_t kExponent = __is_same(T, __half) ? 0x7c00u : 0x7f80u;  // all ones in an infinity or a NaN

// Infinities and NaNs in rows [first, end) of a V tile become zeros. A warp's work.
template <typename T>
__device__ __noinline__ void clear_special(uint8_t* tile, int halves, int first, int end) {
  for (int h = 0; h < halves; ++h) {
    uint32_t* const at = reinterpret_cast<uint32_t*>(tile + h * 128 * 128);
#pragma unroll 1
    for (int i = first * 32 + lane_id(); i < end * 32; i += 32) {
      uint32_t x = at[i];
      if ((x & kExponent<T>) == kExponent<T>) x &= 0xffff0000u;
      if ((x >> 16 & kExponent<T>) == kExponent<T>) x &= 0xffffu;
      at[i] = x;
    }
  }
}

// Whether rows [first, end) of a V tile hold an infinity or a NaN. A warp's work, one load and four
// instructions for 8 values, while the tile's softmax runs. (Four loads at a time: with one the
// products wait for it, 948 us for long prompts where all rows are looked at, and 910 with four; with
// eight the code costs the other roles more instruction fetches.)
template <typename T, int kHalves>
__device__ __forceinline__ bool has_special(const uint8_t* tile, int first, int end) {
  uint32_t sum[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int h = 0; h < kHalves; ++h) {
    const uint4* const at = reinterpret_cast<const uint4*>(tile + h * 128 * 128);
#pragma unroll 4
    for (int i = first * 8 + lane_id(); i < end * 8; i += 32) {
      const uint4 x = at[i];
      sum[0] = add_zero_times<T>(x.x, sum[0]);
      sum[1] = add_zero_times<T>(x.y, sum[1]);
      sum[2] = add_zero_times<T>(x.z, sum[2]);
      sum[3] = add_zero_times<T>(x.w, sum[3]);
    }
  }
  return __any_sync(0xffffffffu, ((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0);
}

// Adds the infinities and NaNs of V's rows [from, to) of the request, which clear_special took out, to
// one row of O (a thread's). Called by all lanes of a warp; it is rare and reads V from memory.
template <typename T, int HD>
__device__ __noinline__ void add_special(const AttnParams& p, const Item& it, uint32_t o_tmem, int from, int to) {
#pragma unroll 1
  for (int c = 0; c < HD; c += 16) {
    uint32_t o[16];
    tmem_ld_x16(o_tmem + c, o);
    tmem_ld_wait();
    reg_fence(o);
#pragma unroll 1
    for (int key = from; key < to; ++key) {
      const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v) + it.hk * p.v_head + c;
      if (p.table) {
        const int id = page_of(p, it.b, key / p.page);
        if (id < 0) continue;
        v += id * p.v_page + key % p.page * p.v_tok;
      } else {
        v += (it.k0 + key) * p.v_tok;
      }
#pragma unroll
      for (int d = 0; d < 16; ++d)
        if ((v[d] & kExponent<T>) == kExponent<T>)
          o[d] = __float_as_uint(__uint_as_float(o[d]) + (float)*reinterpret_cast<const T*>(v + d));
    }
    __syncwarp();
    tmem_st_x16(o_tmem + c, o);
  }
  tmem_st_wait();
}

// A wait that sleeps between polls, for the warps beside the pipeline: they share issue slots
// with softmax warps (2% of a long prompt's time with mbar_wait in their place).
__device__ __forceinline__ bool wait_idle(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_addr(bar);
  if (mbar_try_wait(at, parity)) return true;
  const uint64_t start = global_timer_ns();
  for (uint32_t polls = 1; !mbar_try_wait(at, parity); ++polls) {
    __nanosleep(300);
    if (polls % 64 == 0 && global_timer_ns() - start > kWaitLimitNs) return false;
  }
  return true;
}

// A warp's place in the list of items: it reads each description and lets go of its slot.
struct Reader {
  int slot = 0;
  uint32_t phase = 0;

  // The next item's description, held until done(); null when the wait ran out. All lanes.
  __device__ __forceinline__ const Item* hold(Barriers* bars, const Scratch* scratch) {
    if (!__all_sync(0xffffffffu, mbar_wait(&bars->item_full[slot], phase))) return nullptr;
    return &scratch->items[slot];
  }
  __device__ __forceinline__ void done(Barriers* bars) {
    __syncwarp();
    if (lane_id() == 0) mbar_arrive(&bars->item_empty[slot]);
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }

  // Called by all lanes of the warp, or (kLanes = 1) by one; false when the wait ran out.
  template <int kLanes = 32, bool kIdle = false>
  __device__ __forceinline__ bool next(Barriers* bars, const Scratch* scratch, Item& item) {
    bool ok = kIdle ? wait_idle(&bars->item_full[slot], phase) : mbar_wait(&bars->item_full[slot], phase);
    if (kLanes > 1) ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      item = scratch->items[slot];
      if (kLanes > 1) __syncwarp();
      if (kLanes == 1 || lane_id() == 0) mbar_arrive(&bars->item_empty[slot]);
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
    return ok;
  }
};

// The parts of four rows' columns, added up in their order by one thread (rows at, at + step, ..;
// neighbouring lanes take neighbouring columns): M = max m_i, O = sum 2^(m_i - M) O_i /
// sum 2^(m_i - M) l_i. `store(row, four values)` takes what is done.
template <int HD, typename Store>
__device__ __forceinline__ void join_parts(const float2* stats, const float* rows, int slot0, int stride, int parts,
                                           int at, int step, int end, int column, Store store) {
  constexpr int kRowsAtOnce = 4;
  const auto slot_of = [&](int i) { return (long long)(slot0 + i * stride) * kTileRows; };
  float m[kRowsAtOnce], l[kRowsAtOnce];
  float4 acc[kRowsAtOnce];
#pragma unroll
  for (int k = 0; k < kRowsAtOnce; ++k) {
    m[k] = kLowest;
    l[k] = 0.f;
    acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 2
  for (int i = 0; i < parts; ++i) {
#pragma unroll
    for (int k = 0; k < kRowsAtOnce; ++k) {
      const int row = min(at + k * step, end - 1);
      const float2 st = __ldcg(stats + slot_of(i) + row);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(rows + (slot_of(i) + row) * HD + column));
      const float big = fmaxf(m[k], st.x);
      const float f = exp2_mufu(m[k] - big), g = exp2_mufu(st.x - big);
      m[k] = big;
      l[k] = fmaf(l[k], f, st.y * g);
      acc[k].x = fmaf(acc[k].x, f, o.x * g);
      acc[k].y = fmaf(acc[k].y, f, o.y * g);
      acc[k].z = fmaf(acc[k].z, f, o.z * g);
      acc[k].w = fmaf(acc[k].w, f, o.w * g);
    }
  }
#pragma unroll
  for (int k = 0; k < kRowsAtOnce; ++k) {
    const float inv = l[k] == 0.f ? 0.f : 1.0f / l[k];
    if (at + k * step < end)
      store(at + k * step, make_float4(acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv));
  }
}

template <typename T, int HD>
__device__ __forceinline__ void attention_tiles(const AttnParams& p, const CUtensorMap& tmap_q,
                                                const CUtensorMap& tmap_k, const CUtensorMap& tmap_v,
                                                uint32_t* status) {
  using S = Shape<T, HD>;
  constexpr int OFF_Q = 0, OFF_K = OFF_Q + kQ * S::kTileBytes, OFF_V = OFF_K + 2 * S::kTileBytes,
                OFF_BAR = OFF_V + 2 * S::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + OFF_BAR);
  Scratch* scratch = reinterpret_cast<Scratch*>(smem + OFF_BAR + kTileBarrierBytes);
  const int warp = warp_id(), lane = lane_id();
  const int group = p.heads / p.kv_heads;
  int* const counters = reinterpret_cast<int*>(p.work);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kQ; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_half[i], 4);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->o_full[i], 1);
      mbar_init(&bars->v_raw[i], 1);
      mbar_init(&bars->part_stored[i], 4);
      mbar_init(&bars->part_known[i], 1);
    }
    mbar_init(&bars->drain, 1);
    mbar_init(&bars->item_want, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars->item_full[i], 1);
      mbar_init(&bars->item_empty[i], kItemReaders);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  begin_after_earlier_grids();
  const int turn = p.cut ? counters[kTileTurn] : 0;
  // ---- a CTA's share of the call, in key tiles, and the works (parts of items) of each class ----
  if (threadIdx.x < kClasses) scratch->works[threadIdx.x] = 0;
  long long mine = 0;
  for (int b = threadIdx.x; b < p.batch; b += kTileThreads) {
    const AttnRequest r = request_of(p, b);
    mine += (long long)pairs_of(p, r) * key_tiles(r);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
  if (lane == 0) scratch->sums[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kTileThreads / 32; ++w) total += scratch->sums[w];
  // (Four times a request's key tiles stay below 2^27.)
  const int share =
      (int)min(1ll << 27, max((long long)kTileMinPart, (total * p.kv_heads + gridDim.x - 1) / gridDim.x));
  for (int b = threadIdx.x; b < p.batch; b += kTileThreads) {
    const AttnRequest r = request_of(p, b);
    const int c = class_of(p, r, share);
    const int n = pairs_of(p, r) * (c == 0 ? parts_of(r, share) : 1);
    if (n) atomicAdd(&scratch->works[c], (unsigned long long)n);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;

  if (warp < 4) {
    setmaxnreg_dec<kControlRegs>();
    if (warp == 3) {
      // ---------------- items: the longest rows first, drawn from a counter ----------------
      int w = blockIdx.x, class_end = 0, before = 0;  // works up to the class's end; units before request b
      int c = -1, b = 0;                                     // the walk stands in class c before request b
      // (More than max_items only where cu_seqlens counts rows twice; the rest is then left.)
      long long works = 0;
      for (int i = 0; i < kClasses; ++i) works += (long long)scratch->works[i] * p.kv_heads;
      const int most = works > 0x7fffffff ? 0 : p.max_items + 2 * (int)gridDim.x;
      for (int k = 0;; ++k) {
        const int slot = k % kSlots;
        // An item is drawn only when its predecessor nears its end, so no CTA sits on work that
        // another could begin.
        if (!__all_sync(0xffffffffu, (k == 0 || wait_idle(&bars->item_want, (k - 1) & 1)) &&
                                         wait_idle(&bars->item_empty[slot], ((k / kSlots) & 1) ^ 1))) {
          if (lane == 0) report_status(status, kFailSchedule | 1);
          break;
        }
        if (k > 0) {
          if (lane == 0) w = (int)gridDim.x + atomicAdd(counters + kTileNext, 1);
          w = __shfl_sync(0xffffffffu, w, 0);
        }
        while (c + 1 < kClasses && w >= class_end) {
          class_end += (int)scratch->works[++c] * p.kv_heads;
          b = p.batch;
          before = (int)scratch->works[c];
        }
        const bool more = w < class_end && w < most;
        Item it{};
        it.n = -1;
        if (more) {
          // Units of the class, a pair of tiles or a part of one: the last request's come first.
          const auto units = [&](int at) {
            const AttnRequest r = request_of(p, at);
            return class_of(p, r, share) == c ? pairs_of(p, r) * (c == 0 ? parts_of(r, share) : 1) : 0;
          };
          const int place = class_end - 1 - w, unit = (int)((unsigned)place / (unsigned)p.kv_heads);
          // Back over the requests, 32 at a time, to the one that holds `unit`.
          while (unit < before) {
            const int mine = b - 1 - lane;
            const int own = mine >= 0 ? units(mine) : 0;
            int upto = own;
#pragma unroll 1
            for (int off = 1; off < 32; off <<= 1) {
              const int x = __shfl_up_sync(0xffffffffu, upto, off);
              if (lane >= off) upto += x;
            }
            const uint32_t reached = __ballot_sync(0xffffffffu, before - upto <= unit);
            const int at = reached ? __ffs(reached) - 1 : 31;
            before -= __shfl_sync(0xffffffffu, upto, at);
            b -= at + 1;
          }
          const AttnRequest r = request_of(p, b);
          // Inside a request: groups of key heads whose K and V stay in L2 while the group
          // runs, and in a group the last pairs (with the most keys) of all its heads first.
          const int pairs = pairs_of(p, r), parts = c == 0 ? parts_of(r, share) : 1;
          const int turn = (before + pairs * parts) * p.kv_heads - 1 - place;
          const int heads_at_once =
              min(p.kv_heads, max(1, (int)((unsigned)(kGroupBytes / (4 * HD)) / (unsigned)max(r.lk, 1))));
          const int in_group = heads_at_once * pairs * parts;
          const int groups_before = (int)((unsigned)turn / (unsigned)in_group);
          const int first_head = groups_before * heads_at_once;
          const int rest = turn - groups_before * in_group, heads = min(heads_at_once, p.kv_heads - first_head);
          const int pair = (int)((unsigned)rest / (unsigned)(heads * parts)), at = rest - pair * heads * parts;
          const int tok0 = (pairs - 1 - pair) * 2 * p.tile_tokens;
          const int part = (int)((unsigned)at / (unsigned)heads);
          const bool has_b = tok0 + p.tile_tokens < r.lq;
          // Key tiles that each tile needs (of its last row), and this part's range of them.
          const int end_a = (visible_keys(p, r, min(tok0 + p.tile_tokens, r.lq) - 1) + BN - 1) / BN;
          const int end_b =
              has_b ? (visible_keys(p, r, min(tok0 + 2 * p.tile_tokens, r.lq) - 1) + BN - 1) / BN : 0;
          const int all = max(end_a, end_b);
          const int lo = (int)((unsigned)(part * all) / (unsigned)parts);
          const int hi = (int)((unsigned)((part + 1) * all) / (unsigned)parts);
          it.n = hi - lo;
          it.n_a = max(0, min(hi, end_a) - lo);
          it.n_b = max(0, min(hi, end_b) - lo);
          it.lo = lo;
          it.hk = first_head + at - part * heads;
          it.b = b;
          it.row = r.q0 + tok0;
          it.valid = r.lq - tok0;
          it.base = p.causal ? r.lk - r.lq + tok0 + 1 : r.lk;
          it.lk = r.lk;
          it.k0 = r.k0;
          it.last_rows = it.n > 0 && hi == r.lk / BN + 1 ? (short)(r.lk % BN) : (short)0;
          // (The item's first row sees the fewest keys, `base` of them.)
          it.cut_from = p.causal && it.base < r.lk ? min(max(max(it.base, 0) / BN - lo, 0), it.n) : it.n;
          it.parts = (short)parts;
          it.part = (short)part;
          it.slot = c == 0 ? w - part * heads : 0;
          it.stride = heads;
        }
        if (lane == 0) {
          scratch->items[slot] = it;
          mbar_arrive(&bars->item_full[slot]);
        }
        if (!more) break;
      }
      // The counters are zero again for the next launch, and its turn is another. (Every CTA has
      // read this launch's turn: it did so before its first item.)
      if (lane == 0 && atomicAdd(counters + kTileDone, 1) == (int)gridDim.x - 1) {
        counters[kTileNext] = 0;
        counters[kTileDone] = 0;
        if (p.cut) counters[kTileTurn] = turn ^ 1;
      }
    } else if (warp == 0) {
      // ---------------- producer ----------------
      if (lane == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
      }
      // Lane i copies box i of a key tile: rows [i box, (i + 1) box) of it.
      const bool paged = p.table != 0;
      const int box = paged ? min(p.page, BN) : BN, boxes = BN / box;
      const bool active = lane < boxes;
      // The coordinates of the lane's box of key tile j: (row, page).
      const auto row_of = [&](const Item& it, int j) {
        return paged ? (p.page > BN ? j * BN % p.page : 0) : it.k0 + j * BN;
      };
      const auto page_at = [&](const Item& it, int j) {
        if (!paged || !active || j >= it.lo + it.n) return 0;
        const int index = p.page > BN ? (int)((long long)j * BN / p.page) : j * boxes + lane;
        const int id = (long long)index * p.page < it.lk ? page_of(p, it.b, index) : -1;
        return id < 0 ? p.pages : id;
      };
      const auto load = [&](int off, const CUtensorMap* map, uint64_t* bar, int hk, int row, int w) {
// (Four boxes under one election: one at a time, 16-token pages took 170 us where these take 123.)
#pragma unroll 1
        for (int i = 0; i < boxes; i += 4) {
          int pages[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) pages[k] = __shfl_sync(0xffffffffu, w, i + k);
          if (elected()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (i + k >= boxes) break;
#pragma unroll
              for (int h = 0; h < S::kHalves; ++h)
                tma_load_4d(smem + off + h * S::kHalfBytes + (i + k) * box * 128, map, bar, 64 * h, hk, row, pages[k]);
            }
          }
        }
      };
      int q_slot = 0;
      uint32_t q_phase = 1;  // of q_empty: the first round finds the slots free
      uint32_t q_issued[kQ] = {0, 0, 0}, kv_issued[2] = {0, 0};
      // Query tile x of the item into the next Q slot.
      const auto load_q = [&](const Item& it, int x) {
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->q_empty[q_slot], q_phase))) return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->q_full[q_slot], S::kHalves * p.tile_tokens * group * 128);
          for (int h = 0; h < S::kHalves; ++h)
            tma_load_3d(smem + OFF_Q + q_slot * S::kTileBytes + h * S::kHalfBytes, &tmap_q, &bars->q_full[q_slot],
                        64 * h, it.hk * group, it.row + x * p.tile_tokens);
        }
#pragma unroll
        for (int i = 0; i < kQ; ++i) q_issued[i] += i == q_slot;
        if (++q_slot == kQ) {
          q_slot = 0;
          q_phase ^= 1;
        }
        return true;
      };
      Reader reader;
      Item cur{}, nxt{};
      int j = 0, w_now = 0, w_next = 0, n_w0 = 0, n_w1 = 0;  // pages of the lane's boxes, two key tiles ahead
      bool has_v = false;  // a V tile is owed: the one of the last step's key tile
      int v_hk = 0, v_row = 0, v_page = 0, v_clear = 0;
      uint32_t step = 0;
      bool ok = true;
      while (ok) {
        const bool has_k = cur.n > 0;
        if (!has_k && !has_v) {
          if (cur.n < 0) break;
          ok = reader.next(bars, scratch, cur);
          if (ok && cur.n == 0 && lane == 0) mbar_arrive(&bars->item_want);
          w_now = page_at(cur, cur.lo);
          w_next = page_at(cur, cur.lo + 1);
          continue;
        }
        int w_after = 0;
        if (has_k) {
          if (lane == 0 && j == max(0, cur.n - 3)) mbar_arrive(&bars->item_want);
          w_after = page_at(cur, cur.lo + j + 2);
          if (j == 0 && cur.n_a > 0) ok = load_q(cur, 0);
          if (j + 1 == cur.n && ok) {
            // The item behind it, and its first pages, while this step's stage is still in use.
            // (One item only: everyone has begun the item before this one, so it is there.)
            ok = reader.next(bars, scratch, nxt);
            if (ok && nxt.n == 0 && lane == 0) mbar_arrive(&bars->item_want);
            n_w0 = page_at(nxt, nxt.lo);
            n_w1 = page_at(nxt, nxt.lo + 1);
          }
        }
        const int st = step & 1;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars->kv_empty[st], ((step >> 1) & 1) ^ 1));
        if (!ok) break;
        // A V tile that warp 2 looks at goes to it first; it arrives on kv_full for the step.
        const bool raw = has_v && v_clear;
        if (lane == 0) {
          const uint32_t k_bytes = has_k ? S::kTileBytes : 0, v_bytes = has_v ? S::kTileBytes : 0;
          if (raw) {
            if (k_bytes) mbar_expect_tx(&bars->kv_full[st], k_bytes);
            mbar_arrive_expect_tx(&bars->v_raw[st], v_bytes);
          } else {
            mbar_arrive_expect_tx(&bars->kv_full[st], k_bytes + v_bytes);
          }
        }
        __syncwarp();
        const int k_row = row_of(cur, cur.lo + j);
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if (!(t ? has_k : has_v)) continue;
          load((t ? OFF_K : OFF_V) + st * S::kTileBytes, t ? &tmap_k : &tmap_v,
               !t && raw ? &bars->v_raw[st] : &bars->kv_full[st], t ? cur.hk : v_hk, t ? k_row : v_row, t ? w_now : v_page);
        }
        ++kv_issued[st];
        ++step;
        has_v = has_k;
        if (!has_k) continue;
        v_hk = cur.hk;
        v_row = row_of(cur, cur.lo + j);
        v_page = w_now;
        v_clear = j >= cur.cut_from || (j + 1 == cur.n && cur.last_rows);
        if (j == 0 && cur.n_b > 0) ok = load_q(cur, 1);
        w_now = w_next;
        w_next = w_after;
        if (++j == cur.n) {
          cur = nxt;
          j = 0;
          w_now = n_w0;
          w_next = n_w1;
        }
      }
      if (!ok) {
        if (lane == 0) report_status(status, kFailProducer | 1);
        for (int i = 0; i < kQ; ++i)
          if (q_issued[i] && !mbar_wait(&bars->q_full[i], (q_issued[i] - 1) & 1))
            report_status(status, kFailProducer | 3);
        for (int i = 0; i < 2; ++i)
          if (kv_issued[i] && !mbar_wait(&bars->kv_full[i], (kv_issued[i] - 1) & 1))
            report_status(status, kFailProducer | 4);
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      // Step t: the products P V of the key tile before, then the scores Q K^T of this one,
      // per query tile. The step that begins an item ends the one before it, unless that has
      // no keys (or there is none): then a step without scores comes between.
      if (elected()) {
        Reader reader;
        Item it{};
        bool ok = true, owed = false;
        int n = 0, n_a = 0, n_b = 0, j = 0;
        int pj = 0, pn_a = 0, pn_b = 0;  // the key tile before: its number in its item, and the tiles that need it
        const uint64_t qd0 = sdesc_sw128(smem_addr(smem + OFF_Q), 16, 1024);
        const uint64_t kd0 = sdesc_sw128(smem_addr(smem + OFF_K), 16, 1024);
        const uint64_t vd0 = sdesc_sw128(smem_addr(smem + OFF_V), S::kHalfBytes, 1024);
        int q_slot = 0, q_ab = 0;                     // the next Q slot; those of tiles A (low byte) and B
        uint32_t q_phase = 0, step = 0, parities = 0;  // bit x: parity of tile x's next scores
        uint32_t failed = 0;
        while (ok) {
          if (n <= 0 && !owed) {
            if (n < 0) break;
            ok = reader.next<1>(bars, scratch, it);
            n = it.n;
            n_a = it.n_a;  // 0 in an item without keys, and behind the last one
            n_b = it.n_b;
            continue;
          }
          const int st = step & 1;
          const uint64_t kd = desc_add(kd0, st * (S::kTileBytes >> 4));
          const uint64_t vd = desc_add(vd0, st * (S::kTileBytes >> 4));
          if (!mbar_wait(&bars->kv_full[st], (step >> 1) & 1)) failed = 2;
          // (Not unrolled, here and below: the roles' code competes for the instruction caches.
          // Two copies of this body, and a third for steps inside an item, took 243 -> 310 us
          // for 128 requests of 256 tokens.)
#pragma unroll 1
          for (int x = 0; x < 2 && !failed; ++x) {
            const int nx = x ? n_b : n_a, pnx = x ? pn_b : pn_a;
            const uint32_t s_tmem = tmem + x * BN, o_tmem = tmem + (2 + x) * BN;
            if (pj < pnx) {
              const uint32_t parity = ((parities >> x) & 1) ^ 1;  // of the scores before
#pragma unroll 1
              for (int half = 0; half < 2; ++half) {
                if (!mbar_wait(half ? &bars->p_full[x] : &bars->p_half[x], parity)) failed = 3;
                tc_fence_after_sync();
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  umma_bf16_ts(o_tmem, s_tmem + half * 32 + k * 8, desc_add(vd, half * 4 * (2048 >> 4) + k * (2048 >> 4)),
                               S::kIdescO, (k + half > 0 || pj > 0) ? 1u : 0u);
              }
              if (pj + 1 == pnx) umma_commit(&bars->o_full[x]);
            }
            if (j < nx) {
              if (j == 0) {
                if (!mbar_wait(&bars->q_full[q_slot], q_phase)) failed = 1;
                q_ab = x ? (q_ab & 0xff) | q_slot << 8 : (q_ab & ~0xff) | q_slot;
                if (++q_slot == kQ) {
                  q_slot = 0;
                  q_phase ^= 1;
                }
              }
              const int q_at = (q_ab >> (8 * x)) & 0xff;
              const uint64_t qd = desc_add(qd0, q_at * (S::kTileBytes >> 4));
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t off = (k >> 2) * (S::kHalfBytes >> 4) + (k & 3) * 2;
                umma_bf16_ss(s_tmem, desc_add(qd, off), desc_add(kd, off), S::kIdescS, k > 0 ? 1u : 0u);
              }
              umma_commit(&bars->s_full[x]);
              parities ^= 1u << x;
              if (j + 1 == nx) umma_commit(&bars->q_empty[q_at]);
            }
          }
          if (failed) {
            report_status(status, kFailMma | failed);
            break;
          }
          umma_commit(&bars->kv_empty[st]);
          ++step;
          owed = n > 0;
          pj = j;
          pn_a = n_a;
          pn_b = n_b;
          if (owed && ++j == n) {
            ok = reader.next<1>(bars, scratch, it);
            n = it.n;
            n_a = it.n_a;
            n_b = it.n_b;
            j = 0;
          }
        }
        umma_commit(&bars->drain);
        if (!mbar_wait(&bars->drain, 0)) report_status(status, kFailMma | 5);
      }
    } else {
      // ---------------- what some row may not see of V ----------------
      // (And the counters of the next launch's parts, which nothing here waits for.)
      if (p.cut) clear_next_bank(counters, turn, blockIdx.x * 32 + lane, gridDim.x * 32);
      Reader reader;
      Item it;
      uint32_t step = 0, cleared[2] = {0, 0};
      bool owed = false;
      bool ok = true;
      while (ok) {
        Item* const held = &scratch->items[reader.slot];  // (by the softmax warps, until the item ends)
        if (!reader.next<32, true>(bars, scratch, it) || it.n < 0) break;
        if (it.n == 0 && owed) ++step;  // the step without scores
        owed = it.n > 0;
        // (Of the item's last row. A tile that is looked at holds some key that it sees.)
        const int last_seen = p.causal ? min(it.base + min(it.valid, 2 * p.tile_tokens) - 1, it.lk) : it.lk;
        for (int j = min(it.cut_from, it.last_rows ? it.n - 1 : it.n); j < it.n; ++j) {
          // Its V tile comes with the step behind its scores'.
          const int st = (step + j + 1) & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_raw[st], (st ? cleared[1] : cleared[0]) & 1));
          if (!ok) {
            if (lane == 0) report_status(status, kFailClear | 1);
            break;
          }
          ++(st ? cleared[1] : cleared[0]);
          // Rows that all of the item's rows see, that some see, and that none does.
          uint8_t* const tile = smem + OFF_V + st * S::kTileBytes;
          const int start = (it.lo + j) * BN, some = max(it.base - start, 0), none = min(last_seen - start, BN);
          for (int h = 0; h < S::kHalves; ++h) {
            uint4* const at = reinterpret_cast<uint4*>(tile + h * S::kHalfBytes);
            for (int i = none * 8 + lane; i < BN * 8; i += 32) at[i] = make_uint4(0, 0, 0, 0);
          }
          if (j >= it.cut_from && has_special<T, S::kHalves>(tile, some, none)) {
            clear_special<T>(tile, S::kHalves, some, none);
            if (lane == 0 && j < it.n_a) held->special[0] = true;
            if (lane == 0 && j < it.n_b) held->special[1] = true;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->kv_full[st]);
        }
        step += it.n;
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
    const int i = x * p.tile_tokens + row / group, head = row % group;  // the query row, from tile A's first
    const bool used = row < p.tile_tokens * group;
    const float scale2 = p.scale * 1.4426950408889634f;
    const bool wide = ((p.o | (uint64_t)(2 * (p.o_tok | p.o_head))) & 31) == 0;
    uint32_t s_count = 0, o_count = 0, part_count = 0;
    Reader reader;
    for (;;) {
      const Item* it = reader.hold(bars, scratch);
      if (!it) {
        if (lane == 0) report_status(status, kFailSoftmax | 2);
        break;
      }
      if (it->n < 0) {
        reader.done(bars);
        break;
      }
      // Rows of no query compute on whatever is there and are not stored.
      const int seen = p.causal && used && i < it->valid ? clamp_index((int64_t)it->base + i, 0, it->lk) : it->lk;
      const int nx = x ? it->n_b : it->n_a;
      int valid = seen - it->lo * BN;
      float m = kLowest, l = 0.f;
      bool ok = true;
      for (int j = 0; j < nx; ++j, valid -= BN) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[x], s_count & 1));
        if (!ok) break;
        ++s_count;
        tc_fence_after_sync();
        softmax_step<T, HD>(s_tmem, o_tmem, valid, j > 0, scale2, m, l, &bars->p_half[x], &bars->p_full[x]);
      }
      if (ok && nx > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[x], o_count & 1));
        ++o_count;
        tc_fence_after_sync();
      }
      if (!ok) {
        if (lane == 0) report_status(status, kFailSoftmax | 1);
        break;
      }
      const bool in = used && i < it->valid;
      const int first = it->row, head0 = it->hk * group;
      if (nx > 0 && it->special[x])
        add_special<T, HD>(p, *it, o_tmem, max(it->base, (it->lo + it->cut_from) * BN),
                           min(in ? seen : 0, (it->lo + nx) * BN));
      if (it->parts == 1) {
        reader.done(bars);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* to = reinterpret_cast<T*>(p.o) + (first + i) * p.o_tok + (head0 + head) * p.o_head;
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
          if (in) {
#pragma unroll
            for (int d = 0; d < 32; d += 16) {
              uint32_t w[8];
#pragma unroll
              for (int q = 0; q < 8; ++q)
                w[q] = pack2<T>(__uint_as_float(o[d + 2 * q]) * inv, __uint_as_float(o[d + 2 * q + 1]) * inv);
              store32(to + c + d, w, wide);
            }
          }
          __syncwarp();
        }
        continue;
      }
      // ---- a part: its rows go to the workspace, and who brings the last part joins them ----
      const int parts = it->parts, slot0 = it->slot, stride = it->stride;
      const long long own = (long long)(slot0 + it->part * stride) * kTileRows;
      const int rows = min(p.tile_tokens, it->valid - x * p.tile_tokens) * group;
      reader.done(bars);
      float2* const stats = reinterpret_cast<float2*>(p.work + kWorkFront) + x * 128;
      float* const parts_o = reinterpret_cast<float*>(p.work + tile_rows_at(2 * gridDim.x)) + (long long)x * 128 * HD;
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
#pragma unroll
        for (int k = 0; k < 4; ++k) store32(parts_o + (own + row) * HD + c + 8 * k, &o[8 * k], true);
      }
      stats[own + row] = make_float2(m, l);
      __threadfence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->part_stored[x]);
      if (quarter == 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->part_stored[x], part_count & 1));
        if (ok && lane == 0) {
          scratch->last[x] = atomicAdd(counters + tile_parts_at(turn, slot0, x), 1) == parts - 1;
          mbar_arrive(&bars->part_known[x]);
        }
      }
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars->part_known[x], part_count & 1));
      if (!ok) {
        if (lane == 0) report_status(status, kFailSoftmax | 3);
        break;
      }
      ++part_count;
      if (scratch->last[x]) {
        __threadfence();
        constexpr int kLanes = HD / 4, kStep = 128 / kLanes;  // lanes of a row, rows at a time
        const int column = row % kLanes * 4;
        for (int at = row / kLanes; at < rows; at += 4 * kStep)
          join_parts<HD>(stats, parts_o, slot0, stride, parts, at, kStep, rows, column, [&](int r, float4 v) {
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + (first + x * p.tile_tokens + r / group) * p.o_tok +
                                      (head0 + r % group) * p.o_head + column) =
                make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
          });
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

}  // namespace

// One CTA per SM at 168 registers a thread; the warpgroups re-divide them (88 and 208).
#define TB_TILE_ENTRY(suffix, T, HD)                                                                                \
  extern "C" __global__ void __launch_bounds__(tb::kTileThreads, 1)                                                 \
      attention_tiles_##suffix(const __grid_constant__ tb::AttnParams p, const __grid_constant__ CUtensorMap tmap_q, \
                               const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, \
                               uint32_t* status) {                                                                  \
    attention_tiles<T, HD>(p, tmap_q, tmap_k, tmap_v, status);                                                      \
  }

TB_TILE_ENTRY(bf16_d128, __nv_bfloat16, 128)
TB_TILE_ENTRY(bf16_d64, __nv_bfloat16, 64)
TB_TILE_ENTRY(f16_d128, __half, 128)
TB_TILE_ENTRY(f16_d64, __half, 64)
