// The paged key/value cache: the pages and slots of a step, and the write of its new rows.
#include "attn_params.cuh"
#include "kv_params.cuh"

namespace {

using namespace tb;

// cache[slots[t]] = rows[t] for K and V, in chunks of 2, 4 or 16 bytes.
//
// A copy, bound by the HBM: every row is read and written once. A thread keeps its place in a
// token's row (K or V, head, chunk) and steps over tokens, four at a time, so that the
// divisions are done once and four loads are in flight.
template <typename Chunk>
__device__ __forceinline__ void append_rows(const AppendParams& p) {
  begin_after_earlier_grids();
  const int per = p.heads * p.chunks, places = 2 * per;  // a token's chunks of K, and of both
  const int at_once = max(1, kAppendThreads / places);   // tokens of a pass of the block
  const int local = places <= kAppendThreads ? threadIdx.x / places : 0;
  if (local >= at_once) return;
  const long long step = (long long)gridDim.x * at_once;
  const int* const slots = reinterpret_cast<const int*>(p.slots);
  for (int place = places <= kAppendThreads ? threadIdx.x % places : threadIdx.x; place < places;
       place += kAppendThreads) {
    const bool v = place >= per;
    const int h = (v ? place - per : place) / p.chunks, c = (v ? place - per : place) % p.chunks;
    const char* const from =
        reinterpret_cast<const char*>(v ? p.v : p.k) + h * (v ? p.v_head : p.k_head) + c * (int)sizeof(Chunk);
    char* const to = reinterpret_cast<char*>(v ? p.v_cache : p.k_cache) + h * (v ? p.vc_head : p.kc_head) +
                     c * (int)sizeof(Chunk);
    const long long r_tok = v ? p.v_tok : p.k_tok, c_page = v ? p.vc_page : p.kc_page, c_tok = v ? p.vc_tok : p.kc_tok;
    for (long long t = (long long)blockIdx.x * at_once + local; t < p.tokens; t += 4 * step) {
      Chunk x[4];
      int slot[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = t + i * step < p.tokens;
        slot[i] = in ? slots[t + i * step] : -1;
        if (in) x[i] = *reinterpret_cast<const Chunk*>(from + (t + i * step) * r_tok);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (slot[i] >= 0 && slot[i] < p.limit)
          *reinterpret_cast<Chunk*>(to + (slot[i] / p.page) * c_page + (slot[i] % p.page) * c_tok) = x[i];
    }
  }
}

// The sum of `mine` over the threads before this one, and over all (total). `words` holds one
// word a warp and is free again when the next barrier has passed.
template <int kThreads>
__device__ __forceinline__ long long sum_before(long long mine, long long* words, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += x;
  }
  if (lane == 31) words[warp] = upto;
  __syncthreads();
  long long before = upto - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += words[w];
    total += words[w];
  }
  return before;
}

// Pages and slots of one step. For request b with ctx tokens cached and `add` new ones:
//   held = ceil(ctx / page), wanted = ceil((ctx + add) / page), need = wanted - held;
//   its new pages are free[first .. first + need), first = the sum of need over earlier requests;
//   a new token at position x has slot page_of(x / page) * page + x % page.
// A request is refused, keeping ctx tokens and giving its new tokens slot -1, when a length
// is negative or passes 2^31 - 1, its row of the table is too short, its tokens pass the slot
// map's end, or the free list ends before its pages.
//
// Some kilobytes, so a few memory latencies and the launch are all there is: every block
// repeats the sums over the requests (two scans, of tokens and of pages) instead of waiting for
// another's, keeps each request's first token and first page in shared memory, and fills in its
// share of the tokens, requests and table rows. Old pages are only read and new ones only
// taken from the free list, so no block needs what another writes. A launch takes 5.0 us for
// 64 single tokens (256 threads; 5.5 with 512) and 6.9 us for 700 prompts of 46,000 tokens (512
// threads; 8.4 with 256).
template <int kThreads>
__device__ __forceinline__ void plan_step(const PlanParams& p) {
  extern __shared__ int words[];
  int* const start = words;                 // first token of request b (batch + 1 of them)
  int* const first = words + p.batch + 1;   // its first new page's place in the free list, or -1 when refused
  __shared__ long long sums[2][kThreads / 32];
  __shared__ int given, refused;
  const int* const ctx = reinterpret_cast<const int*>(p.ctx);
  const int* const add = reinterpret_cast<const int*>(p.add);
  const int* const free_pages = reinterpret_cast<const int*>(p.free_pages);
  int* const table = reinterpret_cast<int*>(p.table);
  if (threadIdx.x == 0) given = refused = 0;
  begin_after_earlier_grids();

  const int per = (p.batch + kThreads - 1) / kThreads;
  const int lo = min((int)threadIdx.x * per, p.batch), hi = min(lo + per, p.batch);
  const auto pages = [&](long long tokens) { return (tokens + p.page - 1) / p.page; };
  long long tokens = 0, total = 0;
  for (int b = lo; b < hi; ++b) tokens += max(add[b], 0);
  long long at = sum_before<kThreads>(tokens, sums[0], total);
  long long need = 0;
  for (int b = lo; b < hi; ++b) {
    const long long c = ctx[b], n = add[b];
    const bool fits = c >= 0 && n >= 0 && c + n <= 0x7fffffff && pages(c + n) <= p.width && at + n <= p.tokens;
    const int own = fits ? (int)(pages(c + n) - pages(c)) : -1;
    start[b] = (int)min(at, (long long)p.tokens);
    first[b] = own;
    need += max(own, 0);
    at += max(n, 0ll);
  }
  if (threadIdx.x == 0) start[p.batch] = (int)min(total, (long long)p.tokens);
  long long taken = sum_before<kThreads>(need, sums[1], total);
  int my_given = 0, my_refused = 0;
  for (int b = lo; b < hi; ++b) {
    const int own = first[b];
    const bool served = own >= 0 && taken + own <= p.n_free;
    first[b] = served ? (int)taken : -1;
    taken += max(own, 0);
    my_given += served ? own : 0;
    my_refused += served ? 0 : 1;
  }
  if (blockIdx.x == 0 && (my_given || my_refused)) {
    atomicAdd(&given, my_given);
    atomicAdd(&refused, my_refused);
  }
  __syncthreads();

  const int tid = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;
  if (tid == 0) {
    reinterpret_cast<int*>(p.status)[0] = given;
    reinterpret_cast<int*>(p.status)[1] = refused;
  }
  for (int b = tid; b <= p.batch; b += threads) {
    reinterpret_cast<int*>(p.cu)[b] = start[b];
    if (b < p.batch) {
      const int c = max(ctx[b], 0);
      reinterpret_cast<int*>(p.lens)[b] = first[b] >= 0 ? c + add[b] : c;
    }
  }
  // The new entries of the table, a warp a request.
  for (int b = tid >> 5; b < p.batch; b += threads >> 5) {
    if (first[b] < 0) continue;
    const long long c = ctx[b];
    const int held = (int)pages(c), wanted = (int)pages(c + add[b]);
    for (int i = held + (int)(threadIdx.x & 31); i < wanted; i += 32)
      table[b * p.table_row + i] = free_pages[first[b] + i - held];
  }
  for (int t = tid; t < p.tokens; t += threads) {
    int below = 0, above = p.batch + 1;  // the last request that starts at or before token t
    while (below < above) {
      const int mid = (below + above) >> 1;
      if (start[mid] <= t) below = mid + 1;
      else above = mid;
    }
    const int b = below - 1;
    int slot = -1;
    if (b < p.batch && first[b] >= 0) {
      const int c = ctx[b], x = c + t - start[b], index = x / p.page, held = (int)pages(c);
      const int id = index < held ? table[b * p.table_row + index] : free_pages[first[b] + index - held];
      const long long place = (long long)id * p.page + x % p.page;
      if (id >= 0 && place <= 0x7fffffff) slot = (int)place;
    }
    reinterpret_cast<int*>(p.slots)[t] = slot;
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(tb::kAppendThreads)
    kv_append_16(const __grid_constant__ tb::AppendParams p) {
  append_rows<uint4>(p);
}
extern "C" __global__ void __launch_bounds__(tb::kAppendThreads) kv_append_4(const __grid_constant__ tb::AppendParams p) {
  append_rows<uint32_t>(p);
}
extern "C" __global__ void __launch_bounds__(tb::kAppendThreads) kv_append_2(const __grid_constant__ tb::AppendParams p) {
  append_rows<uint16_t>(p);
}
extern "C" __global__ void __launch_bounds__(256) kv_plan_256(const __grid_constant__ tb::PlanParams p) {
  plan_step<256>(p);
}
extern "C" __global__ void __launch_bounds__(512) kv_plan_512(const __grid_constant__ tb::PlanParams p) {
  plan_step<512>(p);
}
