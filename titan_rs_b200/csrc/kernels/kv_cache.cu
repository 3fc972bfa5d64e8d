// The paged key/value cache: the pages and slots of a step, and the write of its new rows.
#include "kv_params.cuh"

namespace {

using namespace tb;

// One row chunk of B bytes, cache[slot] = rows[token], for K (z = 0) and V (z = 1).
template <typename Chunk>
__device__ __forceinline__ void append_rows(const char* __restrict__ rows, char* __restrict__ cache,
                                            const int* __restrict__ slots, int tokens, int heads, int chunks, int page,
                                            long long limit, long long r_tok, long long r_head, long long c_page,
                                            long long c_tok, long long c_head) {
  const long long per_token = (long long)heads * chunks, total = tokens * per_token;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_token), rest = (int)(i % per_token);
    const int h = rest / chunks, c = rest % chunks;
    const int slot = __ldg(slots + t);
    if (slot < 0 || slot >= limit) continue;
    const Chunk x = *reinterpret_cast<const Chunk*>(rows + t * r_tok + h * r_head + c * (long long)sizeof(Chunk));
    *reinterpret_cast<Chunk*>(cache + (slot / page) * c_page + (slot % page) * c_tok + h * c_head +
                              c * (long long)sizeof(Chunk)) = x;
  }
}

template <typename Chunk>
__device__ __forceinline__ void append_body(const AppendParams& p) {
  const bool v = blockIdx.y != 0;
  append_rows<Chunk>(reinterpret_cast<const char*>(v ? p.v : p.k), reinterpret_cast<char*>(v ? p.v_cache : p.k_cache),
                     reinterpret_cast<const int*>(p.slots), p.tokens, p.heads, p.chunks, p.page, p.limit,
                     v ? p.v_tok : p.k_tok, v ? p.v_head : p.k_head, v ? p.vc_page : p.kc_page,
                     v ? p.vc_tok : p.kc_tok, v ? p.vc_head : p.kc_head);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) kv_append_16(const __grid_constant__ tb::AppendParams p) {
  append_body<uint4>(p);
}
extern "C" __global__ void __launch_bounds__(256) kv_append_4(const __grid_constant__ tb::AppendParams p) {
  append_body<uint32_t>(p);
}
extern "C" __global__ void __launch_bounds__(256) kv_append_2(const __grid_constant__ tb::AppendParams p) {
  append_body<uint16_t>(p);
}

// Pages and slots of one step, one CTA. For request b with ctx tokens cached and `add` new ones:
//   held = ceil(ctx / page), wanted = ceil((ctx + add) / page), need = wanted - held;
//   its new pages are free[first .. first + need), first = the sum of need over earlier requests;
//   a new token at position x has slot page_of(x / page) * page + x % page.
// A request is refused, keeping ctx tokens and giving its new tokens slot -1, when a length
// is negative, its row of the table is too short, its tokens pass the slot map's end, or the
// free list ends before its pages. One thread walks the requests (the sums), then all
// threads fill in the tokens.
extern "C" __global__ void __launch_bounds__(1024)
    kv_plan(const int* __restrict__ ctx, const int* __restrict__ add, const int* __restrict__ free_pages,
            int* __restrict__ table, int* __restrict__ lens, int* __restrict__ cu, int* __restrict__ slots,
            int* __restrict__ status, int batch, int n_free, int width, long long table_row, int tokens, int page) {
  extern __shared__ int first_of[];  // first new page of each request, or -1 when refused
  if (threadIdx.x == 0) {
    long long at = 0, taken = 0, given = 0;
    int refused = 0;
    for (int b = 0; b < batch; ++b) {
      const long long c = max(ctx[b], 0), n = max(add[b], 0);
      const long long held = (c + page - 1) / page, wanted = (c + n + page - 1) / page;
      cu[b] = (int)(at < tokens ? at : tokens);
      const bool fits = ctx[b] >= 0 && add[b] >= 0 && wanted <= width && at + n <= tokens;
      const long long need = fits ? wanted - held : 0;
      const bool served = fits && taken + need <= n_free;
      first_of[b] = served ? (int)taken : -1;
      lens[b] = (int)(served ? c + n : c);
      if (served) given += need;
      refused += served ? 0 : 1;
      taken += need;
      at += n;
    }
    cu[batch] = (int)(at < tokens ? at : tokens);
    status[0] = (int)given;
    status[1] = refused;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < batch; b += blockDim.x) {
    if (first_of[b] < 0) continue;
    const int held = (int)(((long long)ctx[b] + page - 1) / page);
    const int wanted = (int)(((long long)ctx[b] + add[b] + page - 1) / page);
    for (int i = held; i < wanted; ++i) table[b * table_row + i] = free_pages[first_of[b] + i - held];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < tokens; t += blockDim.x) {
    int lo = 0, hi = batch + 1;  // the last request that starts at or before token t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    const int b = lo - 1;
    int slot = -1;
    if (b < batch && first_of[b] >= 0) {
      const int x = ctx[b] + t - cu[b];
      const int id = table[b * table_row + x / page];
      const long long at = (long long)id * page + x % page;
      if (id >= 0 && at <= 0x7fffffff) slot = (int)at;
    }
    slots[t] = slot;
  }
}
