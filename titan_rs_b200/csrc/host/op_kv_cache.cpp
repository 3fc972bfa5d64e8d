// "kv_cache.plan" and "kv_cache.append": the bookkeeping and the write of a paged key/value
// cache, beside the attention that reads it (op_attention.cpp). No counterpart in the
// reference; the checks and messages follow the manner of its operators.
#include <algorithm>

#include "../kernels/kv_params.cuh"
#include "ops_common.hpp"

using namespace tb;

namespace {

// Requests the plan kernel takes in one call (its shared memory holds two words for each).
constexpr uint64_t kMaxPlanRequests = 16384;

bool same_rows(const tb_tensor* rows, const tb_tensor* cache) {
  return rows->rank == 3 && cache->rank == 4 && rows->shape[1] == cache->shape[2] && rows->shape[2] == cache->shape[3];
}

// The widest chunk (16, 4 or 2 bytes) that all of the or-ed addresses, steps and lengths are
// multiples of.
unsigned chunk_of(uint64_t bits) { return (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 2; }

// Whether the kernel's 32-bit count of a token's chunks, of K and V, holds them.
bool chunks_fit(uint64_t heads, uint64_t row_bytes, unsigned chunk) {
  return 2 * heads * (row_bytes / chunk) + kAppendThreads <= 0x7fffffffull;
}

}  // namespace

extern "C" tb_status tb_op_kv_append(tb_session* session, tb_stream* stream, const tb_tensor* k, const tb_tensor* v,
                                     const tb_tensor* slot_map, const tb_tensor* k_cache, const tb_tensor* v_cache,
                                     const tb_attr* attrs, uint32_t num_attrs, tb_event** out) try {
  (void)attrs;
  Session* s = reinterpret_cast<Session*>(session);
  if (!k || !v || !slot_map || !k_cache || !v_cache)
    return contract("kv_cache.append requires K, V and slot_map, and the K and V caches as outputs");
  if (num_attrs) return unsupported("kv_cache.append does not implement attributes");
  const uint32_t dt = k->dtype;
  if ((dt != TB_F32 && dt != TB_F16 && dt != TB_BF16) || v->dtype != dt || k_cache->dtype != dt ||
      v_cache->dtype != dt)
    return contract("kv_cache.append requires F32, F16 or BF16 rows and caches of one dtype");
  if (!same_rows(k, k_cache) || !same_rows(v, v_cache))
    return contract("kv_cache.append requires rank-3 [T, H, D] rows and rank-4 [pages, page, H, D] caches of one H and D");
  if (v->shape[0] != k->shape[0] || v->shape[1] != k->shape[1] || v->shape[2] != k->shape[2])
    return contract("kv_cache.append requires K and V rows of one shape");
  for (int i = 0; i < 4; ++i)
    if (k_cache->shape[i] != v_cache->shape[i]) return contract("kv_cache.append requires K and V caches of one shape");
  const uint64_t T = k->shape[0], H = k->shape[1], D = k->shape[2], pages = k_cache->shape[0], page = k_cache->shape[1];
  if (T == 0 || H == 0 || D == 0 || pages == 0 || page == 0)
    return contract("kv_cache.append requires non-zero dimensions");
  if (T > 0x7fffffffull || H > 0xffffull || D > 0xffffull || pages > 0x7fffffffull || page > 0x7fffffffull ||
      pages * page > 0x7fffffffull)
    return contract("kv_cache.append shape exceeds i32 ABI");
  if (!is_index(slot_map, 1) || slot_map->shape[0] != T)
    return contract("kv_cache.append requires a contiguous I32 slot_map [T]");
  if (!distinct_elements(k_cache) || !distinct_elements(v_cache))
    return contract("kv_cache.append requires caches whose elements do not overlap");
  const int64_t size = (int64_t)dtype_size(dt);  // (a power of two, so it may be multiplied with the or-ed steps)
  uint64_t steps = D;
  for (int i = 0; i < 2; ++i) steps |= (uint64_t)(step_of(k, i) | step_of(v, i));
  for (int i = 0; i < 3; ++i) steps |= (uint64_t)(step_of(k_cache, i) | step_of(v_cache, i));
  steps *= (uint64_t)size;
  if (!chunks_fit(H, D * size, chunk_of(steps))) return contract("kv_cache.append shape exceeds i32 ABI");
  if (!s) return set_error(TB_ERR_INVALID, "contract", "null session");
  tb_status rc;
  Stream* st = nullptr;
  Buffer *bk = nullptr, *bv = nullptr, *bs = nullptr, *bkc = nullptr, *bvc = nullptr;
  if ((rc = check_stream(s, stream, &st)) || (rc = strided_buffer(s, k, "kv_cache.append K", &bk)) ||
      (rc = strided_buffer(s, v, "kv_cache.append V", &bv)) ||
      (rc = strided_buffer(s, slot_map, "kv_cache.append slot_map", &bs)) ||
      (rc = strided_buffer(s, k_cache, "kv_cache.append K cache", &bkc)) ||
      (rc = strided_buffer(s, v_cache, "kv_cache.append V cache", &bvc)) || (rc = activate(s)))
    return rc;
  AppendParams p{};
  p.k = bk->ptr;
  p.v = bv->ptr;
  p.k_cache = bkc->ptr;
  p.v_cache = bvc->ptr;
  p.slots = bs->ptr;
  p.k_tok = step_of(k, 0) * size;
  p.k_head = step_of(k, 1) * size;
  p.v_tok = step_of(v, 0) * size;
  p.v_head = step_of(v, 1) * size;
  p.kc_page = step_of(k_cache, 0) * size;
  p.kc_tok = step_of(k_cache, 1) * size;
  p.kc_head = step_of(k_cache, 2) * size;
  p.vc_page = step_of(v_cache, 0) * size;
  p.vc_tok = step_of(v_cache, 1) * size;
  p.vc_head = step_of(v_cache, 2) * size;
  p.limit = (long long)(pages * page);
  p.tokens = (int)T;
  p.heads = (int)H;
  p.page = (int)page;
  const unsigned chunk = chunk_of(steps | p.k | p.v | p.k_cache | p.v_cache);
  if (!chunks_fit(H, D * size, chunk)) return contract("kv_cache.append shape exceeds i32 ABI");
  const char* entry = chunk == 16 ? "kv_append_16" : chunk == 4 ? "kv_append_4" : "kv_append_2";
  p.chunks = (int)(D * size / chunk);
  CUfunction fn = nullptr;
  if ((rc = builtin_function(s, "kv_cache", entry, &fn))) return rc;
  // A pass of a block covers kAppendThreads chunks of whole tokens. Few passes get a block each;
  // many are taken four to a thread, as the kernel unrolls.
  const uint64_t at_once = std::max<uint64_t>(1, kAppendThreads / (2 * H * (uint64_t)p.chunks));
  const uint64_t passes = (T + at_once - 1) / at_once, few = 2 * (uint64_t)s->sm_count;
  const uint64_t grid = passes <= few ? passes : std::max(few, (passes + 3) / 4);
  void* params[] = {&p};
  if ((rc = launch_overlapped(s, st, fn, (unsigned)grid, 1, kAppendThreads, 0, params, entry))) return rc;
  return record_event(s, st, nullptr, out);
} catch (const std::exception& e) {
  return tb::caught(e);
}

extern "C" tb_status tb_op_kv_plan(tb_session* session, tb_stream* stream, const tb_tensor* context_lens,
                                   const tb_tensor* new_lens, const tb_tensor* free_pages, const tb_tensor* block_table,
                                   const tb_tensor* seq_lens, const tb_tensor* cu_seqlens, const tb_tensor* slot_map,
                                   const tb_tensor* status, const tb_attr* attrs, uint32_t num_attrs, tb_event** out) try {
  Session* s = reinterpret_cast<Session*>(session);
  if (!context_lens || !new_lens || !free_pages || !block_table || !seq_lens || !cu_seqlens || !slot_map || !status)
    return contract("kv_cache.plan requires context_lens, new_lens and free_pages, and the outputs block_table, "
                    "seq_lens, cu_seqlens, slot_map and status");
  if (num_attrs && !attrs) return contract("kv_cache.plan attributes are null");
  for (uint32_t i = 0; i < num_attrs; ++i)
    if (!attrs[i].key || strcmp(attrs[i].key, "page_size") != 0)
      return unsupported("kv_cache.plan does not implement attributes other than page_size");
  int64_t page = 0;
  tb_status rc = int_attr(attrs, num_attrs, "page_size", nullptr, &page);
  if (rc) return rc;
  if (page < 1 || page > 0x7fffffff) return contract("kv_cache.plan page_size must be positive");
  if (!is_index(context_lens, 1) || !is_index(new_lens, 1) || !is_index(free_pages, 1) || !is_index(seq_lens, 1) ||
      !is_index(cu_seqlens, 1) || !is_index(slot_map, 1) || !is_index(status, 1) || !is_index(block_table, 2))
    return contract("kv_cache.plan requires I32 tensors with contiguous rows");
  const uint64_t B = context_lens->shape[0], W = block_table->shape[1], T = slot_map->shape[0],
                 F = free_pages->shape[0];
  if (B == 0 || W == 0 || T == 0 || F == 0) return contract("kv_cache.plan requires non-zero dimensions");
  if (new_lens->shape[0] != B || seq_lens->shape[0] != B || cu_seqlens->shape[0] != B + 1 ||
      block_table->shape[0] != B)
    return contract("kv_cache.plan requires [batch] lengths, a [batch + 1] cu_seqlens and a [batch, pages] block_table");
  if (status->shape[0] != 2) return contract("kv_cache.plan requires a status of two words");
  // (The kernel steps over tokens and table entries in 32 bits.)
  if (W > 0x7f000000ull || T > 0x7f000000ull || F > 0x7fffffffull) return contract("kv_cache.plan shape exceeds i32 ABI");
  if (B > kMaxPlanRequests) return unsupported("kv_cache.plan does not implement batches above 16384 requests");
  if (!distinct_elements(block_table)) return contract("kv_cache.plan requires a block_table whose rows do not overlap");
  if (!s) return set_error(TB_ERR_INVALID, "contract", "null session");
  Stream* st = nullptr;
  Buffer *bc = nullptr, *bn = nullptr, *bf = nullptr, *bt = nullptr, *bl = nullptr, *bcu = nullptr, *bm = nullptr,
         *bs = nullptr;
  if ((rc = check_stream(s, stream, &st)) || (rc = strided_buffer(s, context_lens, "kv_cache.plan context_lens", &bc)) ||
      (rc = strided_buffer(s, new_lens, "kv_cache.plan new_lens", &bn)) ||
      (rc = strided_buffer(s, free_pages, "kv_cache.plan free_pages", &bf)) ||
      (rc = strided_buffer(s, block_table, "kv_cache.plan block_table", &bt)) ||
      (rc = strided_buffer(s, seq_lens, "kv_cache.plan seq_lens", &bl)) ||
      (rc = strided_buffer(s, cu_seqlens, "kv_cache.plan cu_seqlens", &bcu)) ||
      (rc = strided_buffer(s, slot_map, "kv_cache.plan slot_map", &bm)) ||
      (rc = strided_buffer(s, status, "kv_cache.plan status", &bs)) || (rc = activate(s)))
    return rc;
  // The kernel's blocks read the inputs while others write.
  const struct {
    uint64_t ptr, bytes;
  } ranges[] = {{bt->ptr, 4 * ((B - 1) * (uint64_t)step_of(block_table, 0) + W)},
                {bl->ptr, 4 * B},
                {bcu->ptr, 4 * (B + 1)},
                {bm->ptr, 4 * T},
                {bs->ptr, 8},
                {bc->ptr, 4 * B},
                {bn->ptr, 4 * B},
                {bf->ptr, 4 * F}};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 8; ++j)
      if (ranges[i].ptr < ranges[j].ptr + ranges[j].bytes && ranges[j].ptr < ranges[i].ptr + ranges[i].bytes)
        return contract("kv_cache.plan requires outputs that share no memory with the inputs or each other");
  // Large batches want more threads for the sums, small ones fewer to wait for.
  const unsigned threads = B > 256 ? 512 : 256;
  const char* entry = B > 256 ? "kv_plan_512" : "kv_plan_256";
  CUfunction fn = nullptr;
  if ((rc = builtin_function(s, "kv_cache", entry, &fn))) return rc;
  PlanParams p{};
  p.ctx = bc->ptr;
  p.add = bn->ptr;
  p.free_pages = bf->ptr;
  p.table = bt->ptr;
  p.lens = bl->ptr;
  p.cu = bcu->ptr;
  p.slots = bm->ptr;
  p.status = bs->ptr;
  p.table_row = step_of(block_table, 0);
  p.batch = (int)B;
  p.n_free = (int)F;
  p.width = (int)W;
  p.tokens = (int)T;
  p.page = (int)page;
  // A token a thread; more blocks than resident ones would only repeat the sums.
  const uint64_t grid = std::min((std::max(T, 8 * B) + threads - 1) / threads, (uint64_t)s->sm_count * 2);
  void* params[] = {&p};
  if ((rc = launch_overlapped(s, st, fn, (unsigned)grid, 1, threads, (unsigned)((2 * B + 1) * sizeof(int)), params,
                              entry)))
    return rc;
  return record_event(s, st, nullptr, out);
} catch (const std::exception& e) {
  return tb::caught(e);
}
