// "attention.varlen" and "attention.paged": attention over packed sequences of different
// lengths, with grouped key heads, over contiguous K and V or over a paged cache. No
// counterpart in the reference, whose attention takes one [B, H, T, D] block
// (titan-runtime/src/lib.rs:1090-1151); the checks and messages follow its manner.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "../kernels/attn_params.cuh"
#include "ops_common.hpp"

namespace tb {
namespace {

constexpr uint64_t kMaxBatch = 1ull << 30;

struct AttnAttrs {
  bool causal = false;
  double scale = 0.0;  // 0: 1/sqrt(D)
  uint64_t max_query = 0;  // 0: not given
  const char* candidate = nullptr;
};

tb_status parse_attrs(const tb_attr* attrs, uint32_t n, const char* op, bool paged, AttnAttrs* out) {
  out->causal = paged;
  if (n && !attrs) return contract(std::string(op) + " attributes are null");
  for (uint32_t i = 0; i < n; ++i) {
    const char* key = attrs[i].key ? attrs[i].key : "";
    if (strcmp(key, "causal") == 0 && !attrs[i].str && attrs[i].value >= 0 && attrs[i].value <= 1) {
      out->causal = attrs[i].value != 0;
    } else if (strcmp(key, "candidate") == 0 && attrs[i].str) {
      out->candidate = attrs[i].str;
    } else if (strcmp(key, "scale") == 0) {
      char* end = nullptr;
      out->scale = attrs[i].str ? strtod(attrs[i].str, &end) : 0.0;
      // (The kernels hold it, and its product with log2(e), as a float: a hidden score is -inf times
      // it, which is no number where it is zero.)
      const float held = (float)out->scale;
      if (!attrs[i].str || end == attrs[i].str || *end != '\0' || !(held > 0.f) || !std::isfinite(held * 1.4426950408889634f))
        return contract(std::string(op) + " scale must be a positive finite number of a float's range (decimal string)");
    } else if (paged && strcmp(key, "max_query_len") == 0) {
      if (attrs[i].str || attrs[i].value <= 0) return contract("attention.paged max_query_len must be a positive integer");
      out->max_query = (uint64_t)attrs[i].value;
    } else {
      return unsupported(std::string(op) + " does not implement attributes other than causal, scale" +
                         (paged ? ", max_query_len" : "") + " and candidate");
    }
  }
  return TB_OK;
}

struct AttnCall {
  AttnParams p{};
  uint32_t dtype = 0;
};

// Q [T, H, D] and the output of the same shape.
tb_status query_side(const char* op, const tb_tensor* q, const tb_tensor* output, AttnCall* c) {
  const std::string name(op);
  if (q->dtype != TB_BF16 && q->dtype != TB_F16) return contract(name + " requires BF16 or F16 Q, K, V, and output");
  if (output->dtype != q->dtype) return contract(name + " requires Q, K, V, and output of one dtype");
  if (q->rank != 3 || output->rank != 3) return contract(name + " requires rank-3 [T, H, D] Q and output");
  for (int a = 0; a < 3; ++a)
    if (output->shape[a] != q->shape[a]) return contract(name + " output shape mismatch");
  const uint64_t T = q->shape[0], H = q->shape[1], D = q->shape[2];
  if (T == 0 || H == 0 || D == 0) return contract(name + " requires non-zero T, H, and D dimensions");
  if (T > (uint64_t)kMaxRows || H > 0xffffull) return contract(name + " shape exceeds i32 ABI");
  if (D > 256) return unsupported(name + " does not implement head dimensions above 256");
  if (!distinct_elements(output)) return contract(name + " requires an output whose elements do not overlap");
  c->dtype = q->dtype;
  c->p.q_tok = step_of(q, 0);
  c->p.q_head = step_of(q, 1);
  c->p.o_tok = step_of(output, 0);
  c->p.o_head = step_of(output, 1);
  c->p.tq = (int32_t)T;
  c->p.heads = (int32_t)H;
  c->p.dim = (int32_t)D;
  return TB_OK;
}

// The grouping of query heads over key heads.
tb_status heads_match(const char* op, uint64_t kv_heads, AttnCall* c) {
  if (kv_heads == 0 || kv_heads > (uint64_t)c->p.heads || c->p.heads % (int)kv_heads != 0)
    return contract(std::string(op) + " requires a number of query heads that is a multiple of the key heads");
  c->p.kv_heads = (int32_t)kv_heads;
  return TB_OK;
}

// CUDA-core kernel: any head dimension up to 256, any alignment, any page size.
tb_status launch_rows(Session* s, Stream* st, AttnCall* c) {
  const bool bf = c->dtype == TB_BF16;
  const char* entry = bf ? "attention_rows_bf16" : "attention_rows_f16";
  CUfunction fn = nullptr;
  tb_status rc = builtin_function(s, "attn_rows", entry, &fn);
  if (rc) return rc;
  uint64_t grid = ((uint64_t)c->p.tq * c->p.heads + 7) / 8;  // 8 rows (warps) per 256-thread CTA
  if (grid > (uint64_t)s->sm_count * 64) grid = (uint64_t)s->sm_count * 64;
  void* params[] = {&c->p};
  return launch_overlapped(s, st, fn, (unsigned)grid, 1, 256, 0, params, entry);
}

// Whether 16-byte copies reach every row of Q, K and V.
bool rows_aligned(const AttnParams& p) {
  const uint64_t kv = p.k | p.v | (uint64_t)(2 * (p.k_tok | p.k_head | p.k_page | p.v_tok | p.v_head | p.v_page));
  const uint64_t q = p.q | (uint64_t)(2 * (p.q_tok | p.q_head));
  return (p.dim == 64 || p.dim == 128) && ((kv | q) & 15) == 0;
}

// Whether the tile kernel takes the call: 16-byte rows of the output too, a group that
// fits a tile, and pages that cut a 128-key tile evenly (or are cut by it).
bool tiles_fit(const AttnParams& p) {
  const uint64_t o = p.o | (uint64_t)(2 * (p.o_tok | p.o_head));
  const bool pages = !p.table || (p.page >= 8 && 128 % p.page == 0) || p.page % 128 == 0;
  return rows_aligned(p) && (o & 15) == 0 && p.heads / p.kv_heads <= 128 && pages;
}

// A map of rows of `dim` elements with up to three outer dimensions, copied in boxes of 64
// elements x `box`, 128-byte swizzled. A dimension of extent one may have a step of 0 here;
// the map wants some multiple of 16 bytes.
tb_status tmap_rows(CUtensorMap* map, uint32_t dtype, uint64_t base, int rank, const uint64_t* extents,
                    const int64_t* steps, const uint32_t* box) {
  cuuint64_t dims[4], strides[3];
  cuuint32_t boxes[4] = {64, 1, 1, 1}, elem[4] = {1, 1, 1, 1};
  dims[0] = extents[0];
  for (int i = 1; i < rank; ++i) {
    dims[i] = extents[i];
    strides[i - 1] = steps[i] ? (cuuint64_t)steps[i] * 2 : extents[0] * 2;
    boxes[i] = box[i];
    if (strides[i - 1] >= (1ull << 40)) return unsupported("attention strides of 2^40 bytes and more are not implemented");
  }
  TB_CU("cuTensorMapEncodeTiled",
        driver()->cuTensorMapEncodeTiled(
            map, dtype == TB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank,
            reinterpret_cast<void*>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
  return TB_OK;
}

// Tensor-core kernel for all requests but the token kernel's. `longest`: query rows of a request
// at most, as the caller says.
tb_status launch_tiles(Session* s, Stream* st, AttnCall* c, uint64_t longest) {
  AttnParams& p = c->p;
  const std::string suffix = std::string(c->dtype == TB_BF16 ? "bf16" : "f16") + "_d" + std::to_string(p.dim);
  const std::string entry = "attention_tiles_" + suffix;
  CUfunction fn = nullptr;
  tb_status rc = builtin_function(s, "attn_tiles", entry.c_str(), &fn);
  if (rc) return rc;
  // The kernel's warpgroups re-divide the registers the CTA was launched with; a launch
  // with fewer than it assumes would leave the softmax warpgroups waiting for registers.
  int regs = 0;
  TB_CU("cuFuncGetAttribute", driver()->cuFuncGetAttribute(&regs, CU_FUNC_ATTRIBUTE_NUM_REGS, fn));
  if (regs < kTileLaunchRegs)
    return unsupported(entry + " was built with fewer registers than its warpgroups share");
  const int group = p.heads / p.kv_heads;
  p.tile_tokens = 128 / group;
  CUtensorMap mq, mk, mv;
  const uint64_t q_ext[] = {(uint64_t)p.dim, (uint64_t)p.heads, (uint64_t)p.tq};
  const int64_t q_steps[] = {1, p.q_head, p.q_tok};
  const uint32_t q_box[] = {64, (uint32_t)group, (uint32_t)p.tile_tokens};
  const uint64_t kv_ext[] = {(uint64_t)p.dim, (uint64_t)p.kv_heads, (uint64_t)(p.table ? p.page : p.tk),
                             (uint64_t)(p.table ? p.pages : 1)};
  const int64_t k_steps[] = {1, p.k_head, p.k_tok, p.k_page}, v_steps[] = {1, p.v_head, p.v_tok, p.v_page};
  const uint32_t kv_box[] = {64, 1, (uint32_t)(p.table ? std::min(p.page, 128) : 128), 1};
  if ((rc = tmap_rows(&mq, c->dtype, p.q, 3, q_ext, q_steps, q_box)) ||
      (rc = tmap_rows(&mk, c->dtype, p.k, 4, kv_ext, k_steps, kv_box)) ||
      (rc = tmap_rows(&mv, c->dtype, p.v, 4, kv_ext, v_steps, kv_box)))
    return rc;
  // Items (pairs of tiles x key heads) at most: every request may end inside a pair. What the caller
  // says of the longest request only sizes the grid: a longer one has its items all the same,
  // and takes none from the others.
  const uint64_t rows = 2ull * p.tile_tokens, tq = (uint64_t)p.tq, batch = (uint64_t)p.batch;
  const uint64_t pairs = tq / rows + std::min(batch, tq);
  if (pairs * (uint64_t)p.kv_heads > 0x3fffffffull) return contract("attention work list exceeds 2^30 items");
  p.max_items = (int32_t)(pairs * (uint64_t)p.kv_heads);
  uint64_t grid = std::min(pairs, batch * ((longest + rows - 1) / rows)) * (uint64_t)p.kv_heads;
  // One CTA an SM, drawing items until there are no more. The kernel may cut long requests
  // where two parts of the smallest size fit their keys.
  const uint64_t keys = p.table ? (uint64_t)p.width * p.page : (uint64_t)p.tk;
  p.cut = keys > 128 * kTileMinPart ? 1 : 0;
  const uint64_t sms = (uint64_t)std::min(s->sm_count, kTileMaxCtas);
  grid = std::min(p.cut ? grid * kTileMaxParts : grid, sms);
  CUdeviceptr work = 0;
  const size_t bytes = p.cut ? tile_workspace_bytes(2 * (int)grid, p.dim) : kWorkFront;
  if ((rc = stream_workspace(s, st, bytes, &work))) return rc;
  p.work = work;
  CUdeviceptr status = s->status.device;
  void* params[] = {&p, &mq, &mk, &mv, &status};
  rc = launch_overlapped(s, st, fn, (unsigned)grid, 1, kTileThreads, (unsigned)tile_smem_bytes(p.dim), params,
                         entry.c_str());
  return rc;
}

// Decode kernel for the requests of at most p.token_rows (row, head) pairs per key head.
tb_status launch_tokens(Session* s, Stream* st, AttnCall* c) {
  const std::string entry = std::string("attention_tokens_") + (c->dtype == TB_BF16 ? "bf16" : "f16") + "_d" +
                            std::to_string(c->p.dim) + "_r" + std::to_string(c->p.token_rows);
  CUfunction fn = nullptr;
  tb_status rc = builtin_function(s, "attn_tokens", entry.c_str(), &fn);
  if (rc) return rc;
  const int ctas = std::min(token_per_sm(c->p.token_rows) * s->sm_count, kTokenMaxCtas);
  CUdeviceptr work = 0;
  if ((rc = stream_workspace(s, st, token_workspace_bytes(ctas, c->p.token_rows, c->p.dim), &work))) return rc;
  c->p.work = work;
  void* params[] = {&c->p};
  return launch_overlapped(s, st, fn, (unsigned)ctas, 1, kTokenThreads, (unsigned)token_smem_bytes(c->p.dim, c->p.token_rows), params,
                        entry.c_str());
}

tb_status run_attention(Session* s, Stream* st, const char* op, AttnCall* c, const AttnAttrs& a) {
  tb_status rc = activate(s);
  if (rc) return rc;
  c->p.causal = a.causal ? 1 : 0;
  c->p.scale = (float)(a.scale > 0.0 ? a.scale : 1.0 / std::sqrt((double)c->p.dim));
  const std::string only = a.candidate ? a.candidate : "";
  if (!only.empty() && only != "attention_rows" && only != "attention_tiles" &&
      !(c->p.table && only == "attention_tokens"))
    return contract(std::string("unknown ") + op + " candidate " + only);
  const uint64_t group = (uint64_t)(c->p.heads / c->p.kv_heads);
  const uint64_t longest = a.max_query && a.max_query < (uint64_t)c->p.tq ? a.max_query : (uint64_t)c->p.tq;
  const bool tiles = tiles_fit(c->p) && (only.empty() || only == "attention_tiles");
  const bool tokens = c->p.table && rows_aligned(c->p) && (only.empty() || only == "attention_tokens");
  const bool few = tokens && longest * group <= 32;  // every request has few rows: the caller's bound says so
  if ((only == "attention_tiles" && !tiles) || (only == "attention_tokens" && !few))
    return unsupported("candidate " + only + " does not take this shape, page size, alignment or max_query_len");
  std::lock_guard<std::mutex> lock(st->enqueue);
  // Steps of few rows are the token kernel's. Other steps take one launch of the tile kernel for
  // all requests: it reads single tokens' keys more slowly (64 requests of 300-8192 keys 119 us
  // against 97, four of 110-131 thousand 575 against 305), but a launch of each kernel costs
  // more where chunks fill the step (eight requests, two of them single tokens, 136 us
  // against 121). Where tiles do not fit, the token kernel still takes the single tokens.
  if (few || (tokens && !tiles && group <= 32)) {
    const uint64_t rows = few ? longest * group : group;
    c->p.token_rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    if ((rc = launch_tokens(s, st, c)) || few) return rc;
  }
  return tiles ? launch_tiles(s, st, c, longest) : launch_rows(s, st, c);
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" tb_status tb_op_attention_varlen(tb_session* session, tb_stream* stream, const tb_tensor* q,
                                            const tb_tensor* k, const tb_tensor* v, const tb_tensor* cu_seqlens_q,
                                            const tb_tensor* cu_seqlens_k, const tb_tensor* output,
                                            const tb_attr* attrs, uint32_t num_attrs, tb_event** out) try {
  static const char* const op = "attention.varlen";
  Session* s = reinterpret_cast<Session*>(session);
  if (!q || !k || !v || !cu_seqlens_q || !output)
    return contract("attention.varlen requires Q, K, V, cu_seqlens_q and an optional cu_seqlens_k");
  AttnAttrs a;
  AttnCall c;
  tb_status rc;
  if ((rc = parse_attrs(attrs, num_attrs, op, false, &a)) || (rc = query_side(op, q, output, &c))) return rc;
  if (k->dtype != q->dtype || v->dtype != q->dtype)
    return contract("attention.varlen requires Q, K, V, and output of one dtype");
  if (k->rank != 3 || v->rank != 3) return contract("attention.varlen requires rank-3 [T, H, D] K and V");
  for (int i = 0; i < 3; ++i)
    if (k->shape[i] != v->shape[i]) return contract("attention.varlen requires K and V of one shape");
  if (k->shape[0] == 0) return contract("attention.varlen requires non-zero T, H, and D dimensions");
  if (k->shape[0] > (uint64_t)kMaxRows) return contract("attention.varlen shape exceeds i32 ABI");
  if (k->shape[2] != (uint64_t)c.p.dim) return contract("attention.varlen requires Q, K, and V of one head dimension");
  if ((rc = heads_match(op, k->shape[1], &c))) return rc;
  if (!cu_seqlens_k && k->shape[0] != q->shape[0])
    return contract("attention.varlen requires cu_seqlens_k when Q and K have different row counts");
  const tb_tensor* cu_k = cu_seqlens_k ? cu_seqlens_k : cu_seqlens_q;
  if (!is_index(cu_seqlens_q, 1) || !is_index(cu_k, 1) || cu_seqlens_q->shape[0] < 2 ||
      cu_seqlens_q->shape[0] > kMaxBatch + 1 || cu_k->shape[0] != cu_seqlens_q->shape[0])
    return contract("attention.varlen requires contiguous I32 cu_seqlens of one length, batch + 1");
  if (!s) return set_error(TB_ERR_INVALID, "contract", "null session");
  Stream* st = nullptr;
  Buffer *bq = nullptr, *bk = nullptr, *bv = nullptr, *bo = nullptr, *bcq = nullptr, *bck = nullptr;
  if ((rc = check_stream(s, stream, &st)) || (rc = strided_buffer(s, q, "attention.varlen Q", &bq)) ||
      (rc = strided_buffer(s, k, "attention.varlen K", &bk)) || (rc = strided_buffer(s, v, "attention.varlen V", &bv)) ||
      (rc = strided_buffer(s, output, "attention.varlen output", &bo)) ||
      (rc = strided_buffer(s, cu_seqlens_q, "attention.varlen cu_seqlens_q", &bcq)) ||
      (rc = strided_buffer(s, cu_k, "attention.varlen cu_seqlens_k", &bck)))
    return rc;
  c.p.q = bq->ptr;
  c.p.o = bo->ptr;
  c.p.k = bk->ptr;
  c.p.v = bv->ptr;
  c.p.cu_q = bcq->ptr;
  c.p.cu_k = bck->ptr;
  c.p.k_tok = step_of(k, 0);
  c.p.k_head = step_of(k, 1);
  c.p.v_tok = step_of(v, 0);
  c.p.v_head = step_of(v, 1);
  c.p.tk = (int32_t)k->shape[0];
  c.p.batch = (int32_t)cu_seqlens_q->shape[0] - 1;
  if ((rc = run_attention(s, st, op, &c, a))) return rc;
  return record_event(s, st, nullptr, out);
} catch (const std::exception& e) {
  return tb::caught(e);
}

extern "C" tb_status tb_op_attention_paged(tb_session* session, tb_stream* stream, const tb_tensor* q,
                                           const tb_tensor* k_cache, const tb_tensor* v_cache,
                                           const tb_tensor* block_table, const tb_tensor* seq_lens,
                                           const tb_tensor* cu_seqlens_q, const tb_tensor* output,
                                           const tb_attr* attrs, uint32_t num_attrs, tb_event** out) try {
  static const char* const op = "attention.paged";
  Session* s = reinterpret_cast<Session*>(session);
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !cu_seqlens_q || !output)
    return contract("attention.paged requires Q, K cache, V cache, block_table, seq_lens and cu_seqlens_q");
  AttnAttrs a;
  AttnCall c;
  tb_status rc;
  if ((rc = parse_attrs(attrs, num_attrs, op, true, &a)) || (rc = query_side(op, q, output, &c))) return rc;
  if (k_cache->dtype != q->dtype || v_cache->dtype != q->dtype)
    return contract("attention.paged requires Q, K, V, and output of one dtype");
  if (k_cache->rank != 4 || v_cache->rank != 4)
    return contract("attention.paged requires rank-4 [pages, page, H, D] K and V caches");
  for (int i = 0; i < 4; ++i)
    if (k_cache->shape[i] != v_cache->shape[i]) return contract("attention.paged requires K and V caches of one shape");
  const uint64_t pages = k_cache->shape[0], page = k_cache->shape[1];
  if (pages == 0 || page == 0) return contract("attention.paged requires non-zero cache dimensions");
  if (pages > 0x7fffffffull || page > 0x7fffffffull) return contract("attention.paged shape exceeds i32 ABI");
  if (k_cache->shape[3] != (uint64_t)c.p.dim)
    return contract("attention.paged requires Q, K, and V of one head dimension");
  if ((rc = heads_match(op, k_cache->shape[2], &c))) return rc;
  const uint64_t batch = seq_lens->rank == 1 ? seq_lens->shape[0] : 0;
  if (!is_index(seq_lens, 1) || !is_index(cu_seqlens_q, 1) || batch == 0 || batch > kMaxBatch ||
      cu_seqlens_q->shape[0] != batch + 1)
    return contract("attention.paged requires contiguous I32 seq_lens [batch] and cu_seqlens_q [batch + 1]");
  if (!is_index(block_table, 2) || block_table->shape[0] != batch || block_table->shape[1] == 0 ||
      block_table->shape[1] > 0x7fffffffull)
    return contract("attention.paged requires an I32 block_table [batch, pages per request] with contiguous rows");
  if (!s) return set_error(TB_ERR_INVALID, "contract", "null session");
  Stream* st = nullptr;
  Buffer *bq = nullptr, *bk = nullptr, *bv = nullptr, *bo = nullptr, *bt = nullptr, *bl = nullptr, *bcq = nullptr;
  if ((rc = check_stream(s, stream, &st)) || (rc = strided_buffer(s, q, "attention.paged Q", &bq)) ||
      (rc = strided_buffer(s, k_cache, "attention.paged K cache", &bk)) ||
      (rc = strided_buffer(s, v_cache, "attention.paged V cache", &bv)) ||
      (rc = strided_buffer(s, output, "attention.paged output", &bo)) ||
      (rc = strided_buffer(s, block_table, "attention.paged block_table", &bt)) ||
      (rc = strided_buffer(s, seq_lens, "attention.paged seq_lens", &bl)) ||
      (rc = strided_buffer(s, cu_seqlens_q, "attention.paged cu_seqlens_q", &bcq)))
    return rc;
  c.p.q = bq->ptr;
  c.p.o = bo->ptr;
  c.p.k = bk->ptr;
  c.p.v = bv->ptr;
  c.p.table = bt->ptr;
  c.p.lens = bl->ptr;
  c.p.cu_q = bcq->ptr;
  c.p.k_page = step_of(k_cache, 0);
  c.p.k_tok = step_of(k_cache, 1);
  c.p.k_head = step_of(k_cache, 2);
  c.p.v_page = step_of(v_cache, 0);
  c.p.v_tok = step_of(v_cache, 1);
  c.p.v_head = step_of(v_cache, 2);
  c.p.table_row = step_of(block_table, 0);
  c.p.batch = (int32_t)batch;
  c.p.page = (int32_t)page;
  c.p.pages = (int32_t)pages;
  c.p.width = (int32_t)block_table->shape[1];
  if ((rc = run_attention(s, st, op, &c, a))) return rc;
  return record_event(s, st, nullptr, out);
} catch (const std::exception& e) {
  return tb::caught(e);
}
