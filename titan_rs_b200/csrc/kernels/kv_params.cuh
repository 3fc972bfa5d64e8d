// What the cache kernels are told about one call (op_kv_cache.cpp fills it).
#pragma once

#include <stdint.h>

namespace tb {

constexpr int kAppendThreads = 256;

struct AppendParams {
  uint64_t k, v, k_cache, v_cache, slots;
  long long k_tok, k_head, v_tok, v_head;  // strides in bytes
  long long kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head;
  long long limit;                         // slots of the cache
  int tokens, heads, chunks, page;         // chunks of a row, of the kernel's chunk size
};

struct PlanParams {
  uint64_t ctx, add, free_pages;               // int32 [batch], [batch], [n_free]
  uint64_t table, lens, cu, slots, status;     // int32 [batch, width], [batch], [batch + 1], [tokens], [2]
  long long table_row;
  int batch, n_free, width, tokens, page;
};

}  // namespace tb
