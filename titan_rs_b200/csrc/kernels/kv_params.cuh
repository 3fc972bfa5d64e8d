// What the cache-append kernels are told about one call (op_kv_cache.cpp fills it).
#pragma once

#include <stdint.h>

namespace tb {

struct AppendParams {
  uint64_t k, v, k_cache, v_cache, slots;
  long long k_tok, k_head, v_tok, v_head;  // strides in bytes
  long long kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head;
  long long limit;                         // slots of the cache
  int tokens, heads, chunks, page;         // chunks of a row, of the kernel's chunk size
};

}  // namespace tb
