// vpq_kv.cuh -- what the kernels of the attention block share: the paged cache's view on the device,
// its argument checks, and the report of an index outside of its table.
#pragma once

#include "vpq_common.cuh"

namespace vpq {

// What an index report names (vpq_device_status, detail 0x40000 | bits).
enum : uint32_t { kBadPage = 1, kBadSlot = 2, kBadPosition = 4, kBadLength = 8 };

constexpr int kKvGroup = 64;  // values that share a scale and a bias of an 8-bit cache

// A vpq_kv_cache with its strides filled in.
struct KvView {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t num_pages;
  int64_t page_bytes, spage_bytes;                  // k and v; scale pairs
  uint32_t head_bytes, token_bytes, shead_bytes, stoken_bytes;
  int page_size, kv_heads;
  int page_shift;  // log2 of page_size, or -1
};

// Checks a cache descriptor and fills `view`; kv_cache.cu.
int kv_check(const char* who, const vpq_kv_cache* c, KvView* view);
// The current device's word that the kernels report indices in; qmm.cu, beside the word of vpq_device_status.
int index_status_word(uint32_t** word);

}  // namespace vpq
