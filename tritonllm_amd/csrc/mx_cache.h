// A KV cache in MXFP4 as kernels take it, and the integers that a caller keeps on the device, one for a batch or one per row.
#pragma once
#include "mx_common.h"

namespace tllm {

struct MxCache {
  const unsigned char* blocks[2];         // keys, values: 16 bytes per 32 values
  const unsigned char* scales[2];
  int64_t bs, hs, ts;                     // bytes from row to row, head to head, slot to slot of the blocks
  int64_t sbs, shs, sts;                  // ... of the scales
  int n_slots;
};

// Host: what a caller describes, checked.
int mx_cache_of(const TllmMxCache* c, const char* what, MxCache* out);

__device__ __forceinline__ int64_t mx_row_int(const void* p, int is_i64, int64_t i) {
  return is_i64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int*>(p)[i]);
}

}  // namespace tllm
