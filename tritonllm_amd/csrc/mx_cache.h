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
// The same without a branch, whose join would wait for the value (the write waits for it anyway: 21.0 us with, 21.9 without for 8 x 4096 tokens).
__device__ __forceinline__ int64_t mx_row_int_ahead(const void* p, int is_i64, int64_t i) {
  const int64_t two = is_i64 != 0;
  const int* const w = static_cast<const int*>(p) + (i << two);
  const int lo = w[0], hi = w[two];
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<unsigned>(two ? hi : lo >> 31)) << 32 | static_cast<unsigned>(lo));
}

// n / d for n < 2^31 as a product: with 2^(l-1) < d <= 2^l and mul = 2^(31+l) / d + e, 0 < e <= 1, the quotient 2 n mul / 2^(32+l) is n / d and less
// than 2^-l <= 1 / d more.
struct MxDiv {
  unsigned mul, shift;
  __device__ __forceinline__ int operator()(unsigned n) const { return static_cast<int>(__umulhi(2 * n, mul) >> shift); }
};
inline MxDiv mx_div(unsigned d) {
  unsigned l = 0;
  while ((1ull << l) < d) ++l;
  return MxDiv{static_cast<unsigned>((1ull << (31 + l)) / d + 1), l};
}

}  // namespace tllm
