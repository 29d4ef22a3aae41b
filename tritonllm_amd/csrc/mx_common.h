// What the products with MXFP4 weights share: the operands, and which expert's rows a workgroup takes.
//
// An MXFP4 row of K values is K / 32 blocks of 16 bytes (32 e2m1 codes, the low nibble first) and as many e8m0 bytes, each the
// block's power of two, biased by 127; 255 there makes the block NaN. That is how a checkpoint stores the experts
// ([experts, N, K / 32, 16] and [experts, N, K / 32]) and how the kernels read it: nothing is laid out anew.
#pragma once
#include <utility>

#include "common.h"

namespace tllm {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;
typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

// y = x . W^T + b | SwiGLU of it, for rows by expert | a row per pair in fp32, for the weighted sum over a token's experts
enum : int { kMxLinear = 0, kMxSwiglu = 1, kMxPairs = 2 };

struct MxArgs {
  const void* x;                    // rows of bf16, or of MXFP4 blocks
  const unsigned char* x_scales;    // (MXFP4 rows alone)
  int64_t x_pitch;                  // bytes from row to row
  const unsigned char* w;           // blocks
  const unsigned char* w_scales;
  const bf16* bias;                 // [experts, N] or NULL
  void* out;                        // bf16; fp32 for kMxPairs
  int64_t out_stride;               // elements from row to row
  const int* order;                 // pairs (token * top + choice) by expert, or NULL: one weight, rows as they are
  const int* offsets;               // [experts + 1] places in `order`
  int64_t rows;                     // rows, or pairs
  int64_t tokens;
  int experts, top;
  int n, k;                         // weight rows (per expert) and values in each
  float alpha, limit;               // SwiGLU; limit is infinity for none
};

// Items are runs of up to ROWS rows of one expert, in the order of the experts; a launch has as many as there can be
// (mx_items), and the workgroups of those that are not there find no rows. All 64 lanes ask together: each loads one
// expert's two offsets, a scan over the lanes counts the items before it, and a ballot finds the expert whose item this is.
// Offsets are held to [0, rows], so that no content of theirs leads out of the tensors.
struct MxItem {
  int expert, first, rows;          // rows 0: none
};
static inline int64_t mx_items(int64_t rows, int experts, int per_item) {
  return (rows < experts ? rows : experts) + rows / per_item;
}
__device__ __forceinline__ MxItem mx_find_item(const int* offsets, int experts, int rows, int per_item, int item) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    int lo = offsets[e < experts ? e : experts], hi = offsets[e < experts ? e + 1 : experts];
    lo = min(max(lo, 0), rows);
    hi = min(max(hi, lo), rows);
    const int n = hi - lo;
    int mine, upto;                                        // items of this lane's expert, and of all up to it
    if (__ballot(n > per_item) == 0) {                     // at most one each: a count of bits
      const unsigned long long some = __ballot(n > 0);
      mine = n > 0;
      upto = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(some >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(some), mine));
    } else {
      upto = mine = (n + per_item - 1) / per_item;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
      }
    }
    const unsigned long long has = __ballot(before + upto > item);
    if (has) {
      const int l = __builtin_ctzll(has);
      const int at = item - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
      const int first = __builtin_amdgcn_readlane(lo, l) + at * per_item, end = __builtin_amdgcn_readlane(hi, l);
      return {e0 + l, first, min(per_item, end - first)};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, 0, 0};
}

// The same for a grid in the order (expert, tile of weight rows, item): one of `tiles` x items, dealt so that the tiles of an XCD
// (workgroups go to the eight of them in turn) are neighbours -- those of one run of weight rows, then the next run's.
struct MxTile {
  int expert, first, rows, tile_n;  // rows 0: none
};
__device__ __forceinline__ MxTile mx_find_tile(const int* offsets, int experts, int rows, int per_item, int tiles_n, int block) {
  const int lane = threadIdx.x & 63;
  auto counted = [&](int e, int* lo, int* hi) {
    *lo = offsets[e < experts ? e : experts];
    *hi = offsets[e < experts ? e + 1 : experts];
    *lo = min(max(*lo, 0), rows);
    *hi = min(max(*hi, *lo), rows);
    return (*hi - *lo + per_item - 1) / per_item;
  };
  int lo, hi, total = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) total += counted(e0 + lane, &lo, &hi);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  const int all = total * tiles_n, per = (all + 7) / 8, at = block >> 3, t = (block & 7) * per + at;
  if (at >= per || t >= all) return {0, 0, 0, 0};
  int before = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int mine = counted(e0 + lane, &lo, &hi);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const unsigned long long has = __ballot((before + upto) * tiles_n > t);
    if (has) {
      const int l = __builtin_ctzll(has), items = __builtin_amdgcn_readlane(mine, l);
      const int local = t - (before + __builtin_amdgcn_readlane(upto, l) - items) * tiles_n;
      const int tile_n = local / items, first = __builtin_amdgcn_readlane(lo, l) + (local - tile_n * items) * per_item;
      return {e0 + l, first, min(per_item, __builtin_amdgcn_readlane(hi, l) - first), tile_n};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, 0, 0, 0};
}

// Read through the scalar cache, at places that all lanes share.
typedef const __attribute__((address_space(4))) int* ScalarInts;
__device__ __forceinline__ ScalarInts mx_scalar(const int* p) { return (ScalarInts)(uintptr_t)p; }

// A token's row: the pair at place s of the order, held to the pairs there are.
__device__ __forceinline__ unsigned mx_pair(const MxArgs& a, int s) {
  const unsigned p = static_cast<unsigned>(a.order[s]), last = static_cast<unsigned>(a.rows - 1);
  return p < last ? p : last;
}

// Clamped SwiGLU of a gate and a linear value: g sigmoid(alpha g) (l + 1).
__device__ __forceinline__ float mx_swiglu(float g, float l, float alpha, float limit) {
  // (comparisons and not fminf: a NaN stays one)
  g = g > limit ? limit : g;
  l = l > limit ? limit : l < -limit ? -limit : l;
  return g / (1.0f + __expf(-alpha * g)) * (l + 1.0f);
}

// A dword of eight codes times 2^(s - 127) as bf16, exactly (values of 2^128 and more, scale bytes 253 and 254, are infinite);
// `scale` is the byte in an fp32's exponent, 0 there means 2^-127 and 255 NaN.
__device__ __forceinline__ bf16x8 mx_bf16x8(unsigned codes, float scale) {
  u32x4 o;
  o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return __builtin_bit_cast(bf16x8, o);
}

// f(0), f(1), ... f(N - 1) with the numbers as types
template <class F, int... I>
__device__ __forceinline__ void mx_each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void mx_each(F&& f) {
  mx_each(f, std::make_integer_sequence<int, N>{});
}

// A buffer of `bytes` bytes from p on; loads behind its end give zeros and fetch nothing. MX_NONE is behind every end.
constexpr unsigned MX_NONE = 0xfffffff0u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x27000);
}
__device__ __forceinline__ u32x4 mx_load16(__amdgpu_buffer_rsrc_t b, unsigned at) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
}
// The same buffer as four words, for the load that goes straight to LDS: 16 bytes a lane, from `at` + `more` in the buffer to
// `lds` + 16 x lane. The compiler does not know of it: its arrival is waited for by count.
__device__ __forceinline__ u32x4 mx_buffer_words(const void* p, unsigned bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(p);
  u32x4 w;
  w[0] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(b));
  w[1] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(b >> 32) & 0xffffu);
  w[2] = __builtin_amdgcn_readfirstlane(bytes);
  w[3] = 0x27000;
  return w;
}
__device__ __forceinline__ void mx_load_lds(u32x4 buffer, unsigned at, unsigned more, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(at), "s"(buffer), "s"(more) : "memory", "m0");
}
__device__ __forceinline__ unsigned mx_load1(__amdgpu_buffer_rsrc_t b, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b8(b, at, 0, 0); }

// ---- what the tiles share
// Which quarter of a slice's K the lanes of group g = lane / 16 have, in both operands. A 16-byte LDS read is served in four parts, of
// lanes 0 - 3, 12 - 15, 20 - 27; 4 - 11, 16 - 19, 28 - 31; and the same of the upper half (measured). With 128-byte rows whose sixteens
// are XORed with row / 2 % 8 the sixteen lanes of a part are in different banks if the quarters of groups 0 and 1, and of 2
// and 3, are each other's complements.
__device__ __forceinline__ int mx_quarter(int g) { return 0x2130 >> 4 * g & 3; }
// The scale bytes of a tile's rows in LDS, for the whole of K: as they lie in memory, one row behind the other, from the sixteen bytes
// on in which they begin; rows of whole sixteens have sixteen more between them, or sixteen rows' bytes would lie in few banks.
// Byte b of row r is at mx_scale_shift + r mx_scale_pitch + b.
static __host__ __device__ __forceinline__ int mx_scale_pitch(int blocks) { return blocks % 16 ? blocks : blocks + 16; }
static __host__ __device__ __forceinline__ int mx_scale_lds(int rows, int blocks) { return (rows * mx_scale_pitch(blocks) + 47) / 16 * 16; }
__device__ __forceinline__ int mx_scale_shift(const unsigned char* from) { return static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15); }
// The fetch, four loads of a thread on their way together.
template <int THREADS>
__device__ __forceinline__ void mx_fetch_scales(unsigned char* to, const unsigned char* from, int rows, int blocks, int tid) {
  constexpr int FLIGHT = 4;
  const int shift = mx_scale_shift(from), bytes = shift + rows * blocks, units = (bytes + 15) / 16;
  // (to whole words: a word that the end cuts would come as zeros; its other bytes share the last one's sixteen)
  const auto buf = mx_buffer(from - shift, (bytes + 3) & ~3);
  for (int first = 0; first < units; first += THREADS * FLIGHT) {
    u32x4 v[FLIGHT];
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      const int i = first + tid + j * THREADS;
      v[j] = mx_load16(buf, i < units ? 16 * i : MX_NONE);
    }
#pragma unroll
    for (int j = 0; j < FLIGHT; ++j) {
      const int i = first + tid + j * THREADS;
      if (i < units) *reinterpret_cast<u32x4*>(to + 16 * (blocks % 16 ? i : i + i / (blocks / 16))) = v[j];
    }
  }
}

// Whether four neighbours of the bias and of a row of the result are whole accesses
__device__ __forceinline__ bool mx_whole_fours(const MxArgs& a) {
  return a.n % 4 == 0 && a.out_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && reinterpret_cast<uintptr_t>(a.bias) % 8 == 0;
}
__device__ __forceinline__ bf16x4 mx_bias4(const MxArgs& a, bool four, int64_t wrow, int n, int nn) {
  bf16x4 b = {};
  if (a.bias == nullptr) return b;
  if (four) return *reinterpret_cast<const bf16x4*>(a.bias + wrow + (n < nn ? n : 0));
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = a.bias[wrow + (n + i < nn ? n + i : nn - 1)];
  return b;
}
// Sums of weight rows n0 + n .. + 3 (nn of n0's tile are there) for a row of the result: bias, SwiGLU, one rounding
template <int MODE>
__device__ __forceinline__ void mx_store4(const MxArgs& a, bool four, int64_t row, int n0, int n, int nn, f32x4 sum, bf16x4 bias) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = sum[i] + static_cast<float>(bias[i]);
  if constexpr (MODE == kMxSwiglu) {
    bf16* const to = static_cast<bf16*>(a.out) + row * a.out_stride + (n0 + n) / 2;
    const bf16x2 o = {static_cast<bf16>(mx_swiglu(v[0], v[1], a.alpha, a.limit)), static_cast<bf16>(mx_swiglu(v[2], v[3], a.alpha, a.limit))};
    if (four) {
      *reinterpret_cast<bf16x2*>(to) = o;
    } else {
      to[0] = o[0];
      if (n + 2 < nn) to[1] = o[1];
    }
  } else if constexpr (MODE == kMxPairs) {
    float* const to = static_cast<float*>(a.out) + row * a.out_stride + n0 + n;
    if (four) {
      *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < nn) to[i] = v[i];
    }
  } else {
    bf16* const to = static_cast<bf16*>(a.out) + row * a.out_stride + n0 + n;
    const bf16x4 o = {static_cast<bf16>(v[0]), static_cast<bf16>(v[1]), static_cast<bf16>(v[2]), static_cast<bf16>(v[3])};
    if (four) {
      *reinterpret_cast<bf16x4*>(to) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < nn) to[i] = o[i];
    }
  }
}

int mx_stream(const MxArgs& a, int mode, bool a4, hipStream_t st);
int mx_tiles4(const MxArgs& a, hipStream_t st);
bool mx_tiles_take(const MxArgs& a);
bool mx_tiles4_take(const MxArgs& a);
int mx_tiles(const MxArgs& a, int mode, hipStream_t st);

}  // namespace tllm
