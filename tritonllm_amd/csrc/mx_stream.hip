// Products with an MXFP4 weight for few rows: the weight streams past rows that come from the L2.
//
//   D[n, r] = sum_k W[n, k] X[r, k]        W MXFP4 [N, K], X bf16 or MXFP4
//
// What bounds it is the weight's arrival, N K 17 / 32 bytes of every expert that has rows, and with one token the chain of latencies
// before and after. A workgroup of NW wavefronts owns 16 NT weight rows and up to 16 activation rows; the wavefronts deal the
// K steps of 128 between them, U neighbouring ones each (sums meet in LDS, added in a fixed order), and ask for all U at once: with K
// up to 128 NW U everything is on its way together, behind two reads (the plan's offsets, and the rows' numbers where rows are
// gathered). The loads are buffer loads: what lies behind the tensors' end, rows that are not there and steps behind the last one read
// as zeros without a fetch and without a branch.
//
// In a step lane l has block l / 16 of weight row l % 16: one 16-byte load is a whole MXFP4 block. For bf16 activations the four lanes of a
// row exchange their words (two swaps of half and quarter wavefronts each), after which word i of all of them is of block i:
// the i-th of the step's four v_mfma_f32_16x16x32_bf16 then takes k = 32 i + 8 (l / 16) .. + 7, and a load of activations 64
// neighbouring bytes of a row (without the exchange its sixteens were 64 bytes apart, and every line was asked for four times: 33 tokens
// 78 us). The codes become bf16 on the way, exactly, once per step for all rows; the scale bytes lie in LDS, fetched sixteen at a
// time (byte by byte 10 % of the time). With MXFP4 activations the step is one v_mfma_scale_f32_16x16x128_f8f6f4, which takes
// both blocks and scales as they are. The weight's loads carry no nontemporal hint: a step takes half a line, and with the hint
// the other half's request fetched the line again (one token 14.4 us with, 10.1 without).
#include "mx_common.h"

namespace tllm {

// b of the lower half (of the first and third quarter) of the wavefront for a of the upper half (of the second and fourth)
__device__ __forceinline__ void lanes_swap32(unsigned& a, unsigned& b) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, __builtin_amdgcn_permlane32_swap(a, b, false, false));
  a = static_cast<unsigned>(u);
  b = static_cast<unsigned>(u >> 32);
}
__device__ __forceinline__ void lanes_swap16(unsigned& a, unsigned& b) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, __builtin_amdgcn_permlane16_swap(a, b, false, false));
  a = static_cast<unsigned>(u);
  b = static_cast<unsigned>(u >> 32);
}

// What a walk over K reads: the weight rows' buffer, the activation rows' buffer and each lane's row in it, and both scales.
struct MxWalk {
  __amdgpu_buffer_rsrc_t w, x, x_scales;
  const unsigned char* scale_bytes;                        // LDS: this lane's weight row's
  unsigned row_at, row_scales_at;                          // of this lane's activation row; MX_NONE: there is none
  int blocks, pitch;                                       // blocks of a row; scale bytes from row to row
};

// Up to RP bf16 rows, 4, 8 or 16. The columns of a product are sixteen: with up to 8 rows a load of activations takes two of the
// step's four pieces of K for all of them, with up to 4 all four (lane (m, g): row m % RP, piece p + m / RP), and the products with
// piece p's weights then are good in the columns of that piece and nonsense in the others, so each piece has its own sums, of which
// only those columns are kept. `ready` is called when the first loads are on their way.
template <int NT, int RP, int NW, int U, class F>
__device__ __forceinline__ void mx_walk(const MxWalk& m, int wave, int lane, float* sums, int sums_pitch, F&& ready) {
  constexpr int C = 16 / RP, X = 4 / C;                    // pieces that share a load; loads of a step
  const int m16 = lane & 15, g = lane >> 4, steps = (m.blocks + 3) / 4, mine = m16 / RP;
  u32x4 wq[U][NT], xq[U][X];
  f32x4 acc[NT][C];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < steps; base += NW * U) {
    const int step0 = base + wave * U;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s) + g;
#pragma unroll
      for (int t = 0; t < NT; ++t) wq[s][t] = mx_load16(m.w, b < m.blocks ? ((16 * t + m16) * m.blocks + b) * 16 : MX_NONE);
    }
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int j = 0; j < X; ++j) {
        const int b = 4 * (step0 + s) + C * j + mine;
        xq[s][j] = mx_load16(m.x, b < m.blocks && m.row_at != MX_NONE ? m.row_at + 64 * b + 16 * g : MX_NONE);
      }
    if (base == 0) ready();
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        unsigned four = 0;                                  // (of blocks that are not there: 0, not another row's)
        if (b < m.blocks) {
          __builtin_memcpy(&four, m.scale_bytes + 16 * t * m.pitch + b, 4);
          if (b + 4 > m.blocks) four &= (1u << 8 * (m.blocks - b)) - 1;
        }
        unsigned w0 = wq[s][t][0], w1 = wq[s][t][1], w2 = wq[s][t][2], w3 = wq[s][t][3];
        lanes_swap32(w0, w2);
        lanes_swap32(w1, w3);
        lanes_swap16(w0, w1);
        lanes_swap16(w2, w3);
        const unsigned words[4] = {w0, w1, w2, w3};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned e = i == 0 ? four << 23 : four >> (8 * i) << 23;
          const bf16x8 wv = mx_bf16x8(words[i], __builtin_bit_cast(float, e & 0x7f800000u));
          acc[t][i % C] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8, xq[s][i / C]), acc[t][i % C], 0, 0, 0);
        }
      }
    }
  }
  // lane (m16, g) holds weight rows 4 g .. + 3 of its column
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    f32x4 v = acc[t][0];
#pragma unroll
    for (int c = 1; c < C; ++c)
      if (mine == c) v = acc[t][c];
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[m16 * sums_pitch + 16 * t + 4 * g + i] = v[i];
  }
}

// The same for up to 16 rows of MXFP4.
template <int NT, int NW, int U, class F>
__device__ __forceinline__ void mx_walk4(const MxWalk& m, int wave, int lane, float* sums, int sums_pitch, F&& ready) {
  const int m16 = lane & 15, g = lane >> 4, steps = (m.blocks + 3) / 4;
  u32x4 wq[U][NT], xq[U];
  unsigned xs[U];
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < steps; base += NW * U) {
    const int step0 = base + wave * U;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s) + g;
#pragma unroll
      for (int t = 0; t < NT; ++t) wq[s][t] = mx_load16(m.w, b < m.blocks ? ((16 * t + m16) * m.blocks + b) * 16 : MX_NONE);
      const bool ok = b < m.blocks && m.row_at != MX_NONE;
      xq[s] = mx_load16(m.x, ok ? m.row_at + 16 * b : MX_NONE);
      xs[s] = mx_load1(m.x_scales, ok ? m.row_scales_at + b : MX_NONE);
    }
    if (base == 0) ready();
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s) + g;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const unsigned scale = b < m.blocks ? m.scale_bytes[16 * t * m.pitch + b] : 0u;
        i32x8 wv = {}, xv = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          wv[i] = wq[s][t][i];
          xv[i] = xq[s][i];
        }
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[t], 4, 4, 0, scale, 0, xs[s]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[m16 * sums_pitch + 16 * t + 4 * g + i] = acc[t][i];
}

template <int NT, bool A4, int MODE, int NW, int U4, int U8, int U16>
__global__ __launch_bounds__(NW * 64) void mx_stream_kernel(MxArgs a, int tiles_n) {
  constexpr int BN = 16 * NT, BR = 16, THREADS = NW * 64, PITCH = BN + 1;
  __shared__ float sums[NW][BR][PITCH];
  extern __shared__ __align__(16) unsigned char scale_bytes[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15;
  const int item = blockIdx.x / tiles_n, n0 = (blockIdx.x - item * tiles_n) * BN;
  MxItem it;
  if (a.order == nullptr) {
    const int64_t first = static_cast<int64_t>(item) * BR, left = a.rows - first;
    it = {0, static_cast<int>(first), static_cast<int>(left < BR ? left : BR)};
  } else {
    it = mx_find_item(a.offsets, a.experts, static_cast<int>(a.rows), BR, item);
  }
  if (it.rows <= 0) return;
  const int columns = A4 || it.rows > 8 ? 16 : it.rows > 4 ? 8 : 4;         // rows that the walk takes

  const int blocks = a.k / 32;
  const int nn = a.n - n0 < BN ? a.n - n0 : BN;             // weight rows of this tile
  const int64_t wrow = static_cast<int64_t>(it.expert) * a.n + n0;
  MxScaleFetch<THREADS, 1> fetch(a.w_scales + wrow * blocks, nn, blocks, tid);
  fetch.load(0);

  // the rows' numbers, if they are gathered or scattered, and this thread's bias go out ahead of the weight
  constexpr bool gather = MODE == kMxSwiglu;
  const int r16 = m16 & (columns - 1);
  const bool there = r16 < it.rows;
  unsigned row = r16;
  if (gather) row = a.tokens > 1 ? mx_pair(a, it.first + (there ? r16 : 0)) / static_cast<unsigned>(a.top) : 0;
  constexpr int OUTS = BR * BN / (MODE == kMxSwiglu ? 2 : 1), PER = (OUTS + THREADS - 1) / THREADS;   // results of a thread
  unsigned pair[PER] = {};
  float bias[PER][2] = {};
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = tid + p * THREADS, r = MODE == kMxSwiglu ? i / (BN / 2) : i / BN, n = MODE == kMxSwiglu ? i % (BN / 2) * 2 : i % BN;
    if (MODE == kMxPairs) pair[p] = mx_pair(a, it.first + min(r, it.rows - 1));
    if (a.bias) {
      bias[p][0] = static_cast<float>(a.bias[wrow + min(n, nn - 1)]);
      if (MODE == kMxSwiglu) bias[p][1] = static_cast<float>(a.bias[wrow + min(n + 1, nn - 1)]);
    }
  }

  // the rows' bytes: of a token anywhere in x, or counted from the item's first row
  MxWalk m;
  const int row_bytes = A4 ? blocks * 16 : a.k * 2;
  const unsigned char* const xb = static_cast<const unsigned char*>(a.x) + (gather ? 0 : it.first * a.x_pitch);
  m.w = mx_buffer(a.w + wrow * blocks * 16, nn * blocks * 16);
  m.x = mx_buffer(xb, static_cast<unsigned>(((gather ? a.tokens : it.rows) - 1) * a.x_pitch + row_bytes));
  m.x_scales = A4 ? mx_buffer(a.x_scales + static_cast<int64_t>(it.first) * blocks, it.rows * blocks) : m.x;
  m.blocks = blocks;
  m.pitch = mx_scale_pitch(blocks);
  m.scale_bytes = scale_bytes + mx_scale_shift(a.w_scales + wrow * blocks) + m16 * m.pitch;
  m.row_at = there ? static_cast<unsigned>(row * a.x_pitch) : MX_NONE;
  m.row_scales_at = row * blocks;
  auto ready = [&] {
    fetch.write(scale_bytes, 0);
    fetch.rest(scale_bytes, THREADS);
    __syncthreads();
  };
  float* const mine = sums[wave][0];
  if constexpr (A4) mx_walk4<NT, NW, U4>(m, wave, lane, mine, PITCH, ready);
  else if (columns == 4) mx_walk<NT, 4, NW, U4>(m, wave, lane, mine, PITCH, ready);
  else if (columns == 8) mx_walk<NT, 8, NW, U8>(m, wave, lane, mine, PITCH, ready);
  else mx_walk<NT, 16, NW, U16>(m, wave, lane, mine, PITCH, ready);
  __syncthreads();

  auto total = [&](int r, int n) {
    float v = 0.f;
    for (int c = r; c < 16; c += columns)
#pragma unroll
      for (int w = 0; w < NW; ++w) v += sums[w][c][n];
    return v;
  };
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = tid + p * THREADS, r = MODE == kMxSwiglu ? i / (BN / 2) : i / BN, n = MODE == kMxSwiglu ? i % (BN / 2) * 2 : i % BN;
    if (i >= OUTS || r >= it.rows || n >= nn) continue;
    const int64_t at = static_cast<int64_t>(it.first) + r;
    if constexpr (MODE == kMxSwiglu)
      static_cast<bf16*>(a.out)[at * a.out_stride + (n0 + n) / 2] =
          static_cast<bf16>(mx_swiglu(total(r, n) + bias[p][0], total(r, n + 1) + bias[p][1], a.alpha, a.limit));
    else if constexpr (MODE == kMxPairs)
      static_cast<float*>(a.out)[pair[p] * a.out_stride + n0 + n] = total(r, n) + bias[p][0];
    else
      static_cast<bf16*>(a.out)[at * a.out_stride + n0 + n] = static_cast<bf16>(total(r, n) + bias[p][0]);
  }
}

template <int NT, bool A4, int MODE, int NW, int U4, int U8, int U16>
static int launch(const MxArgs& a, hipStream_t st) {
  const int64_t tiles = (a.n + 16 * NT - 1) / (16 * NT);
  const int64_t items = a.order ? mx_items(a.rows, a.experts, 16) : (a.rows + 15) / 16;
  TLLM_REQUIRE(tiles * items < (1ll << 32) / (NW * 64), TLLM_E_SHAPE, "mxfp4 product: %lld rows of %d outputs are too many", (long long)a.rows, a.n);
  const int lds = mx_scale_lds(16 * NT, a.k / 32);
  if (lds > 40 * 1024) {                                   // (long rows; with the sums more than a kernel has without asking)
    static std::atomic<uint64_t> done{0};
    const void* const kernel = reinterpret_cast<const void*>(mx_stream_kernel<NT, A4, MODE, NW, U4, U8, U16>);
    TLLM_REQUIRE(raise_lds_limit(kernel, 140 * 1024, done) == hipSuccess, TLLM_E_LAUNCH, "mxfp4 product: the LDS limit could not be raised");
  }
  hipLaunchKernelGGL((mx_stream_kernel<NT, A4, MODE, NW, U4, U8, U16>), dim3((unsigned)(tiles * items)), dim3(NW * 64), lds, st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

// The workgroup. Wide ones (64 weight rows) read the activations less often and pay where items are full: 128 tokens of 32 experts
// mlp1 114 us with 32 rows, 107 with 64 (33 tokens 63.4 and 67.1), 65 rows of [5120, 2880] 14.8 and 12.3. Narrow ones, with their K
// share in one piece, where the launch would have less than one for each CU otherwise: one row of [2880, 4096] 6.9 us with 32 weight
// rows, 4.7 with 16; 64 rows of [1024, 1024] 5.8 with 64, 4.4 with 32. More steps on their way per wavefront cost wavefronts on the CU and more than
// they bring: 33 tokens 63.8 us with 2 steps, 70 with 3, 85 with 6.
template <int MODE>
static int launch_bf16(const MxArgs& a, hipStream_t st) {
  const int64_t items = a.order ? (a.rows < a.experts ? a.rows : a.experts) + a.rows / 32 : (a.rows + 15) / 16;
  const bool full = a.rows > 12ll * a.experts;
  if (full && (a.n + 63) / 64 * items >= 256 && a.k <= 16384) return launch<4, false, MODE, 4, 2, 2, 1>(a, st);
  if ((a.n + 31) / 32 * items > 128 && a.k <= 32768) return launch<2, false, MODE, 4, 2, 2, 2>(a, st);
  return launch<1, false, MODE, 8, 3, 3, 2>(a, st);
}

int mx_stream(const MxArgs& a, int mode, bool a4, hipStream_t st) {
  if (mode == kMxSwiglu) return launch_bf16<kMxSwiglu>(a, st);
  if (mode == kMxPairs) return launch_bf16<kMxPairs>(a, st);
  if (!a4) return launch_bf16<kMxLinear>(a, st);
  return (a.n + 31) / 32 * ((a.rows + 15) / 16) > 128 && a.k <= 32768 ? launch<2, true, kMxLinear, 4, 4, 1, 1>(a, st) : launch<1, true, kMxLinear, 8, 3, 1, 1>(a, st);
}

}  // namespace tllm
