// Products with an MXFP4 weight for few rows: the weight streams past rows that come from the L2.
//
//   D[n, r] = sum_k W[n, k] X[r, k]        W MXFP4 [N, K], X bf16 or MXFP4
//
// What bounds it is the weight's arrival, N K 17 / 32 bytes of every expert that has rows. A workgroup of four wavefronts owns
// 16 NT weight rows and up to 16 MC activation rows; the wavefronts deal the K steps of 128 between them (sums meet in LDS,
// added in a fixed order). In a step lane l has block l / 16 of weight row l % 16: one 16-byte load is a whole MXFP4 block, and
// the four MFMAs of the step take 8 of its 32 values each, k = 32 (l / 16) + 8 i .. + 7, from both operands
// (v_mfma_f32_16x16x32_bf16; the codes become bf16 on the way, once per step for all rows, exactly). With MXFP4 activations
// the step is one v_mfma_scale_f32_16x16x128_f8f6f4, which takes both blocks and scales as they are.
// A ring of R steps in registers keeps the loads in flight. They are buffer loads: what lies behind the tensors' end, rows
// that are not there and steps behind the last one read as zeros without a fetch and without a branch.
#include "mx_common.h"

namespace tllm {

template <int NT, int MC, bool A4, int MODE, int R>
__global__ __launch_bounds__(256) void mx_stream_kernel(MxArgs a, int tiles_n) {
  constexpr int BN = 16 * NT, BR = 16 * MC;
  __shared__ float sums[4][BR][BN + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, g = lane >> 4;
  const int item = blockIdx.x / tiles_n, n0 = (blockIdx.x - item * tiles_n) * BN;
  MxItem it;
  if (a.order == nullptr) {
    const int64_t first = static_cast<int64_t>(item) * BR, left = a.rows - first;
    it = {0, static_cast<int>(first), static_cast<int>(left < BR ? left : BR)};
  } else {
    it = mx_find_item(a.offsets, a.experts, static_cast<int>(a.rows), BR, item);
  }
  if (it.rows <= 0) return;

  const int blocks = a.k / 32, steps = (blocks + 3) / 4;
  const int nn = a.n - n0 < BN ? a.n - n0 : BN;             // weight rows of this tile
  const int64_t wrow = static_cast<int64_t>(it.expert) * a.n + n0;
  const __amdgpu_buffer_rsrc_t wr = mx_buffer(a.w + wrow * blocks * 16, nn * blocks * 16), sr = mx_buffer(a.w_scales + wrow * blocks, nn * blocks);
  // the rows' bytes: of a token anywhere in x, or counted from the item's first row
  const int row_bytes = A4 ? blocks * 16 : a.k * 2;
  const bool gather = MODE == kMxSwiglu;
  const unsigned char* const xb = static_cast<const unsigned char*>(a.x) + (gather ? 0 : it.first * a.x_pitch);
  const int64_t x_span = ((gather ? a.tokens : it.rows) - 1) * a.x_pitch + row_bytes;
  const __amdgpu_buffer_rsrc_t xr = mx_buffer(xb, static_cast<unsigned>(x_span));
  const __amdgpu_buffer_rsrc_t xsr = A4 ? mx_buffer(a.x_scales + static_cast<int64_t>(it.first) * blocks, it.rows * blocks) : sr;

  unsigned xo[MC], xso[MC];
#pragma unroll
  for (int c = 0; c < MC; ++c) {
    const int r = 16 * c + m16;
    xo[c] = xso[c] = MX_NONE;
    if (r < it.rows) {
      const unsigned row = gather ? mx_pair(a, it.first + r) / static_cast<unsigned>(a.top) : r;
      xo[c] = static_cast<unsigned>(row * a.x_pitch);
      xso[c] = r * blocks;
    }
  }

  u32x4 wq[R][NT];
  unsigned ws[R][NT];
  u32x4 xq[R][MC][A4 ? 1 : 4];
  unsigned xs[R][A4 ? MC : 1];
  auto load = [&](auto slot, int step) {
    constexpr int s = decltype(slot)::value;
    const int b = 4 * step + g;
    const bool in = b < blocks;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned at = (16 * t + m16) * blocks + b;
      wq[s][t] = mx_load16_once(wr, in ? at * 16 : MX_NONE);
      ws[s][t] = mx_load1(sr, in ? at : MX_NONE);
    }
#pragma unroll
    for (int c = 0; c < MC; ++c) {
      const bool ok = in && xo[c] != MX_NONE;
      if constexpr (A4) {
        xq[s][c][0] = mx_load16(xr, ok ? xo[c] + 16 * b : MX_NONE);
        xs[s][c] = mx_load1(xsr, ok ? xso[c] + b : MX_NONE);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) xq[s][c][i] = mx_load16(xr, ok ? xo[c] + 64 * b + 16 * i : MX_NONE);
      }
    }
  };
  f32x4 acc[NT][MC];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < MC; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](auto slot) {
    constexpr int s = decltype(slot)::value;
    if constexpr (A4) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < MC; ++c) {
          i32x8 wv = {}, xv = {};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            wv[i] = wq[s][t][i];
            xv[i] = xq[s][c][0][i];
          }
          acc[t][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[t][c], 4, 4, 0, ws[s][t], 0, xs[s][c]);
        }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float scale = __builtin_bit_cast(float, ws[s][t] << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bf16x8 wv = mx_bf16x8(wq[s][t][i], scale);
#pragma unroll
          for (int c = 0; c < MC; ++c)
            acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8, xq[s][c][i]), acc[t][c], 0, 0, 0);
        }
      }
    }
  };
  mx_each<R>([&](auto s) { load(s, wave + 4 * decltype(s)::value); });
  for (int step = wave; step < steps; step += 4 * R)
    mx_each<R>([&](auto s) {
      multiply(s);
      load(s, step + 4 * (R + decltype(s)::value));
    });

  // lane (m16, g) holds weight rows 4 g .. + 3 of activation row m16
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < MC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][16 * c + m16][16 * t + 4 * g + i] = acc[t][c][i];
  __syncthreads();
  const bf16* const bias = a.bias ? a.bias + wrow : nullptr;
  auto total = [&](int r, int n) {
    return (sums[0][r][n] + sums[1][r][n]) + (sums[2][r][n] + sums[3][r][n]) + (bias ? static_cast<float>(bias[n]) : 0.f);
  };
  if constexpr (MODE == kMxSwiglu) {
    for (int i = threadIdx.x; i < BR * BN / 2; i += 256) {
      const int r = i / (BN / 2), n = i % (BN / 2) * 2;
      if (r >= it.rows || n + 1 >= nn) continue;
      static_cast<bf16*>(a.out)[(it.first + r) * a.out_stride + (n0 + n) / 2] = static_cast<bf16>(mx_swiglu(total(r, n), total(r, n + 1), a.alpha, a.limit));
    }
  } else {
    for (int i = threadIdx.x; i < BR * BN; i += 256) {
      const int r = i / BN, n = i % BN;
      if (r >= it.rows || n >= nn) continue;
      if constexpr (MODE == kMxPairs) static_cast<float*>(a.out)[mx_pair(a, it.first + r) * a.out_stride + n0 + n] = total(r, n);
      else static_cast<bf16*>(a.out)[(static_cast<int64_t>(it.first) + r) * a.out_stride + n0 + n] = static_cast<bf16>(total(r, n));
    }
  }
}

template <int NT, int MC, bool A4, int MODE, int R>
static int launch(const MxArgs& a, hipStream_t st) {
  const int64_t tiles = (a.n + 16 * NT - 1) / (16 * NT), per = 16 * MC;
  const int64_t items = a.order ? mx_items(a.rows, a.experts, 16 * MC) : (a.rows + per - 1) / per;
  TLLM_REQUIRE(tiles * items < (1ll << 31), TLLM_E_SHAPE, "mxfp4 product: %lld rows of %d outputs are too many", (long long)a.rows, a.n);
  hipLaunchKernelGGL((mx_stream_kernel<NT, MC, A4, MODE, R>), dim3((unsigned)(tiles * items)), dim3(256), 0, st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

int mx_stream(const MxArgs& a, int mode, bool a4, hipStream_t st) {
  if (mode == kMxSwiglu) return launch<2, 1, false, kMxSwiglu, 3>(a, st);
  if (mode == kMxPairs) return launch<2, 1, false, kMxPairs, 3>(a, st);
  return a4 ? launch<2, 1, true, kMxLinear, 4>(a, st) : launch<2, 1, false, kMxLinear, 3>(a, st);
}

}  // namespace tllm
