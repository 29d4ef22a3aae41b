// Products with an MXFP4 weight for few rows: the weight streams past rows that come from the L2.
//
//   D[n, r] = sum_k W[n, k] X[r, k]        W MXFP4 [N, K], X bf16 or MXFP4
//
// What bounds it is the weight's arrival, N K 17 / 32 bytes of every expert that has rows (8 tokens of 32 experts, 186 MB: mlp1 34.0 us,
// 5.5 TB/s; a plain read reaches 6.1), and with one token the chain of latencies around it (9.8 us for 35 MB: a workgroup's first weights
// leave with its rows, whose addresses are the pairs'). A workgroup of NW
// wavefronts owns 16 NT weight rows and up to 16 activation rows; the wavefronts deal the K steps of 128 between them (sums meet in
// LDS, added in a fixed order). Weights and activations go straight to LDS, U steps of a wavefront at a time in a ring that is its
// alone, so that nothing but the wavefront's own count of arrivals is waited for. That path is what the addresses ask for: a
// 16-byte load is one access of the cache for four neighbouring lanes with 64 neighbouring bytes and one for each lane otherwise, and a
// matrix operand has its rows in neighbouring lanes (33 tokens, loaded to registers that way: 24.2 million accesses, 63.8 us; this
// way, with 32 weight rows as there, 7.8 million and 59.5).
//
// In a step lane (m, g) of a fragment has block mx_quarter(g) of weight row m, and the four v_mfma_f32_16x16x32_bf16 take 8 of its 32
// values each, from both operands. The codes become bf16 on the way, exactly, once per step for all rows; a lane reads its block's scale
// byte from LDS, where the tile's lie as in memory. With MXFP4 activations, in registers, the step is one
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes both blocks and scales as they are. All loads are buffer loads: what lies behind the
// tensors' end, rows that are not there and blocks behind the last one come as zeros without a fetch. None carries the nontemporal
// hint: a step takes half a line, and with the hint the other half's request fetched the line again (one token 14.4 us with, 10.1
// without).
#include "mx_common.h"

namespace tllm {

// A wavefront's walk over its steps: wave, wave + NW, ... of K, through a ring of its own in LDS.
struct MxWalk {
  u32x4 w, x;                                              // buffers
  __amdgpu_buffer_rsrc_t x_scales;                         // (MXFP4 rows alone)
  const unsigned char* scales;                             // LDS: scale bytes of this lane's weight row
  unsigned char* ring;                                     // LDS: this wavefront's
  int blocks, nn, wave, lane;
};

template <int N, int LOADS>
__device__ __forceinline__ void wait_steps_left(int left) {  // at most `left` (<= N) steps of LOADS loads still on their way
  if constexpr (N == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    if (left >= N) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N * LOADS) : "memory");
    else wait_steps_left<N - 1, LOADS>(left);
  }
}

// Up to RP bf16 rows, 4, 8 or 16. In a step a row is 256 bytes, four loads of four rows; weights 64 bytes, a load of sixteen rows.
// The columns of a product are sixteen: with up to 8 rows they hold two of the step's four pieces of K for all rows (column c: row c %
// RP, piece c / RP), with up to 4 all four. The products with a piece's weights are then good in that piece's columns and nonsense in
// the others, so each piece has its own sums, of which only those columns are kept: fewer reads for the same products.
// In LDS a row's sixteens are XORed so that the lanes that a read serves together (mx_quarter) are in different banks.
// `row_at(RP, r)`: where row r, of up to RP, begins in x. `ready`: called when the first loads are on their way.
template <int NT, int RP, int NW, int U, class Row, class F>
__device__ __forceinline__ void mx_walk(const MxWalk& m, float* sums, int sums_pitch, Row&& row_at, F&& ready) {
  constexpr int C = 16 / RP, X = 4 / C, XI = RP / 4, LOADS = NT + XI, SLOT = LOADS * 1024;
  const int lane = m.lane, m16 = lane & 15, g = lane >> 4, u = mx_quarter(g), steps = (m.blocks + 3) / 4, mine = m16 / RP, r = m16 % RP;
  const int n = (steps - m.wave + NW - 1) / NW;            // steps of this wavefront; may be none
  auto fold = [](int row) { return 4 * (row & 3) + (row >> 2) * C; };
  unsigned wo[NT], xo[XI];
  int xb[XI];                                              // which block of the step this lane loads of x
  const int wrow = lane >> 2, wb = (lane & 3) ^ (wrow >> 3);
#pragma unroll
  for (int t = 0; t < NT; ++t) wo[t] = static_cast<unsigned>(min(16 * t + wrow, m.nn - 1) * m.blocks + wb) * 16;
#pragma unroll
  for (int j = 0; j < XI; ++j) {
    const int row = 4 * j + (lane >> 4), c = (lane & 15) ^ fold(row);
    xo[j] = row_at(std::integral_constant<int, RP>{}, row);
    xb[j] = c >> 2;
    if (xo[j] != MX_NONE) xo[j] += 16 * c;
  }
  const unsigned ring = static_cast<unsigned>(reinterpret_cast<uintptr_t>(m.ring));
  auto issue = [&](int j, int slot) {
    const int b = 4 * (m.wave + NW * j);
#pragma unroll
    for (int t = 0; t < NT; ++t) mx_load_lds(m.w, b + wb < m.blocks ? wo[t] : MX_NONE, b * 16, ring + slot * SLOT + t * 1024);
#pragma unroll
    for (int i = 0; i < XI; ++i) mx_load_lds(m.x, b + xb[i] < m.blocks ? xo[i] : MX_NONE, b * 64, ring + slot * SLOT + (NT + i) * 1024);
  };
  f32x4 acc[NT][C];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int first = n < U ? n : U;
#pragma unroll 1
  for (int j = 0; j < first; ++j) issue(j, j);
  ready(first * LOADS);
  int slot = 0;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int left = n - 1 - j;
    wait_steps_left<U - 1, LOADS>(left < U - 1 ? left : U - 1);
    const unsigned char* const at = m.ring + slot * SLOT;
    const int b = 4 * (m.wave + NW * j) + u;
    u32x4 wq[NT], xq[X];
    unsigned e[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wq[t] = *reinterpret_cast<const u32x4*>(at + t * 1024 + m16 * 64 + ((u ^ (m16 >> 3)) << 4));
      e[t] = b < m.blocks ? m.scales[16 * t * m.blocks + b] : 0u;         // (of blocks that are not there: 0, not another row's)
    }
#pragma unroll
    for (int i = 0; i < X; ++i) xq[i] = *reinterpret_cast<const u32x4*>(at + NT * 1024 + r * 256 + (((4 * u + C * i + mine) ^ fold(r)) << 4));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // read, before the slot is filled again
    if (j + U < n) issue(j + U, slot);
    slot = slot + 1 == U ? 0 : slot + 1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float scale = __builtin_bit_cast(float, e[t] << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[t][i % C] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_bf16x8(wq[t][i], scale), __builtin_bit_cast(bf16x8, xq[i / C]), acc[t][i % C], 0, 0, 0);
    }
  }
  __syncthreads();                                         // (the sums lie over the rings)
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

// The same for up to 16 rows of MXFP4, which come to registers.
template <int NT, int NW, int U, class F>
__device__ __forceinline__ void mx_walk4(const MxWalk& m, __amdgpu_buffer_rsrc_t w, __amdgpu_buffer_rsrc_t x, unsigned row_at, unsigned row_scales_at, float* sums,
                                         int sums_pitch, F&& ready) {
  const int m16 = m.lane & 15, g = m.lane >> 4, steps = (m.blocks + 3) / 4;
  u32x4 wq[U][NT], xq[U];
  unsigned xs[U];
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < steps; base += NW * U) {
    const int step0 = base + m.wave * U;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s) + g;
#pragma unroll
      for (int t = 0; t < NT; ++t) wq[s][t] = mx_load16(w, b < m.blocks ? ((16 * t + m16) * m.blocks + b) * 16 : MX_NONE);
      const bool ok = b < m.blocks && row_at != MX_NONE;
      xq[s] = mx_load16(x, ok ? row_at + 16 * b : MX_NONE);
      xs[s] = mx_load1(m.x_scales, ok ? row_scales_at + b : MX_NONE);
    }
    if (base == 0) ready(0);
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int b = 4 * (step0 + s) + g;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const unsigned scale = b < m.blocks ? m.scales[16 * t * m.blocks + b] : 0u;
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
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[m16 * sums_pitch + 16 * t + 4 * g + i] = acc[t][i];
}

// Scale bytes in LDS as they lie in memory, from the sixteen on in which the first row begins.
static __host__ __device__ __forceinline__ int stream_scale_lds(int rows, int blocks) { return (rows * blocks + 15 + 1023) / 1024 * 1024; }

// LDS of a wavefront's ring: KB a step is NT + RP / 4
template <int NT, bool A4, int U4, int U8, int U16>
constexpr int stream_ring() {
  int most = (NT + 1) * U4;
  if ((NT + 2) * U8 > most) most = (NT + 2) * U8;
  if ((NT + 4) * U16 > most) most = (NT + 4) * U16;
  return A4 ? 0 : most * 1024;
}
template <int NT, bool A4, int NW, int U4, int U8, int U16>
static __host__ __device__ __forceinline__ int stream_lds(int blocks) {
  constexpr int sums = NW * 16 * (16 * NT + 1) * 4, rings = NW * stream_ring<NT, A4, U4, U8, U16>();
  return (sums > rings ? sums : rings) + stream_scale_lds(16 * NT, blocks);
}

template <int NT, bool A4, int MODE, int NW, int U4, int U8, int U16>
__global__ __launch_bounds__(NW * 64) void mx_stream_kernel(MxArgs a, int tiles_n) {
  constexpr int BN = 16 * NT, BR = 16, THREADS = NW * 64, PITCH = BN + 1, RING = stream_ring<NT, A4, U4, U8, U16>();
  extern __shared__ __align__(1024) unsigned char smem[];  // rings, later sums [NW][BR][PITCH]; scale bytes
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
  const unsigned char* const scales_from = a.w_scales + wrow * blocks;
  const int shift = mx_scale_shift(scales_from);
  unsigned char* const scale_bytes = smem + stream_lds<NT, A4, NW, U4, U8, U16>(blocks) - stream_scale_lds(BN, blocks);

  // The pairs of the item's rows, if the rows are gathered: through the scalar cache, since vector loads would come back behind
  // the weights that are asked for on this CU already.
  constexpr bool gather = MODE == kMxSwiglu;
  const ScalarInts order = mx_scalar(a.order) + it.first;
  const unsigned last_pair = static_cast<unsigned>(a.rows - 1);
  auto row_of = [&](auto most, int r) {                     // row r of the item in x; r differs from lane to lane
    constexpr int RP = decltype(most)::value;
    if (!gather) return static_cast<unsigned>(r);
    unsigned pair[RP], mine = 0;                            // (all asked for together)
#pragma unroll
    for (int j = 0; j < RP; ++j) pair[j] = static_cast<unsigned>(order[min(j, it.rows - 1)]);
#pragma unroll
    for (int j = 0; j < RP; ++j) mine = r == j ? pair[j] : mine;
    return min(mine, last_pair) / static_cast<unsigned>(a.top);
  };
  const int row_bytes = A4 ? blocks * 16 : a.k * 2;
  const unsigned char* const xb = static_cast<const unsigned char*>(a.x) + (gather ? 0 : it.first * a.x_pitch);
  const unsigned x_span = static_cast<unsigned>(((gather ? a.tokens : it.rows) - 1) * a.x_pitch + row_bytes);
  MxWalk m;
  m.w = mx_buffer_words(a.w + wrow * blocks * 16, nn * blocks * 16);
  m.x = mx_buffer_words(xb, x_span);
  m.scales = scale_bytes + shift + m16 * blocks;
  m.ring = smem + wave * RING;
  m.blocks = blocks;
  m.nn = nn;
  m.wave = wave;
  m.lane = lane;
  float* const sums = reinterpret_cast<float*>(smem);
  float* const mine = sums + wave * BR * PITCH;

  // the scale bytes, 1 KB a load, dealt to the wavefronts (to whole words: a word that the end cuts would come as zeros)
  {
    const int bytes = (shift + nn * blocks + 3) & ~3;
    const u32x4 from = mx_buffer_words(scales_from - shift, bytes);
    const unsigned to = static_cast<unsigned>(reinterpret_cast<uintptr_t>(scale_bytes));
    for (int i = wave * 1024; i < bytes; i += NW * 1024) mx_load_lds(from, 16 * lane, i, to + i);
  }
  auto ready = [&](int loads) {                             // behind the scales' loads, `loads` others
    if (loads >= 12) asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
    else if (loads >= 6) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if constexpr (A4) {
    const auto w = mx_buffer(a.w + wrow * blocks * 16, nn * blocks * 16), x = mx_buffer(xb, x_span);
    m.x_scales = mx_buffer(a.x_scales + static_cast<int64_t>(it.first) * blocks, it.rows * blocks);
    mx_walk4<NT, NW, U4>(m, w, x, m16 < it.rows ? static_cast<unsigned>(m16 * a.x_pitch) : MX_NONE, m16 * blocks, mine, PITCH, ready);
  } else {
    auto row_at = [&](auto most, int r) {
      const unsigned row = row_of(most, r);
      return r < it.rows ? static_cast<unsigned>(row * a.x_pitch) : MX_NONE;
    };
    if (columns == 4) mx_walk<NT, 4, NW, U4>(m, mine, PITCH, row_at, ready);
    else if (columns == 8) mx_walk<NT, 8, NW, U8>(m, mine, PITCH, row_at, ready);
    else mx_walk<NT, 16, NW, U16>(m, mine, PITCH, row_at, ready);
  }

  // this thread's results: where they go, and their bias
  constexpr int OUTS = BR * BN / (MODE == kMxSwiglu ? 2 : 1), PER = (OUTS + THREADS - 1) / THREADS;
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
  __syncthreads();
  auto total = [&](int r, int n) {
    float v = 0.f;
    for (int c = r; c < 16; c += columns)
#pragma unroll
      for (int w = 0; w < NW; ++w) v += sums[(w * BR + c) * PITCH + n];
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
  const int lds = stream_lds<NT, A4, NW, U4, U8, U16>(a.k / 32);
  static std::atomic<uint64_t> done{0};
  const void* const kernel = reinterpret_cast<const void*>(mx_stream_kernel<NT, A4, MODE, NW, U4, U8, U16>);
  TLLM_REQUIRE(raise_lds_limit(kernel, 160 * 1024, done) == hipSuccess, TLLM_E_LAUNCH, "mxfp4 product: the LDS limit could not be raised");
  TLLM_REQUIRE(lds <= 160 * 1024, TLLM_E_SHAPE, "mxfp4 product: %d values in a row are too many", a.k);
  hipLaunchKernelGGL((mx_stream_kernel<NT, A4, MODE, NW, U4, U8, U16>), dim3((unsigned)(tiles * items)), dim3(NW * 64), lds, st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

// The workgroup. Wide ones (64 weight rows) read the activations less often and pay where items are full: 128 tokens of 32 experts
// mlp1 97.7 us with 32 rows, 89.5 with 64; 33 tokens, four pairs an expert, 58.4 and 57.6, 24 tokens 53.0 and 54.0; mlp2, half as many
// weight rows, 64 tokens 43.7 and 43.6, 33 34.9 and 36.2; 16 rows of [32768, 2880] 13.2 and 12.1, 8 rows 11.6 and 11.7. And where
// there are enough of them: 33 rows of [8192, 2880], 384 workgroups, 8.0 and 9.3; 65 rows of [5120, 2880], 400, 9.2 and 8.8. Narrow
// ones, with their K share in one piece, where the launch would have less than one for every other CU otherwise: one row of
// [2880, 4096] 6.9 us with 32 weight rows, 4.7 with 16; 64 rows of [1024, 1024] 5.8 with 64, 4.4 with 32. Few steps in the rings:
// workgroups on the CU bring more than a longer ring does (33 tokens 59.5 us with rings of 6 KB, 59.8 with 9, 64 with 12, 78 with 18,
// before a row's pairs were asked for together). Beyond 229344 values a row the scale bytes of sixteen weight rows, 112 KB and up to 129, leave
// eight wavefronts' rings (48 KB) no room, four's do: one row of [4096, 229376] 136 us, of [4096, 229344] in eight 99.
template <int MODE>
static int launch_bf16(const MxArgs& a, hipStream_t st) {
  const int64_t items = a.order ? (a.rows < a.experts ? a.rows : a.experts) + a.rows / 32 : (a.rows + 15) / 16;
  const bool full = a.rows > (MODE == kMxSwiglu ? 4ll : MODE == kMxPairs ? 8ll : 12ll) * a.experts;
  if (full && (a.n + 63) / 64 * items > 384 && a.k <= 16384) return launch<4, false, MODE, 4, 1, 1, 1>(a, st);
  if ((a.n + 31) / 32 * items > 128 && a.k <= 32768) return launch<2, false, MODE, 4, 2, 1, 1>(a, st);
  if (stream_lds<1, false, 8, 3, 2, 1>(a.k / 32) > 160 * 1024) return launch<1, false, MODE, 4, 3, 2, 1>(a, st);
  return launch<1, false, MODE, 8, 3, 2, 1>(a, st);
}

int mx_stream(const MxArgs& a, int mode, bool a4, hipStream_t st) {
  if (mode == kMxSwiglu) return launch_bf16<kMxSwiglu>(a, st);
  if (mode == kMxPairs) return launch_bf16<kMxPairs>(a, st);
  if (!a4) return launch_bf16<kMxLinear>(a, st);
  return (a.n + 31) / 32 * ((a.rows + 15) / 16) > 128 && a.k <= 32768 ? launch<2, true, kMxLinear, 4, 4, 1, 1>(a, st) : launch<1, true, kMxLinear, 8, 3, 1, 1>(a, st);
}

}  // namespace tllm
