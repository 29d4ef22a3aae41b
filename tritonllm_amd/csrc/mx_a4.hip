// The product of two MXFP4 matrices for many rows: tiles on v_mfma_scale_f32_16x16x128_f8f6f4, which takes both operands' codes and
// scale bytes as they are, at four times the rate of bf16.
//
//   D[r, n] = sum_k X[r, k] W[n, k]
//
// K goes in slices of 256, eight blocks and a whole cache line of a row (with half lines a CU took in 30 GB/s). A slice is two
// MFMAs deep: in the j-th lane (m, g) of a fragment has block 2 u + j of row m, u = mx_quarter(g), one 16-byte read, and both
// blocks' scale bytes side by side. Slices of both operands come into a ring of S in LDS by buffer loads straight there, block b of a
// row at place b ^ (row / 2 % 8). Scale bytes of all rows lie in LDS for the whole of K. A half slice's fragments are read under
// the MFMAs of the one before.
//
// What bounds it: 2048 rows of [5120, 2880] take 30 us, one 128 x 320 tile to a CU, 2.0 PFLOP/s: 9 us of beginning and end, then 1.7 us a
// slice, of which the MFMAs are 0.7 and the LDS reads as much; 4096 x 4096 x 4096 54 us, 2.5 PFLOP/s.
#include "mx_common.h"

namespace tllm {

template <int TB_, int RB_, int WM_, int WN_, int S_>
struct MxTile4 {
  static constexpr int TB = TB_, RB = RB_, WM = WM_, WN = WN_, S = S_, NW = WM * WN;
  static constexpr int BM = 16 * TB * WM, BN = 16 * RB * WN;
  static constexpr int XB = BM * 128, STAGE = (BM + BN) * 128;
  static constexpr int XL = BM / 8 / NW, WL = BN / 8 / NW, LPW = XL + WL;         // loads of a wavefront per slice: 8 rows each
  static_assert(XL * 8 * NW == BM && WL * 8 * NW == BN && S >= 2, "whole loads");
};

template <class C>
__global__ __launch_bounds__(C::NW * 64) void mx_tile4_kernel(MxArgs a, int tiles_n) {
  constexpr int TB = C::TB, RB = C::RB, S = C::S, BM = C::BM, BN = C::BN, XL = C::XL, WL = C::WL, LPW = C::LPW;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % C::WN, wm = wave / C::WN, m16 = lane & 15, g = lane >> 4;
  const int items = static_cast<int>((a.rows + BM - 1) / BM), all = items * tiles_n, per = (all + 7) / 8, id = blockIdx.x >> 3;
  const int t = (blockIdx.x & 7) * per + id;               // neighbours in an XCD: the same weight rows, then the next
  if (id >= per || t >= all) return;
  const int n0 = t / items * BN;
  const int64_t r0 = static_cast<int64_t>(t % items) * BM, left = a.rows - r0;
  const int rows = static_cast<int>(left < BM ? left : BM), nn = a.n - n0 < BN ? a.n - n0 : BN;
  const int blocks = a.k / 32, slices = (blocks + 7) / 8;

  const u32x4 xr = mx_buffer_words(static_cast<const unsigned char*>(a.x) + r0 * blocks * 16, rows * blocks * 16);
  const u32x4 wr = mx_buffer_words(a.w + static_cast<int64_t>(n0) * blocks * 16, nn * blocks * 16);
  unsigned xo[XL], wo[WL];
  // eight rows to a load, lane l at row l / 8 of them and at place l % 8, where the block (l % 8) ^ (row / 2 % 8) belongs
  auto block_at = [&](int i) { return static_cast<unsigned>((lane & 7) ^ ((4 * i + (lane >> 4)) & 7)) * 16; };
#pragma unroll
  for (int j = 0; j < XL; ++j) xo[j] = min((wave * XL + j) * 8 + (lane >> 3), rows - 1) * (blocks * 16) + block_at(wave * XL + j);
#pragma unroll
  for (int j = 0; j < WL; ++j) wo[j] = min((wave * WL + j) * 8 + (lane >> 3), nn - 1) * (blocks * 16) + block_at(wave * WL + j);
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(smem));
  // Of the last slice blocks may not be there: their lanes ask behind the buffer's end and put zeros into LDS. Behind the last slice
  // it comes again, so that the loads in flight can be counted.
  auto issue = [&](int slice, int place) {
    const int s = slice < slices ? slice : slices - 1;
    const unsigned base = lds0 + place * C::STAGE;
#pragma unroll
    for (int j = 0; j < XL; ++j)
      mx_load_lds(xr, 8 * s + static_cast<int>(block_at(wave * XL + j) / 16) < blocks ? xo[j] : MX_NONE, s * 128, base + (wave * XL + j) * 1024);
#pragma unroll
    for (int j = 0; j < WL; ++j)
      mx_load_lds(wr, 8 * s + static_cast<int>(block_at(wave * WL + j) / 16) < blocks ? wo[j] : MX_NONE, s * 128, base + C::XB + (wave * WL + j) * 1024);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) issue(s, s);

  unsigned char* const sc = smem + S * C::STAGE;
  const int pitch = mx_scale_pitch(blocks), x_part = mx_scale_lds(BM, blocks);
  const unsigned char *const x_scales = a.x_scales + r0 * blocks, *const w_scales = a.w_scales + static_cast<int64_t>(n0) * blocks;
  mx_fetch_scales<C::NW * 64>(sc, x_scales, rows, blocks, tid);
  mx_fetch_scales<C::NW * 64>(sc + x_part, w_scales, nn, blocks, tid);
  const bool four = mx_whole_fours(a);
  bf16x4 bias[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) bias[rb] = mx_bias4(a, four, n0, 16 * (RB * wn + rb) + 4 * g, nn);
  __syncthreads();

  f32x4 acc[TB][RB];
#pragma unroll
  for (int i = 0; i < TB; ++i)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[i][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 x[2][TB], w[2][RB];
  unsigned xs[2][TB], ws[2][RB];                           // two scale bytes each, of this slice and the next
  const int xat = 16 * TB * wm + m16, wat = 16 * RB * wn + m16, flip = m16 >> 1, u = mx_quarter(g);
  auto read = [&](auto half, int place) {
    constexpr int j = decltype(half)::value;
    const unsigned char* const st = smem + place * C::STAGE + (((2 * u + j) ^ flip) << 4);
#pragma unroll
    for (int i = 0; i < TB; ++i) x[j][i] = *reinterpret_cast<const u32x4*>(st + (xat + 16 * i) * 128);
#pragma unroll
    for (int i = 0; i < RB; ++i) w[j][i] = *reinterpret_cast<const u32x4*>(st + C::XB + (wat + 16 * i) * 128);
  };
  const unsigned char *const my_xs = sc + mx_scale_shift(x_scales) + xat * pitch + 2 * u,
                      *const my_ws = sc + x_part + mx_scale_shift(w_scales) + wat * pitch + 2 * u;
  const int rest = blocks - 8 * (slices - 1) - 2 * u;      // of this lane's two blocks of the last slice: how many are there
  const unsigned last_mask = rest >= 2 ? 0xffffu : rest == 1 ? 0xffu : 0u;
  auto read_scales = [&](auto buf, int slice) {
    constexpr int b = decltype(buf)::value;
    const unsigned mask = slice + 1 < slices ? 0xffffu : last_mask;      // (zeros times 2^-127, not times another row's scale)
    auto two = [&](const unsigned char* p) { return (p[0] | static_cast<unsigned>(p[1]) << 8) & mask; };
#pragma unroll
    for (int i = 0; i < TB; ++i) xs[b][i] = two(my_xs + 16 * i * pitch + 8 * slice);
#pragma unroll
    for (int i = 0; i < RB; ++i) ws[b][i] = two(my_ws + 16 * i * pitch + 8 * slice);
  };
  auto multiply = [&](auto half, auto buf) {
    constexpr int j = decltype(half)::value, b = decltype(buf)::value;
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        i32x8 wv = {}, xv = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          wv[e] = w[j][r][e];
          xv[e] = x[j][i][e];
        }
        acc[i][r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[i][r], 4, 4, j, ws[b][r], j, xs[b][i]);
      }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * LPW) : "memory");
  read(I0{}, 0);
  read_scales(I0{}, 0);
  int place = 0;
  auto step = [&](auto buf, auto other, int s) {
    read(I1{}, place);
    multiply(I0{}, buf);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LPW) : "memory");
    issue(s + S, place);
    place = place + 1 == S ? 0 : place + 1;
    read(I0{}, place);                                     // (behind the last slice: the last one again, not used)
    read_scales(other, s + 1);
    multiply(I1{}, buf);
  };
  for (int s = 0; s < slices; s += 2) {
    step(I0{}, I1{}, s);
    if (s + 1 == slices) break;
    step(I1{}, I0{}, s + 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

#pragma unroll
  for (int i = 0; i < TB; ++i) {
    const int r = 16 * (TB * wm + i) + m16;
    if (r >= rows) continue;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int n = 16 * (RB * wn + rb) + 4 * g;
      if (n < nn) mx_store4<kMxLinear>(a, four, r0 + r, n0, n, nn, acc[i][rb], bias[rb]);
    }
  }
}

template <class C>
static int64_t tile4_lds(int k) { return static_cast<int64_t>(C::S) * C::STAGE + mx_scale_lds(C::BM, k / 32) + mx_scale_lds(C::BN, k / 32); }

template <class C>
static int launch_tiles4(const MxArgs& a, hipStream_t st) {
  const int64_t tiles = (a.n + C::BN - 1) / C::BN, items = (a.rows + C::BM - 1) / C::BM;
  TLLM_REQUIRE(tiles * items < (1ll << 32) / (C::NW * 64) - 8, TLLM_E_SHAPE, "mxfp4 product: %lld rows of %d outputs are too many", (long long)a.rows, a.n);
  static std::atomic<uint64_t> done{0};
  TLLM_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(mx_tile4_kernel<C>), 160 * 1024, done) == hipSuccess, TLLM_E_LAUNCH,
               "mxfp4 product: the LDS limit could not be raised");
  hipLaunchKernelGGL(mx_tile4_kernel<C>, dim3((unsigned)((tiles * items + 7) / 8 * 8)), dim3(C::NW * 64), tile4_lds<C>(a.k), st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

// The tiles, and what a launch of them takes: `fixed` us and, for each slice of K, `one` with up to one tile to a CU, `more` for each
// of a CU's tiles beyond. Measured with 2880 and 4096 values a row (us; 128 x 256, 128 x 320, 128 x 128, 64 x 128, 64 x 64):
//   2048 rows of [5120, 2880] 43.3 29.9 45.8 42.4 49.2     2048 of [4096, 2880] 25.1 28.4 31.9 33.0 40.9     1000 of [2880, 4096] 24.8 82.3 18.8 20.0 21.0
//   512 of [4096, 2880] 21.3 25.9 16.0 13.7 12.8     300 of [5120, 2880] 21.6 25.6 15.6 13.1 11.9     64 of [5120, 2880] 18.5 21.5 13.1 11.1 8.7
template <int TB, int RB, int WM, int WN, int S>
static void weigh(const MxArgs& a, float fixed, float one, float more, int number, float* best, int* which) {
  typedef MxTile4<TB, RB, WM, WN, S> C;
  if (tile4_lds<C>(a.k) > 160 * 1024) return;
  const int64_t tiles = (a.n + C::BN - 1) / C::BN * ((a.rows + C::BM - 1) / C::BM), each = (tiles + 255) / 256;
  const float t = fixed + (a.k + 255) / 256 * (each == 1 ? one : more * each);
  if (*which == 0 || t < *best) {
    *best = t;
    *which = number;
  }
}
static int tile4_of(const MxArgs& a) {
  float best = 0.f;
  int which = 0;
  weigh<4, 4, 2, 4, 2>(a, 9.4f, 1.36f, 1.36f, 1, &best, &which);
  weigh<4, 5, 2, 4, 2>(a, 9.6f, 1.70f, 1.70f, 2, &best, &which);
  weigh<4, 2, 2, 4, 2>(a, 7.5f, 0.71f, 1.02f, 3, &best, &which);
  weigh<2, 2, 2, 4, 2>(a, 6.0f, 0.64f, 0.56f, 4, &best, &which);
  weigh<2, 2, 2, 2, 3>(a, 5.0f, 0.37f, 0.35f, 5, &best, &which);
  return which;
}

// The weight stream and the tiles meet between 64 and 80 rows: 64 rows of [5120, 2880] 8.2 us and 8.8 in tiles, 80 9.9 and 8.6, 128 11.8 and 9.1.
bool mx_tiles4_take(const MxArgs& a) { return a.rows > 80 && tile4_of(a) != 0; }

int mx_tiles4(const MxArgs& a, hipStream_t st) {
  switch (tile4_of(a)) {
    case 1: return launch_tiles4<MxTile4<4, 4, 2, 4, 2>>(a, st);
    case 2: return launch_tiles4<MxTile4<4, 5, 2, 4, 2>>(a, st);
    case 3: return launch_tiles4<MxTile4<4, 2, 2, 4, 2>>(a, st);
    case 4: return launch_tiles4<MxTile4<2, 2, 2, 4, 2>>(a, st);
    default: return launch_tiles4<MxTile4<2, 2, 2, 2, 3>>(a, st);
  }
}

}  // namespace tllm
