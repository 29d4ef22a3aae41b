// The product of two MXFP4 matrices for many rows: tiles on v_mfma_scale_f32_16x16x128_f8f6f4, which takes both operands' codes and
// scale bytes as they are, at four times the rate of bf16.
//
//   D[r, n] = sum_k X[r, k] W[n, k]
//
// K goes in slices of 128, 64 bytes (four blocks) of a row: lane (m, g) of a fragment has block g of row m, one 16-byte read. Slices
// of both operands come into a ring of S in LDS by buffer loads straight there, a row's four blocks in an order (block g at place g ^
// (row / 4 % 2)) that keeps the sixteen lanes that a read serves together in different banks. Scale bytes of all rows lie in LDS
// for the whole of K. A slice's fragments are read under the MFMAs of the one before.
#include "mx_common.h"

namespace tllm {

template <int TB_, int RB_, int WM_, int WN_, int S_>
struct MxTile4 {
  static constexpr int TB = TB_, RB = RB_, WM = WM_, WN = WN_, S = S_, NW = WM * WN;
  static constexpr int BM = 16 * TB * WM, BN = 16 * RB * WN;
  static constexpr int XB = BM * 64, STAGE = (BM + BN) * 64;
  static constexpr int XL = BM / 16 / NW, WL = BN / 16 / NW, LPW = XL + WL;       // loads of a wavefront per slice: 16 rows each
  static_assert(XL * 16 * NW == BM && WL * 16 * NW == BN && S >= 2, "whole loads");
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
  const int blocks = a.k / 32, slices = (blocks + 3) / 4;

  const u32x4 xr = mx_buffer_words(static_cast<const unsigned char*>(a.x) + r0 * blocks * 16, rows * blocks * 16);
  const u32x4 wr = mx_buffer_words(a.w + static_cast<int64_t>(n0) * blocks * 16, nn * blocks * 16);
  unsigned xo[XL], wo[WL];
  const unsigned place_of = ((lane & 3) ^ (lane >> 4 & 1)) * 16;
#pragma unroll
  for (int j = 0; j < XL; ++j) xo[j] = min((wave * XL + j) * 16 + (lane >> 2), rows - 1) * (blocks * 16) + place_of;
#pragma unroll
  for (int j = 0; j < WL; ++j) wo[j] = min((wave * WL + j) * 16 + (lane >> 2), nn - 1) * (blocks * 16) + place_of;
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(smem));
  auto issue = [&](int slice, int place) {
    const int s = slice < slices ? slice : slices - 1;     // (behind the last slice it again, so that the loads in flight can be counted)
    const unsigned base = lds0 + place * C::STAGE;
#pragma unroll
    for (int j = 0; j < XL; ++j) mx_load_lds(xr, xo[j], s * 64, base + (wave * XL + j) * 1024);
#pragma unroll
    for (int j = 0; j < WL; ++j) mx_load_lds(wr, wo[j], s * 64, base + C::XB + (wave * WL + j) * 1024);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) issue(s, s);

  unsigned* const sc = reinterpret_cast<unsigned*>(smem + S * C::STAGE);
  const int pitch = mx_scale_words(blocks);
  mx_fetch_scales<C::NW * 64>(sc, a.x_scales + r0 * blocks, rows, blocks, tid);
  mx_fetch_scales<C::NW * 64>(sc + BM * pitch, a.w_scales + static_cast<int64_t>(n0) * blocks, nn, blocks, tid);
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
  const unsigned char* const scb = reinterpret_cast<const unsigned char*>(sc);
  u32x4 x[2][TB], w[2][RB];
  unsigned xs[2][TB], ws[2][RB];
  const int xat = 16 * TB * wm + m16, wat = 16 * RB * wn + m16, at = (g ^ (m16 >> 2 & 1)) << 4;
  auto read = [&](auto buf, int slice, int place) {
    constexpr int b = decltype(buf)::value;
    const unsigned char* const st = smem + place * C::STAGE;
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      x[b][i] = *reinterpret_cast<const u32x4*>(st + (xat + 16 * i) * 64 + at);
      xs[b][i] = scb[(xat + 16 * i) * pitch * 4 + 4 * slice + g];
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      w[b][i] = *reinterpret_cast<const u32x4*>(st + C::XB + (wat + 16 * i) * 64 + at);
      ws[b][i] = scb[(BM + wat + 16 * i) * pitch * 4 + 4 * slice + g];
    }
  };
  auto multiply = [&](auto buf, int slice) {
    constexpr int b = decltype(buf)::value;
    if (slice + 1 == slices && 4 * slice + g >= blocks) {  // blocks of the last slice that are not there
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        x[b][i] = u32x4{0, 0, 0, 0};
        xs[b][i] = 127;
      }
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        w[b][i] = u32x4{0, 0, 0, 0};
        ws[b][i] = 127;
      }
    }
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        i32x8 wv = {}, xv = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          wv[j] = w[b][r][j];
          xv[j] = x[b][i][j];
        }
        acc[i][r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[i][r], 4, 4, 0, ws[b][r], 0, xs[b][i]);
      }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * LPW) : "memory");
  read(I0{}, 0, 0);
  int place = 0;
  auto step = [&](auto buf, auto other, int s) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LPW) : "memory");
    issue(s + S, place);
    place = place + 1 == S ? 0 : place + 1;
    read(other, s + 1, place);                             // (behind the last slice: the last one again, not used)
    multiply(buf, s);
  };
  for (int s = 0; s < slices; s += 2) {
    step(I0{}, I1{}, s);
    if (s + 1 < slices) step(I1{}, I0{}, s + 1);
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
static int launch_tiles4(const MxArgs& a, hipStream_t st) {
  const int64_t tiles = (a.n + C::BN - 1) / C::BN, items = (a.rows + C::BM - 1) / C::BM;
  const int lds = C::S * C::STAGE + (C::BM + C::BN) * mx_scale_words(a.k / 32) * 4 + 16;
  TLLM_REQUIRE(tiles * items < (1ll << 30), TLLM_E_SHAPE, "mxfp4 product: %lld rows of %d outputs are too many", (long long)a.rows, a.n);
  TLLM_REQUIRE(lds <= 160 * 1024, TLLM_E_SHAPE, "mxfp4 product: %d values in a row are too many for its tiles", a.k);
  static std::atomic<uint64_t> done{0};
  TLLM_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(mx_tile4_kernel<C>), 160 * 1024, done) == hipSuccess, TLLM_E_LAUNCH,
               "mxfp4 product: the LDS limit could not be raised");
  hipLaunchKernelGGL(mx_tile4_kernel<C>, dim3((unsigned)((tiles * items + 7) / 8 * 8)), dim3(C::NW * 64), lds, st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

#ifndef MX_SHAPE4
#define MX_SHAPE4 4, 4, 2, 4, 4
#endif

int mx_tiles4(const MxArgs& a, hipStream_t st) { return launch_tiles4<MxTile4<MX_SHAPE4>>(a, st); }

}  // namespace tllm
