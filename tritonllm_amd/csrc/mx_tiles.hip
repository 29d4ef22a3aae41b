// Products with an MXFP4 weight for many rows of bf16: tiles on the matrix cores.
//
//   D[r, n] = sum_k X[r, k] W[n, k]        X bf16, W MXFP4, a run of one expert's rows to a tile
//
// K goes in slices of 64: a slice of X is 128 bytes a row, of W 32 (two blocks). Both come into a ring of S slices in LDS as they are
// (buffer loads straight to LDS); the codes become bf16 in registers, in front of v_mfma_f32_16x16x32_bf16, weight rows on M: a
// wavefront converts each of its weight fragments once per slice, five issue cycles a pair of values next to the sixteen of an MFMA,
// and they run side by side. In a slice lane (m, g) of a fragment has the values k = 16 u .. 16 u + 15, u = mx_quarter(g), half a block,
// eight for each of two MFMAs, of both operands. The next half slice's fragments are read under the MFMAs of this one. The
// scale bytes of the tile's weight rows lie in LDS for the whole of K, a lane reads one for a fragment's slice. A lane ends up with four
// neighbouring weight rows of one row of X and stores them from its registers.
//
// What bounds it: the matrix cores at the clock that they leave (one 128 x 256 tile to a CU, [4096] outputs of 2048 rows, goes
// through K at 1.18 PFLOP/s, where a large library product reaches 1.24), behind 11 us of a launch's beginning and end per round
// of tiles, which workgroups that share a CU cover for one another, and the rows that an expert's last tile lacks. 2048 tokens of
// 32 experts, four each, hidden and inner 2880: mlp1 312 us (870 TFLOP/s), mlp2's product 173 and its weighted sum 17. Built and
// slower: three slices in the ring of the 128 x 128 tile (two workgroups to a CU instead of three; 340 us), 64 x 512 (472), 128 x 256 (367).
#include "mx_common.h"

namespace tllm {

template <int TB_, int RB_, int WM_, int WN_, int S_>
struct MxTileShape {
  static constexpr int TB = TB_, RB = RB_, WM = WM_, WN = WN_, S = S_, NW = WM * WN;
  static constexpr int BM = 16 * TB * WM, BN = 16 * RB * WN;
  static constexpr int XB = BM * 128, WB = BN * 32, STAGE = XB + WB;
  static constexpr int XL = BM / 8 / NW, WL = BN / 32 / NW, LPW = XL + WL;        // loads of a wavefront per slice: 8 rows of X, 32 of W
  static_assert(XL * 8 * NW == BM && WL * 32 * NW == BN && S >= 2, "whole loads");
};

template <class C, int MODE>
__global__ __launch_bounds__(C::NW * 64) void mx_tile_kernel(MxArgs a, int tiles_n) {
  constexpr int TB = C::TB, RB = C::RB, S = C::S, BM = C::BM, BN = C::BN, XL = C::XL, WL = C::WL, LPW = C::LPW;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % C::WN, wm = wave / C::WN, m16 = lane & 15, g = lane >> 4;
  MxTile it;
  if (a.order == nullptr) {
    const int items = static_cast<int>((a.rows + BM - 1) / BM), all = items * tiles_n, per = (all + 7) / 8, at = blockIdx.x >> 3;
    const int t = (blockIdx.x & 7) * per + at;
    if (at >= per || t >= all) return;
    const int64_t first = static_cast<int64_t>(t % items) * BM, left = a.rows - first;
    it = {0, static_cast<int>(first), static_cast<int>(left < BM ? left : BM), t / items};
  } else {
    it = mx_find_tile(a.offsets, a.experts, static_cast<int>(a.rows), BM, tiles_n, blockIdx.x);
  }
  if (it.rows <= 0) return;
  const int n0 = it.tile_n * BN, blocks = a.k / 32, slices = (blocks + 1) / 2;
  const int nn = a.n - n0 < BN ? a.n - n0 : BN;
  const int64_t wrow = static_cast<int64_t>(it.expert) * a.n + n0;
  constexpr bool gather = MODE == kMxSwiglu;

  // ---- loads
  const unsigned char* const xb = static_cast<const unsigned char*>(a.x) + (gather ? 0 : it.first * a.x_pitch);
  const unsigned x_span = static_cast<unsigned>(((gather ? a.tokens : it.rows) - 1) * a.x_pitch + a.k * 2);
  const auto xr = mx_buffer_words(xb, x_span), wr = mx_buffer_words(a.w + wrow * blocks * 16, nn * blocks * 16);
  unsigned xo[XL], wo[WL];
#pragma unroll
  for (int j = 0; j < XL; ++j) {
    const int r = (wave * XL + j) * 8 + (lane >> 3), rr = r < it.rows ? r : 0;
    const unsigned row = gather ? mx_pair(a, it.first + rr) / static_cast<unsigned>(a.top) : rr;
    xo[j] = static_cast<unsigned>(row * a.x_pitch) + (((lane & 7) ^ (r >> 1 & 7)) << 4);
  }
#pragma unroll
  for (int j = 0; j < WL; ++j) {
    const int r = (wave * WL + j) * 32 + (lane >> 1);
    wo[j] = (r < nn ? r : nn - 1) * (blocks * 16) + ((lane ^ lane >> 4) & 1) * 16;
  }
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>(smem));
  // The last slice's second block may not be there: its lanes ask behind the buffer's end and put zeros into LDS. Behind the last
  // slice it comes again, so that the loads in flight can be counted.
  auto issue = [&](int slice, int place) {
    const int s = slice < slices ? slice : slices - 1;
    const unsigned base = lds0 + place * C::STAGE;
    const bool cut = (blocks & 1) && s + 1 == slices;
#pragma unroll
    for (int j = 0; j < XL; ++j)
      mx_load_lds(xr, cut && (((lane & 7) ^ (4 * (wave * XL + j) + (lane >> 4))) & 4) ? MX_NONE : xo[j], s * 128, base + (wave * XL + j) * 1024);
#pragma unroll
    for (int j = 0; j < WL; ++j) mx_load_lds(wr, cut && ((lane ^ lane >> 4) & 1) ? MX_NONE : wo[j], s * 32, base + C::XB + (wave * WL + j) * 1024);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) issue(s, s);

  // ---- while they are on their way: scale bytes and bias
  unsigned char* const sc = smem + S * C::STAGE;
  const unsigned char* const scales = a.w_scales + wrow * blocks;
  const int pitch = mx_scale_pitch(blocks);
  mx_fetch_scales<C::NW * 64>(sc, scales, nn, blocks, tid);
  const bool four = mx_whole_fours(a);
  bf16x4 bias[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) bias[rb] = mx_bias4(a, four, wrow, 16 * (RB * wn + rb) + 4 * g, nn);
  __syncthreads();

  // ---- the walk over K
  f32x4 acc[TB][RB];
#pragma unroll
  for (int t = 0; t < TB; ++t)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;
  u32x2 q[RB];                                             // a slice's codes, and its scales as fp32
  float qs[RB];
  bf16x8 w[2][RB];
  u32x4 x[2][TB];
  const int xat = 16 * TB * wm + m16, wat = 16 * RB * wn + m16, flip = m16 >> 1, u = mx_quarter(g);
  const unsigned char* const my_scales = sc + mx_scale_shift(scales) + wat * pitch + (u >> 1);
  const bool absent = (blocks & 1) && u >= 2;              // the last slice's second block is not there: zeros times 2^-127
  auto read_w = [&](int slice, int place) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      q[rb] = *reinterpret_cast<const u32x2*>(smem + place * C::STAGE + C::XB + (wat + 16 * rb) * 32 + (u ^ (m16 >> 2 & 2)) * 8);
      unsigned e = my_scales[16 * rb * pitch + 2 * slice];
      if (absent && slice + 1 >= slices) e = 0;
      qs[rb] = __builtin_bit_cast(float, e << 23);
    }
  };
  auto read_x = [&](auto half, int place) {
    constexpr int i = decltype(half)::value;
#pragma unroll
    for (int t = 0; t < TB; ++t)
      x[i][t] = *reinterpret_cast<const u32x4*>(smem + place * C::STAGE + (xat + 16 * t) * 128 + (((2 * u + i) ^ flip) << 4));
  };
  auto convert = [&](auto half) {
    constexpr int i = decltype(half)::value;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) w[i][rb] = mx_bf16x8(q[rb][i], qs[rb]);
  };
  auto multiply = [&](auto half) {
    constexpr int i = decltype(half)::value;
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) acc[t][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i][rb], __builtin_bit_cast(bf16x8, x[i][t]), acc[t][rb], 0, 0, 0);
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * LPW) : "memory");
  // a wavefront whose rows, or weight rows, are not there keeps step and leaves the matrix cores to others
  const bool live = 16 * TB * wm < it.rows && 16 * RB * wn < nn;
  if (live) {
    read_w(0, 0);
    read_x(I0{}, 0);
  }
  int place = 0;
  for (int s = 0; s < slices; ++s) {
    if (live) {
      read_x(I1{}, place);
      convert(I0{});
      multiply(I0{});
      convert(I1{});
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LPW) : "memory");
    issue(s + S, place);
    place = place + 1 == S ? 0 : place + 1;
    if (live) {
      read_w(s + 1, place);                                // (behind the last slice: the last one again, not used)
      read_x(I0{}, place);
      multiply(I1{});
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- lane (m16, g) holds weight rows 4 g .. + 3 of row m16 of X in each fragment pair
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    const int r = 16 * (TB * wm + t) + m16;
    if (r >= it.rows) continue;
    int64_t row = it.first + r;
    if constexpr (MODE == kMxPairs) row = mx_pair(a, it.first + r);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int n = 16 * (RB * wn + rb) + 4 * g;
      if (n >= nn) continue;
      mx_store4<MODE>(a, four, row, n0, n, nn, acc[t][rb], bias[rb]);
    }
  }
}

template <class C>
static int64_t tile_lds(int k) { return static_cast<int64_t>(C::S) * C::STAGE + mx_scale_lds(C::BN, k / 32); }

template <class C, int MODE>
static int launch_tiles(const MxArgs& a, hipStream_t st) {
  const int64_t tiles = (a.n + C::BN - 1) / C::BN;
  const int64_t items = a.order ? mx_items(a.rows, a.experts, C::BM) : (a.rows + C::BM - 1) / C::BM;
  TLLM_REQUIRE(tiles * items < (1ll << 32) / (C::NW * 64) - 8, TLLM_E_SHAPE, "mxfp4 product: %lld rows of %d outputs are too many", (long long)a.rows, a.n);
  static std::atomic<uint64_t> done{0};
  const void* const kernel = reinterpret_cast<const void*>(mx_tile_kernel<C, MODE>);
  TLLM_REQUIRE(raise_lds_limit(kernel, 160 * 1024, done) == hipSuccess, TLLM_E_LAUNCH, "mxfp4 product: the LDS limit could not be raised");
  hipLaunchKernelGGL((mx_tile_kernel<C, MODE>), dim3((unsigned)((tiles * items + 7) / 8 * 8)), dim3(C::NW * 64), tile_lds<C>(a.k), st, a, (int)tiles);
  return check_launch("mxfp4 product");
}

typedef MxTileShape<4, 4, 2, 2, 2> Tall;          // 128 x 128, four wavefronts of 64 x 64, three workgroups to a CU
typedef MxTileShape<4, 2, 1, 8, 3> Wide;          // 64 x 256, eight of 64 x 32, two to a CU
typedef MxTileShape<4, 2, 1, 4, 2> Middle;        // 64 x 128, four of 64 x 32, four to a CU
typedef MxTileShape<2, 2, 1, 4, 3> Small;         // 32 x 128

// Tall tiles where an expert's rows fill them: 2048 tokens of 32 experts, 256 rows each, mlp1 315 us (wide ones 349), 512 tokens 168 (149);
// 2048 rows of [5120, 2880] 62.7 (73.0). Small ones where the others would leave CUs without any: 300 rows of [5120, 2880] 30.2 in
// wide, 20.6 in small ones. Between tall and small, for one weight, middle ones where a CU gets one and a quarter to three (rows of [5120, 2880]
// in middle tiles and in what is chosen otherwise: 400, 280 tiles, 25.3 and 24.6; 512, 320, 26.1 and 29.9; 700 26.8 and 39.1; 1000
// 35.0 and 42.0; 1300, 840, 49.4 and 43.7; 700 of [8192, 2880], 704, 38.2 and 42.4; 2000 of [2880, 4096], 736, 52.5 and 57.2).
// Experts' rows have no use for them (512 tokens of 32 mlp1 166, wide ones 147; mlp2 110 and 100).
template <int MODE>
static int tiles_of(const MxArgs& a, hipStream_t st) {
  auto count = [&](int64_t bm, int64_t bn) { return (a.n + bn - 1) / bn * ((a.rows + bm - 1) / bm + (a.order ? a.experts / 2 : 0)); };
  auto fits = [&](int64_t lds) { return lds <= 160 * 1024; };
  if constexpr (MODE == kMxLinear) {
    const int64_t middle = count(64, 128);
    if (middle >= 320 && middle <= 768 && fits(tile_lds<Middle>(a.k))) return launch_tiles<Middle, MODE>(a, st);
  }
  if (a.rows > 128ll * a.experts && count(128, 128) >= 256 && fits(tile_lds<Tall>(a.k))) return launch_tiles<Tall, MODE>(a, st);
  if constexpr (MODE != kMxLinear)
    if (count(64, 256) >= 256 && fits(tile_lds<Wide>(a.k))) return launch_tiles<Wide, MODE>(a, st);
  return launch_tiles<Small, MODE>(a, st);
}

// Whether a product of these sizes is the tiles'. Below, the weight stream is ahead: 130 rows of [5120, 2880] 12.4 us, 16.4 in tiles,
// 200 16.8 and 19.2, 300 21.5 and 21.2; 32 experts of 24 rows each on average mlp1 113.3 and 113.8 in tiles, of 32 rows 129.4 and 120.5.
bool mx_tiles_take(const MxArgs& a) {
  return a.rows > (a.order ? 24ll : 200ll) * a.experts && tile_lds<Small>(a.k) <= 160 * 1024;
}

int mx_tiles(const MxArgs& a, int mode, hipStream_t st) {
  if (mode == kMxSwiglu) return tiles_of<kMxSwiglu>(a, st);
  if (mode == kMxPairs) return tiles_of<kMxPairs>(a, st);
  return tiles_of<kMxLinear>(a, st);
}

}  // namespace tllm
