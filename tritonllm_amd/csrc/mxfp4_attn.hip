// Attention over an MXFP4 KV cache with learned sinks and an optional sliding window, one or several new tokens per batch row:
//
//   query i of row b sits at p = start_q[b] + i and sees the slots n <= p, n < n_slots, n > p - window (when a window is set)
//   s[i, h, n] = sm_scale * <q[i, h], k[n, kv(h)]>                      kv(h) = h / G   (G query heads share a KV head)
//   out[i, h]  = sum_n exp(s - m) v[n, kv(h)] / (sum_n exp(s - m) + exp(sink[h] - m)),    m = max(sink[h], max_n s)
//
// with k and v the values that the cache's codes and scale bytes stand for, exactly (an e2m1 value times a power of two is a bf16 value).
// A scale byte of 255 makes its 32 values NaN, and values of 2^128 and more (scale bytes 253 and 254) are infinite in bf16: for the queries that see
// the slot, and for no other.
// Logits, sums, references and denominators are fp32. The weights are rounded to bf16 ahead of the second product, whose matrix instruction takes
// them so (at most 2^-8 of a weight, as in the kernels over a bf16 cache: results are 1.9e-3 - 2.1e-3 from the definition, of which 1.6e-3 - 1.7e-3 is
// the result's own rounding). Where many rows share a tile the denominator sums what they were rounded to, on the matrix cores; else the fp32 ones.
// Weighted values are summed ahead of the division, at weights of up to 2^8: values beyond 2^120 / (the keys seen) may pass fp32's range.
#include "mx_cache.h"

namespace tllm {

struct MxAttnArgs {
  const bf16* q;          // [B, n_q, n_heads, 64]: batch and token strides in elements, heads adjacent
  const bf16* sinks;      // [n_heads] or null (logit 0)
  bf16* out;              // [B, n_q, n_heads * 64]: batch and token strides
  float* part;            // [splits][B][n_q][n_heads][66]: acc[64], max, sum (when splits > 1)
  const void* start_q;
  int start_is_i64, start_stride;
  int64_t q_bs, q_ts, out_bs, out_ts;
  MxCache c;
  int batch, n_q, n_kv_heads, group, window;
  int row_groups;         // runs of rows (queries x heads of a KV head) that a workgroup takes
  int splits, fill, one;  // planned splits; workgroups a stream that fill the CUs; whether this is the kernel for one query
  float scale_log2;       // sm_scale * log2 e
  MxDiv by_group, by_heads, by_batch, by_row_groups, by_n_q;      // the latter two for the kernels that need them
};

namespace {
constexpr int PART = 66;              // floats of a record in the workspace
// Splits, one query of 8 heads, us (a line's figures are of one sweep in graphs; from one machine to another they differ by up to 5 %). One workgroup
// walks up to kUnsplit keys alone (no second launch): 300 keys 4.9, split 6.7; 600 5.7, 6.7; 1000 6.4, 6.8; 8 rows of 1024 6.4, 7.9; but 2000 9.0 and
// 6.8. A workgroup to a CU: 49 rows of up to 2048 11.9, with two 17.2; 32 of 4096 16.1, 19.2; one of 32768 11.2, 13.2 -- until each has 2^kMostShift
// keys: 8 rows of 32768 28.6, with one of 8192 31.6 and two of 2048 30.4; 8 of 131072 96, 94 and 104. At least 2^kLeastShift keys: one row of 4096
// 7.3, of 512 and more 7.6 - 9.0. (Eight wavefronts instead of four, with as many splits or half: 300 keys 5.4, 8 rows of 4096 10.5 and 11.7 against
// 10.1, 32 of 2048 10.5 against 10.2.)
constexpr int kUnsplit = 1024, kLeastShift = 8, kMostShift = 12, kFill = 256, kDeep = 4096;
constexpr float kLog2e = 1.4426950408889634f;
// Weights are exp2(logit - reference). The reference of one query and of a few rows is the largest logit that it was raised to, and stays there
// until a lane's weights of a block sum to more than kMostSum; that of many rows lies kLift above it, and stays until a weight reaches 2.
constexpr float kNoRef = -3.0e38f;    // no key has been seen (finite, so that a masked logit's weight is exp2(-inf); the first key's is infinite and raises it)
constexpr float kLift = 7.f;
constexpr float kMostSum = 256.f;
constexpr int kShare = 34 * 64;       // floats that a wavefront hands over for a tile of 32 rows
}  // namespace

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((__vector_size__(8 * sizeof(short)))) short i16x8;

// Context splits over `ctx` visible keys where `fill` workgroups a stream (or a run of rows) fill the CUs, by the rules above and at the plan below;
// at most 64. The host plans the launch with it from the size of the cache (or the caller's hint), the kernels evaluate it again with
// the length that they read.
__host__ __device__ inline int mx_attn_splits(bool one, int fill, int ctx) {
  const int cap = ((ctx - 1) >> kLeastShift) + 1, by_work = ((ctx - 1) >> kMostShift) + 1;
  int s = one ? (fill > by_work ? fill : by_work) : fill >= 4 || ctx > kDeep ? fill : 1;
  s = s < cap ? s : cap;
  s = s > 1 && ctx > kUnsplit ? s : 1;
  return s < 64 ? s : 64;
}

// The keys lo .. hi-1 that any of the rows first .. last of a batch row that starts at `start` sees, and the number of splits that take part.
struct MxSpan {
  int64_t start;
  int lo, hi, live;
};
__device__ __forceinline__ int64_t mx_start(const MxAttnArgs& a, int b) { return mx_row_int_ahead(a.start_q, a.start_is_i64, static_cast<int64_t>(b) * a.start_stride); }
__device__ __forceinline__ MxSpan mx_span(const MxAttnArgs& a, int64_t start, int first_row, int last_row) {
  MxSpan s;
  s.start = start;
  const int64_t far = 1ll << 40;                               // (beyond any slot; sums of it stay within 64 bits)
  s.start = s.start < -far ? -far : s.start > far ? far : s.start;
  const int q0 = a.n_q == 1 ? 0 : a.by_group(first_row), q1 = a.n_q == 1 ? 0 : a.by_group(last_row);
  int64_t hi = s.start + (q1 < a.n_q ? q1 : a.n_q - 1) + 1;
  hi = hi < 0 ? 0 : hi < a.c.n_slots ? hi : a.c.n_slots;
  int64_t lo = a.window > 0 ? s.start + q0 - a.window + 1 : 0;
  lo = lo < 0 ? 0 : lo < hi ? lo : hi;
  s.lo = static_cast<int>(lo);
  s.hi = static_cast<int>(hi);
  const int live = mx_attn_splits(a.one != 0, a.fill, hi > lo ? s.hi - s.lo : 1);
  s.live = live < a.splits ? live : a.splits;
  return s;
}

// A head's sink: asked for at a kernel's beginning (its latency would stand at the end), without a branch that would wait for it, and looked at
// at the end, as an exponent of two.
__device__ __forceinline__ bf16 mx_sink(const MxAttnArgs& a, int head) {
  const bf16* const p = a.sinks ? a.sinks : a.q;
  return p[a.sinks ? head : 0];
}

// What the weighted sum of a row's values is multiplied with: the sink joins the denominator. Nothing at all to attend to -- no key and a
// sink of -infinity -- gives zeros.
__device__ __forceinline__ float mx_norm(const MxAttnArgs& a, bf16 sink_of, float m, float l) {
  const float sink = a.sinks ? static_cast<float>(sink_of) * kLog2e : 0.f;
  const float top = fmaxf(m, sink);
  const float f = __builtin_amdgcn_exp2f(m - top);
  const float z = l * f + __builtin_amdgcn_exp2f(sink - top);
  return z == 0.f ? 0.f : f / z;
}

__device__ __forceinline__ float mx_power(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

// Values that are no number in bf16 -- NaN of scale byte 255, infinities of 254 (2 x 2^127 and more) and 253 (4 and 6 x 2^126) -- may not stand in a tile of
// V that several rows share: to a row that does not see the key they would be 0 x NaN or 0 x infinity. kFinite bytes have none.
constexpr unsigned kFinite = 252;
// Which of a dword's eight codes they are, in the low bit of each nibble; `byte` is beyond kFinite.
__device__ __forceinline__ unsigned mx_not_finite(unsigned codes, unsigned byte) {
  const unsigned two = codes >> 2, four = codes >> 2 & codes >> 1;      // (codes of a magnitude of 2 and more, of 4 and more)
  return 0x11111111u & (byte == 255u ? ~0u : byte == 254u ? two : four);
}
// Sixteen bytes of codes without them, and the scale byte for what stays.
__device__ __forceinline__ void mx_set_aside(u32x4* codes, unsigned* byte) {
  if (*byte <= kFinite) return;
#pragma unroll
  for (int w = 0; w < 4; ++w) (*codes)[w] &= ~(15u * mx_not_finite((*codes)[w], *byte));
  *byte = *byte == 255u ? 0u : *byte;
}
// What was set aside of the 32 values at `from`, for a row that sees them: its lane's sixteen, 8 (r / 4) + 4 h + r % 4. A weight above zero times an
// infinity is the infinity. The codes come once more from memory, so that no register waits for this, and by scalar loads: behind vector loads here
// the kernels would wait for the block that is on its way.
__device__ __forceinline__ void mx_add_aside(f32x16* o, const unsigned char* from, unsigned byte, int h) {
  const auto codes = (const __attribute__((address_space(4))) unsigned*)from;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const unsigned x = codes[w] >> 16 * h, aside = mx_not_finite(x, byte);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const unsigned bits = byte == 255u ? 0x7fc00000u : 0x7f800000u | (x >> 4 * r & 8u) << 28;
      (*o)[4 * w + r] += aside >> 4 * r & 1u ? __builtin_bit_cast(float, bits) : 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}
// Pieces (bits) with values that are set aside, and which of them have scale bytes of 255 and of 254.
struct MxAside {
  unsigned long long any, nan, large;
  __device__ __forceinline__ unsigned byte(int at) const { return nan >> at & 1 ? 255u : large >> at & 1 ? 254u : 253u; }
};

// Where 16 bytes (eight values) of a V tile's row are in LDS: rows of 128 bytes, their chunks XORed so that the transposing reads (eight
// rows x two chunks at a time) and the writes (eight rows x one chunk of either half) have every bank once.
__device__ __forceinline__ int mx_v_chunk(int key, int chunk) { return key * 128 + ((chunk ^ ((key >> 1 & 3) << 1) ^ (chunk >> 2)) << 4); }

// The same for tiles of 32 rows, whose transposing reads take four rows x four chunks at a time.
__device__ __forceinline__ int mx_v_chunk4(int key, int chunk) { return key * 128 + ((chunk ^ ((key >> 1 & 1) << 2) ^ (key >> 2 & 1) ^ (chunk >> 2 << 1)) << 4); }

// yes ? a : b for a condition that all lanes share, on a scalar mask in one instruction.
__device__ __forceinline__ unsigned mx_choose(bool yes, unsigned a, unsigned b) {
  unsigned x;
  asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(x) : "s"(yes ? ~0u : 0u), "v"(a), "v"(b));
  return x;
}

// The scale bytes of two neighbouring slots. DENSE: a head's lie next to each other (two bytes from slot to slot, at even addresses).
template <bool DENSE>
__device__ __forceinline__ unsigned mx_scale_pair(const unsigned char* p, int64_t sts, int behind) {
  typedef unsigned __attribute__((aligned(2))) u32_a2;
  if constexpr (DENSE) {
    return *reinterpret_cast<const u32_a2*>(p);
  } else {
    const unsigned char* const q = behind > 0 ? p + sts : p;   // (two single bytes each: a slot's may lie anywhere)
    return p[0] | p[1] << 8 | q[0] << 16 | static_cast<unsigned>(q[1]) << 24;
  }
}

// One query of up to eight heads. A wavefront takes 64 keys at a time: keys 0 - 31 and 32 - 63 of a block are dealt to the two halves of the
// matrix instruction's sixteen columns, so that eight heads fill it.
//   S^T = K . Q^T, keys on M, in two tiles of 16 x 2 keys: the k slots of the lane groups g = 0, 1 are a key's two blocks of 32 values, those of
//   g = 2, 3 the key 32 places on; the columns 0 - 7 have Q in the former and zeros in the latter, the columns 8 - 15 the reverse.
//   A lane's scores are then four of a tile, all of use.
//   O = P . V, the weights' registers being the A operand for the block's keys 0 - 31 in the rows 0 - 7 and for 32 - 63 in the rows 8 - 15: two
//   accumulators, each of which is looked at in one half of its rows. V passes LDS as bf16, for transposing reads.
// Bound by the cache's bytes where contexts are long -- in a graph, 8 rows of 32768 keys 28.2 us (143 MB, 5.1 TB/s, the joining launch among them), of
// 131072 96 - 98 (5.9 TB/s; loads of this pattern alone 6.8) --, else by a chain of latencies: 300 keys of one row planned for 300 4.7 us, 8 rows of
// 4096 9.7, about 2 of which are the second launch, a window of 128 keys 4.2 (the start position comes ahead of the first keys there).
template <bool DENSE>
__global__ __launch_bounds__(256, 3) void mxfp4_attn_one_kernel(MxAttnArgs a) {
  constexpr int NW = 4;                                        // wavefronts
  constexpr int VTILE = 64 * 128;
  constexpr int AROW = 64 + 1;                                 // accumulator row in LDS, floats
  __shared__ __align__(16) unsigned char vt[NW * VTILE];
  __shared__ float s_m[NW][16], s_l[NW][16];
  static_assert(16 * AROW * 4 <= VTILE, "an accumulator fits a tile");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;

  // the splits are the slowest part of the index: those that a context does not need are the last
  const int id = a.by_heads(blockIdx.x), kvh = blockIdx.x - id * a.n_kv_heads;
  const int split = a.by_batch(id), b = id - split * a.batch;
  const int G = a.group;

  bf16x8 qf[4];
  {
    const int head = kvh * G + ((r16 & 7) < G ? r16 & 7 : G - 1);                  // (columns beyond the group repeat its last head; never stored)
    const bf16* const qr = a.q + b * a.q_bs + head * 64 + 32 * (g & 1);
    const bool mine = (g >> 1) == (r16 >> 3);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(qr + 8 * t);
      qf[t] = __builtin_bit_cast(bf16x8, mine ? w : u32x4{0u, 0u, 0u, 0u});
    }
  }
  // Without a window the keys begin at slot 0 and the wavefront's first block is known ahead of the start position, whose load takes as long as
  // the block's own: it is asked for at once (and not looked at where the context turns out to be shorter).
  int lo = 0;
  if (a.window > 0) lo = min(mx_span(a, mx_start(a, b), 0, 0).lo, a.c.n_slots - 1);      // (a slot of the cache, also where a window behind its end has none)
  const int first = split * NW + wave;
  constexpr int TPR = NW * 64 / 8, DPT = 64 / TPR;             // at the end: thread -> (head, every TPR-th of its 64 values)
  const int eh = tid / TPR, ed = tid % TPR;
  const bf16 sink = mx_sink(a, kvh * G + (eh < G ? eh : G - 1));
  const int nall = (a.c.n_slots - lo + 63) >> 6;                // blocks that the cache has from there on

  const int64_t kv_off = b * a.c.bs + kvh * a.c.hs + lo * a.c.ts, sc_off = b * a.c.sbs + kvh * a.c.shs + lo * a.c.sts;
  const unsigned char *const kp = a.c.blocks[0] + kv_off, *const vp = a.c.blocks[1] + kv_off;
  const unsigned char *const ksp = a.c.scales[0] + sc_off, *const vsp = a.c.scales[1] + sc_off;
  unsigned char* const vtile = vt + wave * VTILE;

  // Loads: 32 keys' codes at a time, 16 bytes a lane as they lie in memory (a CU's cache serves four neighbouring lanes' 64 bytes in one access, and
  // lanes whose pieces lie apart one by one); the scale bytes of 64 keys and 64 values in one load, two keys' to a lane. K's codes go
  // through LDS into the operand's order, scale bytes from lane to lane.
  // Behind the last slot of the cache rows are held to the last one (whose pair of keys ends with it).
  const int64_t blk_bytes = 64 * a.c.ts, blk_scales = 64 * a.c.sts;
  const int slots = a.c.n_slots - lo - 64 * (nall - 1);         // in the last one of them
  const unsigned char* const sbase = (lane < 32 ? ksp : vsp) - 2;      // (two bytes ahead, so that offsets from it are positive)
  unsigned off[2][2];                                          // [whole, last]: rows lane / 2 and 32 + lane / 2
  unsigned soff[2];
  const int pair = 2 * (lane & 31);
  {
    const unsigned ts = static_cast<unsigned>(a.c.ts);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = 32 * t + (lane >> 1);
      off[0][t] = static_cast<unsigned>(r) * ts + 16 * (lane & 1);
      off[1][t] = static_cast<unsigned>(min(r, slots - 1)) * ts + 16 * (lane & 1);
    }
    soff[0] = pair * static_cast<unsigned>(a.c.sts) + 2;
    soff[1] = (DENSE ? min(pair, slots - 2) : min(pair, slots - 1)) * static_cast<int>(a.c.sts) + 2;
  }
  const int pair_shift = DENSE && pair == slots - 1 ? 16 : 0;  // (in the last block)
  struct Block {
    u32x4 k[2], v[2];
    unsigned s;
  };
  auto load_block = [&](int at, Block& r) __attribute__((always_inline)) {
    const int blk = at < nall ? at : nall - 1;                 // (a block that is not there: any)
    const unsigned char *const kb = kp + blk * blk_bytes, *const vb = vp + blk * blk_bytes;
    const bool end = blk == nall - 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned x = mx_choose(end, off[1][t], off[0][t]);
      r.k[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb + x));
      r.v[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vb + x));
    }
    r.s = mx_scale_pair<DENSE>(sbase + blk * blk_scales + mx_choose(end, soff[1], soff[0]), a.c.sts, end ? slots - 1 - pair : 1);
  };
  Block even, odd;
  load_block(first, even);
  __builtin_amdgcn_sched_barrier(0);                           // (in the loop's order, so that it can wait for the one and not the other)
  const MxSpan sp = mx_span(a, mx_start(a, b), 0, 0);
  if (split >= sp.live) return;
  const int len = sp.hi - sp.lo, nblk = (len + 63) >> 6, step = sp.live * NW;      // the stream's wavefronts take its blocks in turn
  load_block(first + step, odd);
  __builtin_amdgcn_sched_barrier(0);
  // where the lane's 64 bytes of V go, and where the transposing reads want them from: within 16 lanes, lane 4 r + c has the address of four d
  // (quad c of sixteen) of key r and gets one d (its own of the sixteen) of the four keys
  unsigned char* const v_to = vtile + (lane >> 1) * 128;
  int v_chunk[4], v_from[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) v_chunk[t] = mx_v_chunk(lane >> 1, 4 * (lane & 1) + t) - (lane >> 1) * 128;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) v_from[nb] = mx_v_chunk(4 * g + (r16 >> 2), 2 * nb + (r16 >> 1 & 1)) + (r16 & 1) * 8;

  // K's codes in the operand's order: tile t, lane (key 16 t + r16 + 32 (g / 2), block g % 2). Scale bytes: a lane of the load has four, of two
  // neighbouring slots; lanes 0 - 31 keys', 32 - 63 values'.
  const int k_from = (r16 + 32 * (g >> 1)) * 32 + 16 * (g & 1);
  const int k_lane = 4 * ((r16 + 32 * (g >> 1)) >> 1), k_shift = 16 * (r16 & 1) + 8 * (g & 1);
  const int v_lane = 4 * (32 + (lane >> 2)), v_shift = 8 * (lane & 3);

  float ref = kNoRef, l_run = 0.f;                             // of column r16 (the sum: this lane's share of it)
  f32x4 acc[2][4];                                             // [half of the keys]; lane (d = 16 nb + r16, rows 4 g + i)
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[h][nb] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A block's arithmetic; in its middle the block after the next is asked for (unconditionally: also one behind the last that is looked at).
  auto process = [&](int blk, Block& r) __attribute__((always_inline)) {
    const bool end = blk == nblk - 1;
    // K's codes through LDS; the tile of V follows in the same place (a wavefront's LDS operations stay in order)
#pragma unroll
    for (int t = 0; t < 2; ++t) *reinterpret_cast<u32x4*>(vtile + 1024 * t + 16 * lane) = r.k[t];
    const unsigned pairs = blk == nall - 1 ? r.s >> pair_shift : r.s;
    unsigned ks[2], vs[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ks[t] = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(k_lane + 32 * t, static_cast<int>(pairs))) >> k_shift & 255u;
      vs[t] = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(v_lane + 64 * t, static_cast<int>(pairs))) >> v_shift & 255u;
    }
    u32x4 kc[2], vc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      kc[t] = *reinterpret_cast<const u32x4*>(vtile + k_from + 512 * t);
      vc[t] = r.v[t];
    }
    if (__builtin_expect(end, 0)) {                            // what lies behind the last key may be anything: zeros
      const int left = len - 64 * blk;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool k_in = 16 * t + r16 + 32 * (g >> 1) < left, v_in = 32 * t + (lane >> 1) < left;
        kc[t] = k_in ? kc[t] : u32x4{0u, 0u, 0u, 0u};
        ks[t] = k_in ? ks[t] : 0u;
        vc[t] = v_in ? vc[t] : u32x4{0u, 0u, 0u, 0u};
        vs[t] = v_in ? vs[t] : 0u;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) *reinterpret_cast<bf16x8*>(v_to + 4096 * t + v_chunk[w]) = mx_bf16x8(vc[t][w], mx_power(vs[t]));
    f32x4 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_bf16x8(kc[t][w], mx_power(ks[t])), qf[w], st[t], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // half of V on its way while the weights are made (8 rows of 4096 9.9 -> 9.7 us, 49 of up to 2048 11.9 -> 11.6; all of it takes the registers of a
    // third wavefront)
    bf16x8 vf[2][4];
    auto read_v = [&](int h) __attribute__((always_inline)) {
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        i16x4 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(vtile + v_from[nb] + 4096 * h + 2048 * u));
        vf[h][nb] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    read_v(0);
    load_block(blk + 2 * step, r);

    // ---- weights: this lane has keys 16 t + 4 g + i of its half of the block
    float sc[8], p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sc[j] = st[j >> 2][j & 3];
    if (end) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = 64 * blk + 16 * (j >> 2) + 4 * g + (j & 3) + 32 * (r16 >> 3) < len ? sc[j] : -INFINITY;
    }
    auto weights = [&]() __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(fmaf(sc[j], a.scale_log2, -ref));
        sum += p[j];
      }
      return sum;
    };
    float sum = weights();
    // The reference -- the largest logit, when it was last raised -- is raised only where a lane's weights have outgrown it.
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum > kMostSum) != 0, 0)) {
      float top = sc[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, sc[j]);
      top = max_over_lane_bits_16_32(top) * a.scale_log2;
      const float moved = top > ref ? top : ref;
      const float alpha = __builtin_amdgcn_exp2f(ref - moved);
      ref = moved;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float al = __shfl(alpha, 4 * g + i, 64);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) acc[h][nb][i] *= al;
      }
      // (pinned as whole registers: the copies that join the two paths stay in this one)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) asm volatile("" : "+v"(acc[h][nb]));
      sum = weights();
    }
    l_run += sum;
    bf16x8 pa;                                                 // A operand of P . V: k slot j <-> key 4 g + j (j < 4), 16 + 4 g + j - 4 of the half
#pragma unroll
    for (int j = 0; j < 8; ++j) pa[j] = static_cast<bf16>(p[j]);
    read_v(1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) acc[h][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa, vf[h][nb], acc[h][nb], 0, 0, 0);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  int blk = first;
  for (; blk + step < nblk; blk += 2 * step) {
    process(blk, even);
    process(blk + step, odd);
  }
  if (blk < nblk) process(blk, even);

  // ---- the wavefronts meet: sixteen columns of each, the heads over either half of the keys
  const float l = sum_over_lane_bits_16_32(l_run);
  if (g == 0) {
    s_m[wave][r16] = ref;
    s_l[wave][r16] = l;
  }
  float* const mine = reinterpret_cast<float*>(vtile);         // (this wavefront is past its last read of the tile)
#pragma unroll
  for (int nb = 0; nb < 4; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = acc[0][nb][i], y = acc[1][nb][i];
      mine[(4 * g + i) * AROW + 16 * nb + r16] = g < 2 ? x : y;
    }
  __syncthreads();
  if (eh >= G) return;
  float m_all = kNoRef;
#pragma unroll
  for (int w = 0; w < 2 * NW; ++w) m_all = fmaxf(m_all, s_m[w >> 1][8 * (w & 1) + eh]);
  float l_all = 0.f, o[DPT] = {};
#pragma unroll
  for (int w = 0; w < 2 * NW; ++w) {
    const int row = 8 * (w & 1) + eh;
    const float f = __builtin_amdgcn_exp2f(s_m[w >> 1][row] - m_all);      // (0 for a wavefront that saw no key)
    l_all += s_l[w >> 1][row] * f;
    const float* const from = reinterpret_cast<const float*>(vt + (w >> 1) * VTILE) + row * AROW + ed;
#pragma unroll
    for (int j = 0; j < DPT; ++j) o[j] += from[TPR * j] * f;
  }
  const int head = kvh * G + eh;
  if (sp.live > 1) {
    float* const p = a.part + ((static_cast<int64_t>(split) * a.batch + b) * (a.n_kv_heads * G) + head) * PART;
#pragma unroll
    for (int j = 0; j < DPT; ++j) p[ed + TPR * j] = o[j];
    if (ed == 0) {
      p[64] = m_all;
      p[65] = l_all;
    }
    return;
  }
  const float f = mx_norm(a, sink, m_all, l_all);
  bf16* const to = a.out + b * a.out_bs + head * 64;
#pragma unroll
  for (int j = 0; j < DPT; ++j) to[ed + TPR * j] = static_cast<bf16>(o[j] * f);
}

// RT tiles of 32 of the rows r = query * G + head of a KV head, 32 keys at a time. The KG wavefronts of a workgroup share the keys and meet in
// LDS at the end.
//   S^T = K . Q^T on 32 x 32 x 16, keys on M: lanes l and l + 32 have the two blocks of 32 values of key l, 16 bytes of codes and a scale byte as
//   they lie in the cache, and a lane owns one row (column) with 16 of the 32 keys, so that maximum, sum and rescaling are its own but for
//   one exchange between the halves of the wavefront.
//   O^T = V^T . P^T: the scores' registers are, pairwise, the B operand when the k slots are read as a permutation of the keys; V passes LDS
//   as bf16 for transposing reads, as above.
// Bound by the vector ALU (a wavefront converts its keys and values for its own rows alone, an exponential for each weight) beside the matrix cores
// where there is enough to do -- 512 queries behind 4000 tokens 48 - 49 us, 36 GFLOP: 0.7 PFLOP/s --, else by latencies as above: four drafts to each of
// 8 rows of 4096 12.4 us, 97 behind 1500 9.7, one query of sixteen heads a KV head 8 x 4096 11.5 (all in graphs).
template <bool DENSE, int RT, int KG>
__global__ __launch_bounds__(KG * 64, 2) void mxfp4_attn_rows_kernel(MxAttnArgs a) {
  constexpr int RB = 32 * RT;                                  // rows
  constexpr int VTILE = 32 * 128;
  static_assert(kShare * 4 >= VTILE, "the shares are what needs most LDS");
  extern __shared__ __align__(16) unsigned char smem[];        // KG shares

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;

  // the splits are the slowest part of the index: those that a context does not need are the last
  const int i0 = a.by_heads(blockIdx.x), kvh = blockIdx.x - i0 * a.n_kv_heads;
  const int i1 = a.by_batch(i0), b = i0 - i1 * a.batch;
  const int split = a.by_row_groups(i1), rg = a.row_groups - 1 - (i1 - split * a.row_groups);
  const int rows = a.n_q * a.group, row0 = rg * RB;

  bf16x8 qf[RT][4];
  int query[RT], head[RT];
  bf16 sink[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int row = row0 + 32 * rt + l31;
    row = row < rows ? row : rows - 1;                         // (rows that are not there repeat the last one; never stored)
    query[rt] = a.by_group(row);
    head[rt] = kvh * a.group + row - query[rt] * a.group;
    sink[rt] = mx_sink(a, head[rt]);
    const bf16* const qr = a.q + b * a.q_bs + query[rt] * a.q_ts + head[rt] * 64 + 32 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t) qf[rt][t] = *reinterpret_cast<const bf16x8*>(qr + 8 * t);
  }

  // Without a window the keys begin at slot 0, and the first block is asked for ahead of the start position (whose load takes as long as its own).
  int lo = 0;
  if (a.window > 0) lo = min(mx_span(a, mx_start(a, b), row0, row0 + RB - 1).lo, a.c.n_slots - 1);
  const int first = split * KG + wave;
  const int nall = (a.c.n_slots - lo + 31) >> 5;                // blocks that the cache has from there on

  const int64_t kv_off = b * a.c.bs + kvh * a.c.hs + lo * a.c.ts, sc_off = b * a.c.sbs + kvh * a.c.shs + lo * a.c.sts;
  const unsigned char *const kp = a.c.blocks[0] + kv_off, *const vp = a.c.blocks[1] + kv_off;
  const unsigned char *const ksp = a.c.scales[0] + sc_off, *const vsp = a.c.scales[1] + sc_off;
  unsigned char* const vtile = smem + wave * VTILE;

  // Loads as above: 32 keys' codes, 16 bytes a lane as they lie in memory, and in one load the scale bytes of two neighbouring slots to a lane,
  // keys' in lanes 0 - 15, values' in 16 - 31 (and the same in the other 32).
  const int64_t blk_bytes = 32 * a.c.ts, blk_scales = 32 * a.c.sts;
  const int slots = a.c.n_slots - lo - 32 * (nall - 1);         // in the last one of them
  const unsigned char* const sbase = (lane & 16 ? vsp : ksp) - 2;
  const int pair = 2 * (lane & 15);
  unsigned off[2];                                             // [whole, last]
  unsigned soff[2];
  off[0] = static_cast<unsigned>(lane >> 1) * static_cast<unsigned>(a.c.ts) + 16 * (lane & 1);
  off[1] = static_cast<unsigned>(min(lane >> 1, slots - 1)) * static_cast<unsigned>(a.c.ts) + 16 * (lane & 1);
  soff[0] = pair * static_cast<unsigned>(a.c.sts) + 2;
  soff[1] = (DENSE ? min(pair, slots - 2) : min(pair, slots - 1)) * static_cast<int>(a.c.sts) + 2;
  const int pair_shift = DENSE && pair == slots - 1 ? 16 : 0;  // (in the last block)
  struct Block {
    u32x4 k, v;
    unsigned s;
  };
  auto load_block = [&](int at, Block& r) __attribute__((always_inline)) {
    const int blk = at < nall ? at : nall - 1;                 // (a block that is not there: any)
    const bool end = blk == nall - 1;
    const unsigned x = mx_choose(end, off[1], off[0]);
    r.k = *reinterpret_cast<const u32x4*>(kp + blk * blk_bytes + x);
    r.v = *reinterpret_cast<const u32x4*>(vp + blk * blk_bytes + x);
    r.s = mx_scale_pair<DENSE>(sbase + blk * blk_scales + mx_choose(end, soff[1], soff[0]), a.c.sts, end ? slots - 1 - pair : 1);
  };
  Block even, odd;
  load_block(first, even);
  __builtin_amdgcn_sched_barrier(0);                           // (in the loop's order, so that it can wait for the one and not the other)
  const MxSpan sp = mx_span(a, mx_start(a, b), row0, row0 + RB - 1);
  if (split >= sp.live) return;
  const int len = sp.hi - sp.lo, nblk = (len + 31) >> 5, step = sp.live * KG;
  load_block(first + step, odd);
  __builtin_amdgcn_sched_barrier(0);

  int upper[RT], lower[RT];                                    // the keys that the lane's row sees, counted from sp.lo
  int seen_hi, seen_lo;                                        // keys that every row of the wavefront sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t up = sp.start + query[rt] - sp.lo, low = up - a.window + 1;
    upper[rt] = static_cast<int>(up < -1 ? -1 : up < len - 1 ? up : len - 1);
    lower[rt] = static_cast<int>(a.window == 0 || low < 0 ? 0 : low < len ? low : len);
  }
  {
    const int q0 = a.by_group(row0), q1r = a.by_group(row0 + RB - 1), q1 = q1r < a.n_q ? q1r : a.n_q - 1;
    const int64_t up = sp.start + q0 - sp.lo, low = sp.start + q1 - sp.lo - a.window + 1;
    seen_hi = static_cast<int>(up < -1 ? -1 : up < len - 1 ? up : len - 1);
    seen_lo = static_cast<int>(a.window == 0 || low < 0 ? 0 : low < len ? low : len);
  }

  // K's codes pass LDS into the operand's order, lane (key l31, block h); the keys 16 - 31 have their blocks the other way round there, for the banks
  const int k_to = 16 * (lane ^ (lane >> 5)), k_from = l31 * 32 + 16 * (h ^ (l31 >> 4));
  const int k_lane = 4 * (l31 >> 1), k_shift = 16 * (l31 & 1) + 8 * h, v_lane = 4 * (16 + (lane >> 2)), v_shift = 8 * (lane & 3);
  unsigned char* const v_to = vtile + (lane >> 1) * 128;
  int v_chunk[4], v_from[2];
#pragma unroll
  for (int t = 0; t < 4; ++t) v_chunk[t] = mx_v_chunk4(lane >> 1, 4 * (lane & 1) + t) - (lane >> 1) * 128;
  // V^T fragment (A operand of O^T): lane = d; lane j of each 16 has the address of four d (quad j % 4 of the lane group's sixteen) of key j / 4 of
  // the four that this half of the wavefront takes
#pragma unroll
  for (int db = 0; db < 2; ++db) v_from[db] = mx_v_chunk4(4 * h + ((lane & 15) >> 2), 4 * db + 2 * (l31 >> 4) + (lane >> 1 & 1)) + (lane & 1) * 8;      // + 8 keys u, + 16 keys cc

  float ref[RT], l_run[RT];
  f32x16 o[RT][2];
  const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    ref[rt] = kNoRef;
    l_run[rt] = 0.f;
    o[rt][0] = zero;
    o[rt][1] = zero;
  }

  // A block's arithmetic; in its middle the block after the next is asked for.
  auto process = [&](int blk, Block& r) __attribute__((always_inline)) {
    const int k0 = 32 * blk;
    const bool end = blk == nblk - 1;
    // K's codes through LDS; the tile of V follows in the same place (a wavefront's LDS operations stay in order)
    *reinterpret_cast<u32x4*>(vtile + k_to) = r.k;
    const unsigned pairs = blk == nall - 1 ? r.s >> pair_shift : r.s;
    const unsigned ks = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(k_lane, static_cast<int>(pairs))) >> k_shift & 255u;
    unsigned vs = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(v_lane, static_cast<int>(pairs))) >> v_shift & 255u;
    const u32x4 kc = *reinterpret_cast<const u32x4*>(vtile + k_from);
    u32x4 vc = r.v;
    // ---- V into the wavefront's tile, as bf16
    // What lies behind the last key may be anything: zeros. What only some of the rows may see is set aside as zeros and added behind (rare). (A
    // key's NaN or infinity goes no further than its own scores.)
    if (__builtin_expect(end, 0)) {
      const bool in = k0 + (lane >> 1) < len;
      vc = in ? vc : u32x4{0u, 0u, 0u, 0u};
      vs = in ? vs : 0u;
    }
    MxAside aside{__builtin_amdgcn_ballot_w64(vs > kFinite), 0, 0};
    if (__builtin_expect(aside.any != 0, 0)) {
      aside.nan = __builtin_amdgcn_ballot_w64(vs == 255u);
      aside.large = __builtin_amdgcn_ballot_w64(vs == 254u);
      mx_set_aside(&vc, &vs);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) *reinterpret_cast<bf16x8*>(v_to + v_chunk[w]) = mx_bf16x8(vc[w], mx_power(vs));
    // ---- S^T
    f32x16 s[RT];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bf16x8 kf = mx_bf16x8(kc[t], mx_power(ks));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[rt][t], t == 0 ? zero : s[rt], 0, 0, 0);
    }
    load_block(blk + 2 * step, r);

    const bool masked = k0 + 31 > seen_hi || k0 < seen_lo;
    u32x4 p[RT][2];                                            // P^T in bf16, as operand registers
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (__builtin_expect(masked, 0)) {
        int du = upper[rt] - k0 - 4 * h, dl = lower[rt] - k0 - 4 * h;
        asm volatile("" : "+v"(du), "+v"(dl));                 // (or the comparisons are made for every block)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[rt][r] = 8 * (r >> 2) + (r & 3) <= du && 8 * (r >> 2) + (r & 3) >= dl ? s[rt][r] : -INFINITY;
      }
      auto weights = [&]() __attribute__((always_inline)) {
        float sum = 0.f;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[rt][2 * m], a.scale_log2, -ref[rt])), y = __builtin_amdgcn_exp2f(fmaf(s[rt][2 * m + 1], a.scale_log2, -ref[rt]));
          sum += x + y;
          const bf16x2 v = {static_cast<bf16>(x), static_cast<bf16>(y)};
          p[rt][m >> 2][m & 3] = __builtin_bit_cast(unsigned, v);
        }
        return sum;
      };
      float sum = weights();
      // The reference -- the largest logit, when it was last raised -- is raised only where a lane's weights have outgrown it.
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum > kMostSum) != 0, 0)) {
        float top = s[rt][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[rt][r]);
        float x, y;
        lane_xor32_pair(top, &x, &y);
        top = fmaxf(x, y) * a.scale_log2;
        const float moved = top > ref[rt] ? top : ref[rt];
        const float alpha = __builtin_amdgcn_exp2f(ref[rt] - moved);
        ref[rt] = moved;
        l_run[rt] *= alpha;
#pragma unroll
        for (int db = 0; db < 2; ++db) {
          asm volatile("" : "+v"(o[rt][db]));
#pragma unroll
          for (int r = 0; r < 16; ++r) o[rt][db][r] *= alpha;
          asm volatile("" : "+v"(o[rt][db]));
        }
        sum = weights();
      }
      l_run[rt] += sum;
    }
    // ---- O^T += V^T . P^T
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        i16x4 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(vtile + v_from[db] + 2048 * cc + 1024 * u));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, __builtin_bit_cast(bf16x8, p[rt][cc]), o[rt][db], 0, 0, 0);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (__builtin_expect(aside.any != 0, 0)) {
      for (unsigned long long left = aside.any; left != 0; left &= left - 1) {
        const int at = __builtin_ctzll(left), key = k0 + (at >> 1);         // (one of the span's)
        const unsigned char* const from = vp + key * a.c.ts + 16 * (at & 1);
        const unsigned byte = aside.byte(at);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if (key >= lower[rt] && key <= upper[rt]) {
            if (at & 1) mx_add_aside(&o[rt][1], from, byte, h);
            else mx_add_aside(&o[rt][0], from, byte, h);
          }
      }
    }
  };
  if (first < nblk) {
    int blk = first;
    for (; blk + step < nblk; blk += 2 * step) {
      process(blk, even);
      process(blk + step, odd);
    }
    if (blk < nblk) process(blk, even);
  }

  // ---- the sink joins the denominator, or a record leaves. A lane has 16-byte runs of one row's values; the wavefronts,
  // which share the rows, meet in LDS: 32 / KG of the 32 values a lane to each.
  constexpr int RPG = 32 / KG;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float l, m = ref[rt];
    {
      float x, y;
      lane_xor32_pair(l_run[rt], &x, &y);
      l = x + y;
    }
    float v[RPG];
    float* const shares = reinterpret_cast<float*>(smem);
    __syncthreads();                                         // (all are past their last read of the tiles, or of the tile of rows before)
    float* const mine = shares + wave * kShare + lane;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const float x = o[rt][r >> 4][r & 15];
      mine[r * 64] = x;
    }
    mine[32 * 64] = m;
    mine[33 * 64] = l;
    __syncthreads();
    const float* const from = shares + lane;
    m = kNoRef;
#pragma unroll
    for (int k = 0; k < KG; ++k) m = fmaxf(m, from[k * kShare + 32 * 64]);
    l = 0.f;
#pragma unroll
    for (int r = 0; r < RPG; ++r) v[r] = 0.f;
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      const float f = __builtin_amdgcn_exp2f(from[k * kShare + 32 * 64] - m);      // (0 for a wavefront that saw no key)
      l = fmaf(from[k * kShare + 33 * 64], f, l);
#pragma unroll
      for (int r = 0; r < RPG; ++r) v[r] = fmaf(from[k * kShare + (RPG * wave + r) * 64], f, v[r]);
    }
    if (row0 + 32 * rt + l31 >= rows) continue;
    // value rr = RPG wave + r: d = 32 (rr / 16) + 8 (rr / 4 % 4) + 4 h + rr % 4
    if (sp.live > 1) {
      float* const p = a.part + (((static_cast<int64_t>(split) * a.batch + b) * a.n_q + query[rt]) * (a.n_kv_heads * a.group) + head[rt]) * PART;
#pragma unroll
      for (int r = 0; r < RPG; ++r) {
        const int rr = RPG * wave + r;
        p[32 * (rr >> 4) + 8 * (rr >> 2 & 3) + 4 * h + (rr & 3)] = v[r];
      }
      if (wave == 0) p[64 + h] = h == 0 ? m : l;
      continue;
    }
    const float f = mx_norm(a, sink[rt], m, l);
    bf16* const to = a.out + b * a.out_bs + query[rt] * a.out_ts + head[rt] * 64;
#pragma unroll
    for (int r = 0; r < RPG; r += 4) {
      const int rr = RPG * wave + r;
      bf16x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<bf16>(v[r + e] * f);
      *reinterpret_cast<bf16x4*>(to + 32 * (rr >> 4) + 8 * (rr >> 2 & 3) + 4 * h) = w;
    }
  }
}

// Many rows: a workgroup's wavefronts have 64 neighbouring rows each, RUNS of them walk the same keys, and these come to bf16 once for all of
// them: a thread has 16 bytes of codes of a unit of 16 RUNS keys, and writes their 32 values into one of three stages in LDS while the
// units before are worked on. One barrier a unit. Four runs, or two with two groups of wavefronts that take the units in turn and meet at the end.
//   The matrix cores and the vector ALU work at the same time: with one tile's weights (32 keys x 32 rows) the next one's scores are issued in
//   turn, and the products of the one before. Of block j (32 keys), S^T of tile 1, weights of tile 0 and P . V of block j - 1 in tile 1; then S^T of
//   block j + 1 in tile 0, weights of tile 1 and P . V of tile 0. Operands of K and of V live from one such half to the next.
// Bound by what the two units take together at the clock that the power limit leaves (1.8 - 1.9 GHz): a prompt of 8192 513 - 536 us (550 GFLOP: 1.0 -
// 1.07 PFLOP/s; 431 with the LDS traffic left out); of 2048 47.5 - 48.8 (0.7), of which a workgroup's beginning and end are 4 each.
template <int RUNS, int KG>
__global__ __launch_bounds__(RUNS * KG * 64, 2) void mxfp4_attn_many_kernel(MxAttnArgs a) {
  static_assert(RUNS == 4 || RUNS == 2, "runs of a workgroup");
  constexpr int UNIT = 16 * RUNS, HALVES = UNIT / 32, RB = 64 * RUNS;
  constexpr int KTILE = UNIT * 128, STAGE = 2 * KTILE;         // bytes: K [UNIT keys][64 values], then V
  __shared__ __align__(16) unsigned char smem[KG * 3 * STAGE];
  __shared__ __align__(8) unsigned s_any[KG][3][2];            // whether a stage's values hold NaN or infinities, by 32 keys,
  __shared__ MxAside s_aside[KG][3][2];                        // and (where they do) in which of the 32 x 2 pieces
  static_assert(KG == 1 || RUNS * 2 * kShare * 4 <= KG * 3 * STAGE, "the shares fit the stages");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int run = wave % RUNS, kg = wave / RUNS;

  // the rows that see most keys come first, and where the launch is two workgroups to a CU the second ones are taken in the opposite order, so
  // that a CU with a long walk gets a short one next to it
  unsigned id = a.by_heads(blockIdx.x);
  const int kvh = blockIdx.x - id * a.n_kv_heads;
  {
    const unsigned per_round = a.n_kv_heads < 256 ? a.by_heads(256) : 1, n = a.by_heads(gridDim.x);
    if (RUNS * KG == 4 && n <= 2 * per_round && id >= per_round) id = n + per_round - 1 - id;
  }
  const int i1 = a.by_batch(id), b = id - i1 * a.batch, rg = a.row_groups - 1 - i1;
  const int rows = a.n_q * a.group, row0 = rg * RB + run * 64;

  // Without a window the keys begin at slot 0, and the first unit is asked for ahead of the start position (whose load takes as long as its own).
  int lo = 0;
  if (a.window > 0) lo = min(mx_span(a, mx_start(a, b), rg * RB, rg * RB + RB - 1).lo, a.c.n_slots - 1);
  const int nall = (a.c.n_slots - lo + UNIT - 1) / UNIT;       // units that the cache has from there on
  // ---- the movers
  const int kv = run / (RUNS / 2), piece = tid & (UNIT * 2 - 1);      // 0: keys, 1: values; (key piece / 2, block piece % 2) of a unit
  const unsigned char* const src = a.c.blocks[kv] + b * a.c.bs + kvh * a.c.hs + lo * a.c.ts + 16 * (piece & 1);
  const unsigned char* const ssrc = a.c.scales[kv] + b * a.c.sbs + kvh * a.c.shs + lo * a.c.sts + (piece & 1);
  const int64_t unit_bytes = UNIT * a.c.ts, unit_scales = UNIT * a.c.sts;
  const unsigned off = (piece >> 1) * static_cast<unsigned>(a.c.ts), soff = (piece >> 1) * static_cast<unsigned>(a.c.sts);
  const int at_end = min(piece >> 1, (a.c.n_slots - lo - 1) & (UNIT - 1));      // behind the last slot of the cache rows are held to it
  const unsigned off_end = at_end * static_cast<unsigned>(a.c.ts), soff_end = at_end * static_cast<unsigned>(a.c.sts);
  unsigned to[4];                                              // where the piece's four chunks of 16 bytes go
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int key = piece >> 1, c = 4 * (piece & 1) + t;
    to[t] = kv == 0 ? key * 128 + ((c ^ (key >> 1 & 7)) << 4) : KTILE + mx_v_chunk4(key, c);
  }
  u32x4 raw;
  unsigned raw_s;
  auto load_unit = [&](int u) __attribute__((always_inline)) {
    const int v = min(KG * u + kg, nall - 1);                  // (one that is not there: any)
    const bool end = v == nall - 1;
    raw = *reinterpret_cast<const u32x4*>(src + v * unit_bytes + mx_choose(end, off_end, off));
    raw_s = (ssrc + v * unit_scales)[mx_choose(end, soff_end, soff)];
  };
  load_unit(0);
  __builtin_amdgcn_sched_barrier(0);

  int query[2];
  bf16 sink[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    int row = row0 + 32 * rt + l31;
    row = row < rows ? row : rows - 1;                         // (rows that are not there repeat the last one; never stored)
    query[rt] = a.by_group(row);
    sink[rt] = mx_sink(a, kvh * a.group + row - query[rt] * a.group);
  }
  // Q and the outputs pass LDS, for whole rows of 128 bytes from and to memory (a lane's own pieces of them are 64 accesses an instruction): eight
  // rows at a time, lane / 8 of them, 16 bytes lane % 8; in LDS the pieces of a row are XORed with its number.
  const int last_row = rows - 1, q_first = a.by_group(row0 < last_row ? row0 : last_row);
  auto place = [&](int j, int* q_of, int* h_of) __attribute__((always_inline)) {     // row 8 j + lane / 8's query and head
    const int row = row0 + 8 * j + (lane >> 3), x = (row < rows ? row : last_row) - q_first * a.group;
    const int qx = a.by_group(x);
    *q_of = q_first + qx;
    *h_of = kvh * a.group + x - qx * a.group;
  };
  bf16x8 qf[2][4];
  u32x4 q_raw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int qq, hh;
    place(j, &qq, &hh);
    q_raw[j] = *reinterpret_cast<const u32x4*>(a.q + b * a.q_bs + qq * a.q_ts + hh * 64 + 8 * (lane & 7));
  }
  const MxSpan sp = mx_span(a, mx_start(a, b), rg * RB, rg * RB + RB - 1);
  const int len = sp.hi - sp.lo, all = (len + UNIT - 1) / UNIT;
  const int units = (all + KG - 1) / KG;                       // of each group: the wavefronts meet as often in all of them
  auto key_of = [&](int u) { return UNIT * (KG * u + kg); };   // a unit's first key

  int upper[2], lower[2];                                      // the keys that the lane's row sees, counted from sp.lo
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int64_t up = sp.start + query[rt] - sp.lo, low = up - a.window + 1;
    upper[rt] = static_cast<int>(up < -1 ? -1 : up < len - 1 ? up : len - 1);
    lower[rt] = static_cast<int>(a.window == 0 || low < 0 ? 0 : low < len ? low : len);
  }
  int seen_hi, seen_lo, w_lo, w_hi;                            // keys that every row of the wavefront sees; units of which any row sees a key
  {
    const int last = rows - 1, r0 = row0 < last ? row0 : last, r1 = row0 + 63 < last ? row0 + 63 : last;
    const int64_t up0 = sp.start + a.by_group(r0) - sp.lo, up1 = sp.start + a.by_group(r1) - sp.lo;
    auto held = [&](int64_t x, int least, int most) { return static_cast<int>(x < least ? least : x < most ? x : most); };
    seen_hi = held(up0, -1, len - 1);
    seen_lo = a.window == 0 ? 0 : held(up1 - a.window + 1, 0, len);
    const int n_hi = (held(up1, -1, len - 1) + UNIT) / UNIT, n_lo = a.window == 0 ? 0 : held(up0 - a.window + 1, 0, len) / UNIT;
    w_hi = (n_hi - kg + KG - 1) / KG;                          // (n_hi >= 0, kg < KG)
    w_lo = (n_lo - kg + KG - 1) / KG;
    w_lo = w_lo < w_hi ? w_lo : w_hi;
  }

  // What lies behind the last key of values is zeros in the tile (nothing there is seen; keys' scores are masked). What only some rows may see is
  // set aside as zeros, and added to the rows that see it.
  float power;
  auto prepare = [&](int u, int stage) __attribute__((always_inline)) {   // the unit about to be written
    if (kv != 0) {
      const bool in = key_of(u) + (piece >> 1) < len;
      const unsigned long long bad = __builtin_amdgcn_ballot_w64(raw_s > kFinite && in);
      if (lane == 0) s_any[kg][stage][run % HALVES] = bad != 0;
      if (__builtin_expect(key_of(u) + UNIT > len || bad != 0, 0)) {
        const MxAside pieces{bad, __builtin_amdgcn_ballot_w64(raw_s == 255u && in), __builtin_amdgcn_ballot_w64(raw_s == 254u && in)};
        if (lane == 0) s_aside[kg][stage][run % HALVES] = pieces;
        raw = in ? raw : u32x4{0u, 0u, 0u, 0u};
        raw_s = in ? raw_s : 0u;
        mx_set_aside(&raw, &raw_s);
      }
    }
    power = mx_power(raw_s);
  };
  unsigned char* const ring = smem + kg * 3 * STAGE;
  auto write_chunk = [&](int stage, int t) __attribute__((always_inline)) { *reinterpret_cast<bf16x8*>(ring + stage * STAGE + to[t]) = mx_bf16x8(raw[t], power); };
  // Ahead of the last block of unit u: every wavefront has written its share of unit u + 1, and has read the last of unit u - 1, whose stage takes
  // unit u + 2.
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto after = [](int stage) { return stage == 2 ? 0 : stage + 1; };

  // ---- operands
  unsigned k_off[4], v_off[2];                                 // K: lane (key l31, block h), four chunks; V: transposing reads, as above
#pragma unroll
  for (int m = 0; m < 4; ++m) k_off[m] = l31 * 128 + (((4 * h + m) ^ (l31 >> 1 & 7)) << 4);
#pragma unroll
  for (int db = 0; db < 2; ++db) v_off[db] = KTILE + mx_v_chunk4(4 * h + ((lane & 15) >> 2), 4 * db + 2 * (l31 >> 4) + (lane >> 1 & 1)) + (lane & 1) * 8;      // + 8 keys u, + 16 keys cc
  bf16x8 kf[4], vf[2][2];
  auto load_k = [&](int stage, int half) __attribute__((always_inline)) {
    const unsigned char* const t = ring + stage * STAGE + half * 4096;
#pragma unroll
    for (int m = 0; m < 4; ++m) kf[m] = *reinterpret_cast<const bf16x8*>(t + k_off[m]);
  };
  auto load_v = [&](int stage, int half) __attribute__((always_inline)) {
    const unsigned char* const t = ring + stage * STAGE + half * 4096;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        i16x4 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(t + v_off[db] + 2048 * cc + 1024 * u));
        vf[cc][db] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
  };

  const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float ref[2] = {kNoRef, kNoRef};
  f32x4 sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  f32x16 o[2][2] = {{zero, zero}, {zero, zero}}, s[2];
  u32x4 p[2][2];                                               // P^T in bf16, as operand registers
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      p[i][j] = u32x4{0u, 0u, 0u, 0u};
      vf[i][j] = __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
    }
  auto scores = [&](int rt, int m) __attribute__((always_inline)) { s[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[m], qf[rt][m], m == 0 ? zero : s[rt], 0, 0, 0); };
  auto product = [&](int rt, int m) __attribute__((always_inline)) {
    o[rt][m & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[m >> 1][m & 1], __builtin_bit_cast(bf16x8, p[rt][m >> 1]), o[rt][m & 1], 0, 0, 0);
  };
  // weights in pairs; a pair is summed and rounded while the next one's exponentials are on their way
  float e[2][2];
  auto weigh = [&](int rt, int m) __attribute__((always_inline)) {
    e[m & 1][0] = __builtin_amdgcn_exp2f(fmaf(s[rt][2 * m], a.scale_log2, -ref[rt]));
    e[m & 1][1] = __builtin_amdgcn_exp2f(fmaf(s[rt][2 * m + 1], a.scale_log2, -ref[rt]));
  };
  auto keep = [&](int rt, int m) __attribute__((always_inline)) {
    const bf16x2 v = {static_cast<bf16>(e[m & 1][0]), static_cast<bf16>(e[m & 1][1])};
    p[rt][m >> 2][m & 3] = __builtin_bit_cast(unsigned, v);
  };
  // the rounded weights, as the products take them, summed on the matrix cores as well: ones times a lane's own four
  const i16x4 ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80};
  auto add_up = [&](int rt, int m) __attribute__((always_inline)) {
    typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;
    const u32x2 four = {p[rt][m >> 1][2 * (m & 1)], p[rt][m >> 1][2 * (m & 1) + 1]};
    sum[rt] = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_bit_cast(i16x4, four), sum[rt], 0, 0, 0);
  };
  auto mask = [&](int rt, int k0) __attribute__((always_inline)) {
    int du = upper[rt] - k0 - 4 * h, dl = lower[rt] - k0 - 4 * h;
    asm volatile("" : "+v"(du), "+v"(dl));                     // (or the comparisons are made for every block)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[rt][r] = 8 * (r >> 2) + (r & 3) <= du && 8 * (r >> 2) + (r & 3) >= dl ? s[rt][r] : -INFINITY;
  };
  // The reference lies kLift above the largest logit that it was raised to, and is raised only where a weight has reached 2 (or is no number): one
  // OR over the rounded weights' bits tells.
  auto settle = [&](int rt) __attribute__((always_inline)) {
    unsigned bits = 0;
#pragma unroll
    for (int m = 0; m < 8; ++m) bits |= p[rt][m >> 2][m & 3];
    if (__builtin_expect(__builtin_amdgcn_ballot_w64((bits & 0x40004000u) != 0) != 0, 0)) {
      float top = s[rt][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[rt][r]);
      float x, y;
      lane_xor32_pair(top, &x, &y);
      top = fmaf(fmaxf(x, y), a.scale_log2, kLift);
      const float moved = top > ref[rt] ? top : ref[rt];
      const float alpha = __builtin_amdgcn_exp2f(ref[rt] - moved);
      ref[rt] = moved;
      auto scale = [&](auto& v, int n) __attribute__((always_inline)) {
        asm volatile("" : "+v"(v));
#pragma unroll
        for (int r = 0; r < n; ++r) v[r] *= alpha;
        asm volatile("" : "+v"(v));
      };
      scale(sum[rt], 4);
      scale(o[rt][0], 16);
      scale(o[rt][1], 16);
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        weigh(rt, m);
        keep(rt, m);
      }
      asm volatile("" : "+v"(p[rt][0]), "+v"(p[rt][1]));
    }
  };
  // A block, `half` of unit u in `stage`. The last of a unit meets the other wavefronts ahead; a unit is written on the way of the first one -- of two
  // blocks' units the next one, of one block's the one after it. `any`: the unit's flags, asked for a unit ago.
  typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;
  u32x2 any;
  auto block = [&](int u, int stage, auto tag) __attribute__((always_inline)) {
    constexpr int half = decltype(tag)::value;
    constexpr bool FIRST = half == 0, LAST = half == HALVES - 1;
    constexpr int AHEAD = 3 - HALVES;
    const int k0 = key_of(u) + 32 * half;
    const unsigned mine = any[half];
    const unsigned aside = __builtin_amdgcn_readfirstlane(mine);
    const int next = after(stage), to_stage = AHEAD == 1 ? next : after(next);
    if constexpr (LAST) {
      meet();
      any = *reinterpret_cast<const u32x2*>(s_any[kg][next]);
    }
    const bool masked = k0 + 31 > seen_hi || k0 < seen_lo;
    if (__builtin_expect(masked, 0)) mask(0, k0);
    if constexpr (FIRST) prepare(u + AHEAD, to_stage);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      scores(1, m);
      if constexpr (FIRST) write_chunk(to_stage, m);
      weigh(0, m);
      if (m > 0) keep(0, m - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    load_k(LAST ? next : stage, LAST ? 0 : half + 1);          // (the next block's, half a block ahead)
    if constexpr (FIRST) load_unit(u + AHEAD + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 4; m < 8; ++m) {
      product(1, m - 4);
      add_up(1, m - 4);
      weigh(0, m);
      keep(0, m - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    keep(0, 7);
    load_v(stage, half);
    settle(0);
    if (__builtin_expect(masked, 0)) mask(1, k0);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      scores(0, m);
      weigh(1, m);
      if (m > 0) keep(1, m - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = 4; m < 8; ++m) {
      product(0, m - 4);
      add_up(0, m - 4);
      weigh(1, m);
      keep(1, m - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    keep(1, 7);
    settle(1);
    // (behind both tiles' products of the keys ahead, at the references that the tiles have now)
    if (__builtin_expect(aside != 0, 0)) {
      auto scalar = [](unsigned long long x) { return static_cast<unsigned long long>(__builtin_amdgcn_readfirstlane(static_cast<unsigned>(x >> 32))) << 32 | static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<unsigned>(x))); };
      const MxAside pieces{scalar(s_aside[kg][stage][half].any), scalar(s_aside[kg][stage][half].nan), scalar(s_aside[kg][stage][half].large)};
      for (unsigned long long left = pieces.any; left != 0; left &= left - 1) {
        const int at = __builtin_ctzll(left), key = k0 + (at >> 1);
        const unsigned char* const from = a.c.blocks[1] + b * a.c.bs + kvh * a.c.hs + (lo + key) * a.c.ts + 16 * (at & 1);
        const unsigned byte = pieces.byte(at);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
          if (key >= lower[rt] && key <= upper[rt]) {
            if (at & 1) mx_add_aside(&o[rt][1], from, byte, h);
            else mx_add_aside(&o[rt][0], from, byte, h);
          }
      }
    }
  };
  constexpr int AHEAD = 3 - HALVES;
  auto write_unit = [&](int u, int stage) __attribute__((always_inline)) {
    prepare(u, stage);
#pragma unroll
    for (int t = 0; t < 4; ++t) write_chunk(stage, t);
    load_unit(u + 1);
  };
  auto move = [&](int u, int stage) __attribute__((always_inline)) {      // a unit that only other wavefronts look at
    const int next = after(stage);
    if constexpr (AHEAD == 1) write_unit(u + 1, next);
    meet();
    any = *reinterpret_cast<const u32x2*>(s_any[kg][next]);
    if constexpr (AHEAD == 2) write_unit(u + 2, after(next));
  };

  unsigned char* const q_lds = smem + wave * 8192;
  static_assert(RUNS * KG * 8192 <= KG * 3 * STAGE, "Q fits the stages");
#pragma unroll
  for (int j = 0; j < 8; ++j) *reinterpret_cast<u32x4*>(q_lds + 1024 * j + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4)) = q_raw[j];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int m = 0; m < 4; ++m) qf[rt][m] = *reinterpret_cast<const bf16x8*>(q_lds + (32 * rt + l31) * 128 + (((4 * h + m) ^ (l31 & 7)) << 4));
  __syncthreads();
  if (units > 0) {
    write_unit(0, 0);
    if constexpr (AHEAD == 2) write_unit(1, 1);
    meet();
    any = *reinterpret_cast<const u32x2*>(s_any[kg][0]);
    int u = 0, stage = 0;
    for (; u < w_lo; ++u, stage = after(stage)) move(u, stage);
    if (w_lo < w_hi) {
      load_k(stage, 0);
#pragma unroll
      for (int m = 0; m < 4; ++m) scores(0, m);
      for (; u < w_hi; ++u, stage = after(stage)) {
        block(u, stage, std::integral_constant<int, 0>{});
        if constexpr (HALVES == 2) block(u, stage, std::integral_constant<int, 1>{});
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        product(1, m);
        add_up(1, m);
      }
    }
    for (; u < units; ++u, stage = after(stage)) move(u, stage);
  }

  float l[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    float x, y;
    lane_xor32_pair(sum[rt][0], &x, &y);
    l[rt] = x + y;
  }
  // A tile's end: the sink joins the denominator; a lane has 8-byte runs of one row's values, which leave through 4 KB of LDS of the wavefront's own.
  auto lay = [&](auto tag, unsigned char* lds) __attribute__((always_inline)) {
    constexpr int rt = decltype(tag)::value;
    const float f = mx_norm(a, sink[rt], ref[rt], l[rt]);
#pragma unroll
    for (int r = 0; r < 32; r += 4) {
      bf16x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = o[rt][r >> 4][(r & 15) + e];
        w[e] = static_cast<bf16>(v * f);
      }
      *reinterpret_cast<bf16x4*>(lds + l31 * 128 + ((r >> 2 ^ (l31 & 7)) << 4) + 8 * h) = w;
    }
  };
  auto leave = [&](auto tag, const unsigned char* lds) __attribute__((always_inline)) {
    constexpr int rt = decltype(tag)::value;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(lds + 1024 * j + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4));
      int qq, hh;
      place(4 * rt + j, &qq, &hh);
      if (row0 + 32 * rt + 8 * j + (lane >> 3) < rows) *reinterpret_cast<u32x4*>(a.out + b * a.out_bs + qq * a.out_ts + hh * 64 + 8 * (lane & 7)) = w;
    }
  };
  typedef std::integral_constant<int, 0> first_tile;
  typedef std::integral_constant<int, 1> second_tile;
  __syncthreads();                                             // (all are past their last read of the stages)
  if constexpr (KG == 2) {
    // each group hands one tile over and finishes the other
    auto share = [&](int rt) { return reinterpret_cast<float*>(smem) + (run * 2 + rt) * kShare; };
    auto give = [&](auto tag) __attribute__((always_inline)) {
      constexpr int rt = decltype(tag)::value;
      float* const to = share(rt);
#pragma unroll
      for (int r = 0; r < 32; r += 4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[rt][r >> 4][(r & 15) + e];
        *reinterpret_cast<f32x4*>(to + 64 * r + 4 * lane) = v;
      }
      to[32 * 64 + lane] = ref[rt];
      to[33 * 64 + lane] = l[rt];
    };
    auto take = [&](auto tag) __attribute__((always_inline)) {
      constexpr int rt = decltype(tag)::value;
      const float* const from = share(rt);
      const float other = from[32 * 64 + lane], m = fmaxf(ref[rt], other);
      const float f0 = __builtin_amdgcn_exp2f(ref[rt] - m), f1 = __builtin_amdgcn_exp2f(other - m);
      ref[rt] = m;
      l[rt] = l[rt] * f0 + from[33 * 64 + lane] * f1;
#pragma unroll
      for (int r = 0; r < 32; r += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(from + 64 * r + 4 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[rt][r >> 4][(r & 15) + e] = o[rt][r >> 4][(r & 15) + e] * f0 + v[e] * f1;
      }
      unsigned char* const lds = reinterpret_cast<unsigned char*>(share(rt));      // (read by this wavefront alone)
      lay(tag, lds);
      leave(tag, lds);
    };
    if (kg == 0) give(second_tile{});
    else give(first_tile{});
    __syncthreads();
    if (kg == 0) take(first_tile{});
    else take(second_tile{});
  } else {
    unsigned char* const lds = smem + wave * 8192;
    lay(first_tile{}, lds);
    lay(second_tile{}, lds + 4096);
    leave(first_tile{}, lds);
    leave(second_tile{}, lds + 4096);
  }
}

// A wavefront per (batch row, query, head): the splits' records and the sink. Lane s has the (max, sum) of split s. Two reads' latency and a launch:
// for 512 heads of four splits 2.8 us as traced (1.9 at least), and a graph is 1.8 longer with it than a call that is not split (8 rows of 1000).
__global__ __launch_bounds__(64) void mxfp4_attn_reduce_kernel(MxAttnArgs a, int rows_per_group) {
  const int lane = threadIdx.x;
  const int n_heads = a.n_kv_heads * a.group;
  const int i0 = a.by_group(blockIdx.x), i1 = a.by_heads(i0), kvh = i0 - i1 * a.n_kv_heads;      // (the block is ((batch row, query), head))
  const int head = blockIdx.x - i1 * n_heads, b = a.by_n_q(i1), i = i1 - b * a.n_q;
  const int row = i * a.group + head - kvh * a.group, row0 = row & -rows_per_group;      // (a power of two)
  const int64_t stride = static_cast<int64_t>(a.batch) * a.n_q * n_heads * PART;
  const float* const p0 = a.part + ((static_cast<int64_t>(b) * a.n_q + i) * n_heads + head) * PART;
  // requested before the start position is known; what splits that take no part have there is not used
  const float m_raw = lane < a.splits ? p0[lane * stride + 64] : kNoRef, l_raw = lane < a.splits ? p0[lane * stride + 65] : 0.f;
  float v[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = p0[(u < a.splits ? u : a.splits - 1) * stride + lane];
  const bf16 sink = mx_sink(a, head);
  const int live = mx_span(a, mx_start(a, b), row0, row0 + rows_per_group - 1).live;
  if (live == 1) return;                                       // (whoever walked the keys alone has stored the answer)
  const float m_s = lane < live ? m_raw : kNoRef;
  const float m_all = wave_max(m_s);
  const float f_s = __builtin_amdgcn_exp2f(m_s - m_all);
  const float l_all = wave_sum(lane < live ? l_raw * f_s : 0.f);
  float o = 0.f;
  for (int s0 = 0; s0 < live; s0 += 8) {
    if (s0 > 0) {
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p0[(s0 + u < live ? s0 + u : live - 1) * stride + lane];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f_s), __builtin_amdgcn_readfirstlane(s0 + u < live ? s0 + u : 0)));
      o += s0 + u < live ? v[u] * f : 0.f;
    }
  }
  const float f = mx_norm(a, sink, m_all, l_all);
  a.out[b * a.out_bs + i * a.out_ts + static_cast<int64_t>(head) * 64 + lane] = static_cast<bf16>(o * f);
}

}  // namespace tllm

using namespace tllm;

namespace {
struct MxAttnPlan {
  bool one, many;                     // the kernel for one query, for many rows; otherwise the one for any
  int tiles, waves;                   // of the latter: tiles of 32 rows; wavefronts of a workgroup
  int row_groups, rows;               // runs of rows that workgroups take, rows in each
  int splits, fill;
};

// Which kernel, by the runs of rows and of streams that there are (eight KV heads of eight query heads, us; "n behind m": n queries behind m tokens;
// the figures of one sweep compare kernels with each other, and some of those they name have become faster since, or serve other sizes now):
//   Many rows, 256 to a workgroup, from 385 runs of 256 on -- one prompt of 2048 51.9, in 128 rows a workgroup 55.7, 64 56.7, 32 62.5; 4096 158, 174, 183,
//   213 -- and from 513 runs of 128 on where walks are short, up to 768 keys: 2 x 700 24.3, 26.2, 27.6, 27.2; 2048 with a window of 128 19, 25, 32, 31.
//   Between, two workgroups to a CU do not come out even: 1200 33.7, 25.7, 28.8, 29; 1200 behind 6800 223, 213, 178, 202; 1500 behind 2500 104, 104, 102,
//   116.
//   Of those, 321 to 512 runs of 256 of prompts (walks up to twice as long as there are queries, and longer than 1024): two groups of wavefronts that
//   take the keys in turn, one workgroup to a CU after the other. Otherwise the longest walks' workgroups, which alone have a CU's matrix cores
//   at 0.7 of their rate, are what the launch takes: 2048 48.4, without 51.5; 1800 42.7, 45.6; 1500 32.8, 39.0, in 64 rows 35.3; 1300 28.7, 34.6, 30.6;
//   but 1200 26.8, 32.3, 27.5; 2 x 978 32.5, 30.5; 4 x 500 24.9, 20.6; 2048 behind 2048 113.5, 111.9.
//   128 to a workgroup from 385 to 512 runs of them, one or two workgroups to a CU: 2 x 512 15.8, in 256 rows 18.8, 64 18.8, 32 18.9; 4 x 256 13.0,
//   13.6, 17.0, 17.2; 3 x 333 13.9, 16.0, 17.5, 17.8; 8 x 128 behind 2000 47.6, 51.4, 49.8, 56; 1000 behind 8000 162, 188, 165, 188; 800 behind 4000
//   85.4, 103, 86.8, 89; but 700 behind 4000 (352) 84, 101, 70, 77, and 512 behind 4000 64, 96, 48, 56. To 640 for prompts: 1200 24.5, 31.7, 27.6, 27.5;
//   1100 23.1, 30.2, 25.5, 24.4 (behind 1000 52, 53, 47.6, 50). (Not the best where walks are shortest or longest: 16 x 64 10.2, in 256 rows 8.8; 1000
//   behind 8000 164, in 256 rows with two groups of wavefronts 151.)
//   32 rows shared out between eight wavefronts up to 256 runs of 32: 97 behind 1500 10.0, between four 11.7; 97 behind 8000 31, 39; 64 behind 8000
//   24.2, 26.9; with four from there on: 150 behind 1350 17.3, 13.8; 256 behind 2000 22, 18.2; 64 x 4 of 1000 16.1, 12.5.
//   64 rows to a workgroup from 768 such runs on: 512 behind 4000 48, with 32 rows 56; 700 behind 4000 70, 77; 512 9.9, 11.4; but 350 behind 4000 44.6,
//   40; 333 9.2, 7.8; 64 x 4 of 1000 16.4, 12.5; not where that is a little more than two workgroups to a CU: 600 15.2, 12.9; 600 behind 4000 68, 65.5;
//   prompts of 700 16.8, 14.3, of 800 18.1, 17.2.
// Workgroups that share rows' keys, as many as there are CUs for, up to kDeep keys only if that is four: 8 x 4 of 4096 (64 runs) 12.5, none 16.8;
// 64 behind 8000 (128) two 22.2, none 28.9; 72 x 2 of 11000 in four heads of four (72) three 22.3, none 36; but 8 x 8 of 2000 (128) two 13.9, none
// 11.2; 97 behind 8000 (200) two 38, none 28.7; 512 behind 4000 in 64 rows (512) two 67, none 48.
MxAttnPlan mx_attn_plan(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window) {
  MxAttnPlan p{};
  const int64_t rows = n_q * group, streams = batch * n_kv_heads;
  auto seen = [&](int64_t run) {                               // keys that the queries of a run of rows can see together
    const int64_t span = (int64_t)window + (run + group - 1) / group;
    return window > 0 && span < n_slots ? span : n_slots;
  };
  const int64_t wide = (rows + 255) / 256 * streams, half = (rows + 127) / 128 * streams, narrow = (rows + 31) / 32 * streams;
  p.one = n_q == 1 && group <= 8;
  const bool prompt = window == 0 && n_slots <= 2 * n_q, unlike = prompt && n_slots > 1024 && wide > 320 && wide <= 512;
  const bool halves = !unlike && half > 384 && half <= (prompt && n_slots > 768 ? 640 : 512);
  p.many = !p.one && rows > 128 && (unlike || halves || wide > 384 || (half > 512 && seen(256) <= 768));
  p.tiles = narrow < 768 || (narrow > 1024 && narrow <= (prompt ? 1600 : 1300)) ? 1 : 2;
  p.waves = !p.one && (p.many ? unlike : narrow <= 256) ? 8 : 4;
  p.rows = p.one ? 8 : p.many ? (halves ? 128 : 256) : 32 * p.tiles;
  p.row_groups = (int)((rows + p.rows - 1) / p.rows);
  const int64_t units = streams * p.row_groups;
  p.fill = p.one ? (int)((kFill + units - 1) / units) : kFill / units > 0 ? (int)(kFill / units) : 1;
  p.splits = p.many ? 1 : mx_attn_splits(p.one, p.fill, (int)seen(p.rows));
  return p;
}

int64_t mx_attn_ctx(int64_t n_slots, int64_t hint) { return hint > 0 && hint < n_slots ? hint : n_slots; }
}  // namespace

extern "C" int tllm_mxfp4_attention_shape(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window, int64_t kv_len_hint) {
  if (batch < 1 || batch > 65535 || n_q < 1 || n_q >= (1ll << 24) || n_slots < 1 || n_slots >= (1ll << 30) || n_kv_heads < 1 || n_kv_heads > 65535 || group < 1 ||
      group > 64 || window < 0 || kv_len_hint < 0)
    return 0;
  const MxAttnPlan p = mx_attn_plan(batch, n_q, mx_attn_ctx(n_slots, kv_len_hint), n_kv_heads, group, window);
  return p.rows << 16 | p.waves << 8 | p.splits;
}

extern "C" int64_t tllm_mxfp4_attention_workspace_bytes(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window, int64_t kv_len_hint) {
  const int s = tllm_mxfp4_attention_shape(batch, n_q, n_slots, n_kv_heads, group, window, kv_len_hint) & 0xff;
  return s > 1 ? (int64_t)s * batch * n_q * n_kv_heads * group * PART * 4 : 0;
}

template <bool DENSE, int RT, int KG>
static int launch_rows(const MxAttnArgs& a, dim3 grid, hipStream_t st) {
  constexpr int SMEM = KG * kShare * 4;
  static std::atomic<uint64_t> done{0};
  const hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(mxfp4_attn_rows_kernel<DENSE, RT, KG>), SMEM, done);
  TLLM_REQUIRE(e == hipSuccess, TLLM_E_LAUNCH, "mxfp4_attention: cannot raise LDS limit: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((mxfp4_attn_rows_kernel<DENSE, RT, KG>), grid, dim3(KG * 64), SMEM, st, a);
  return TLLM_OK;
}

template <bool DENSE>
static int launch_attention(const MxAttnPlan& p, const MxAttnArgs& a, dim3 grid, hipStream_t st) {
  if (p.many) {
    if (p.waves == 8) hipLaunchKernelGGL((mxfp4_attn_many_kernel<4, 2>), grid, dim3(512), 0, st, a);
    else if (p.rows == 256) hipLaunchKernelGGL((mxfp4_attn_many_kernel<4, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mxfp4_attn_many_kernel<2, 2>), grid, dim3(256), 0, st, a);
  }
  else if (p.one) hipLaunchKernelGGL((mxfp4_attn_one_kernel<DENSE>), grid, dim3(256), 0, st, a);
  else if (p.waves == 8) return launch_rows<DENSE, 1, 8>(a, grid, st);
  else return p.tiles == 1 ? launch_rows<DENSE, 1, 4>(a, grid, st) : launch_rows<DENSE, 2, 4>(a, grid, st);
  return TLLM_OK;
}

extern "C" int tllm_mxfp4_attention_bf16(const void* q, int64_t q_batch_stride, int64_t q_token_stride, const TllmMxCache* cache, const void* sinks, void* out,
                                         int64_t out_batch_stride, int64_t out_token_stride, int64_t n_q, int group, float sm_scale, int window,
                                         const void* start_q, int start_q_is_i64, int start_q_per_row, int64_t kv_len_hint, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  MxAttnArgs a{};
  if (const int rc = mx_cache_of(cache, "mxfp4_attention", &a.c); rc != TLLM_OK) return rc;
  const int64_t batch = cache->batch, n_slots = cache->n_slots;
  const int n_kv_heads = cache->n_kv_heads;
  TLLM_REQUIRE(cache->head_dim == 64, TLLM_E_SHAPE, "mxfp4_attention: head_dim %d (only 64 is built)", cache->head_dim);
  TLLM_REQUIRE(n_slots >= 1, TLLM_E_SHAPE, "mxfp4_attention: a cache of no slots");
  TLLM_REQUIRE(n_q >= 0 && n_q < (1ll << 24), TLLM_E_SHAPE, "mxfp4_attention: %lld queries", (long long)n_q);
  TLLM_REQUIRE(group >= 1 && group <= 64, TLLM_E_SHAPE, "mxfp4_attention: %d query heads per KV head (1..64)", group);
  TLLM_REQUIRE(window >= 0, TLLM_E_ARG, "mxfp4_attention: window %d", window);
  TLLM_REQUIRE(sm_scale > 0.f && sm_scale < __builtin_inff(), TLLM_E_ARG, "mxfp4_attention: sm_scale %g must be positive", (double)sm_scale);
  TLLM_REQUIRE(kv_len_hint >= 0, TLLM_E_ARG, "mxfp4_attention: kv_len_hint %lld", (long long)kv_len_hint);
  if (batch == 0 || n_q == 0) return TLLM_OK;
  TLLM_REQUIRE(q && out && start_q, TLLM_E_ARG, "mxfp4_attention: q, out and start_q must not be NULL");
  const int64_t n_heads = (int64_t)n_kv_heads * group;
  TLLM_REQUIRE(aligned16(q) && aligned16(out) && q_batch_stride % 8 == 0 && q_token_stride % 8 == 0 && out_batch_stride % 8 == 0 && out_token_stride % 8 == 0,
               TLLM_E_ALIGN, "mxfp4_attention: q and out must be 16-byte aligned with strides that are multiples of 8 elements");
  TLLM_REQUIRE(n_q * group < (1ll << 30) && batch * n_q * n_heads < (1ll << 31), TLLM_E_SHAPE, "mxfp4_attention: %lld x %lld queries of %lld heads are too many",
               (long long)batch, (long long)n_q, (long long)n_heads);
  const int64_t plan_ctx = mx_attn_ctx(n_slots, kv_len_hint);
  const MxAttnPlan p = mx_attn_plan(batch, n_q, plan_ctx, n_kv_heads, group, window);
  const int64_t need = tllm_mxfp4_attention_workspace_bytes(batch, n_q, n_slots, n_kv_heads, group, window, kv_len_hint);
  TLLM_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 4 == 0), TLLM_E_ARG,
               "mxfp4_attention: workspace of %lld bytes needed (tllm_mxfp4_attention_workspace_bytes), got %lld", (long long)need, (long long)workspace_bytes);
  const int64_t wgs = (int64_t)p.splits * batch * n_kv_heads * p.row_groups;
  TLLM_REQUIRE(wgs < (1ll << 24) && (p.splits == 1 || batch * n_q * n_heads < (1ll << 26)), TLLM_E_SHAPE, "mxfp4_attention: %lld workgroups are too many for one launch", (long long)wgs);
  a.q = (const bf16*)q;
  a.sinks = (const bf16*)sinks;
  a.out = (bf16*)out;
  a.part = (float*)workspace;
  a.start_q = start_q;
  a.start_is_i64 = start_q_is_i64;
  a.start_stride = start_q_per_row != 0;
  a.q_bs = q_batch_stride;
  a.q_ts = q_token_stride;
  a.out_bs = out_batch_stride;
  a.out_ts = out_token_stride;
  a.batch = (int)batch;
  a.n_q = (int)n_q;
  a.n_kv_heads = n_kv_heads;
  a.group = group;
  a.window = window;
  a.row_groups = p.row_groups;
  a.splits = p.splits;
  a.fill = p.fill;
  a.one = p.one;
  a.scale_log2 = sm_scale * kLog2e;
  a.by_group = mx_div((unsigned)group);
  a.by_heads = mx_div((unsigned)n_kv_heads);
  a.by_batch = mx_div((unsigned)batch);
  a.by_row_groups = mx_div((unsigned)p.row_groups);
  a.by_n_q = mx_div((unsigned)n_q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)wgs);
  const uintptr_t scales_at = reinterpret_cast<uintptr_t>(cache->k_scales) | reinterpret_cast<uintptr_t>(cache->v_scales) | static_cast<uintptr_t>(cache->scale_batch_stride | cache->scale_head_stride);
  int rc = cache->scale_slot_stride == 2 && n_slots > 1 && scales_at % 2 == 0 ? launch_attention<true>(p, a, grid, st) : launch_attention<false>(p, a, grid, st);
  if (rc != TLLM_OK) return rc;
  rc = check_launch("mxfp4_attention");
  if (rc != TLLM_OK || p.splits == 1) return rc;
  hipLaunchKernelGGL(mxfp4_attn_reduce_kernel, dim3((unsigned)(batch * n_q * n_heads)), dim3(64), 0, st, a, p.rows);
  return check_launch("mxfp4_attention(reduce)");
}
