// Attention over an MXFP4 KV cache with learned sinks and an optional sliding window, one or several new tokens per batch row:
//
//   query i of row b sits at p = start_q[b] + i and sees the slots n <= p, n < n_slots, n > p - window (when a window is set)
//   s[i, h, n] = sm_scale * <q[i, h], k[n, kv(h)]>                      kv(h) = h / G   (G query heads share a KV head)
//   out[i, h]  = sum_n exp(s - m) v[n, kv(h)] / (sum_n exp(s - m) + exp(sink[h] - m)),    m = max(sink[h], max_n s)
//
// with k and v the values that the cache's codes and scale bytes stand for, exactly (an e2m1 value times a power of two is a bf16 value).
// A scale byte of 255 makes its 32 values NaN, for the queries that see the slot and for no other.
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
  int splits, fill, keys_shift;
  float scale_log2;       // sm_scale * log2 e
};

namespace {
constexpr int kNW = 4;                // wavefronts of a workgroup
constexpr int VROW = 128 + 32;        // V tile row in LDS, bytes: eight keys' 32-byte pieces in different banks
constexpr int VTILE = 32 * VROW;
constexpr int AROW = 64 + 1;          // accumulator row in LDS, floats
constexpr int PART = 66;              // floats of a record in the workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;         // log2 units by which a block must exceed the running maximum to move it
}  // namespace

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((__vector_size__(8 * sizeof(short)))) short i16x8;
typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;

// Context splits for `fill` workgroups a stream over `ctx` visible keys: enough to fill the CUs, beyond that about 2^keys_shift keys each,
// never less than 128, at most 64. The host plans the launch with it from the size of the cache (or the caller's hint), the kernels evaluate
// it again with the length that they read.
__host__ __device__ inline int mx_attn_splits(int fill, int ctx, int keys_shift) {
  const int cap = ((ctx - 1) >> 7) + 1, by_work = ((ctx - 1) >> keys_shift) + 1;
  int s = fill > by_work ? fill : by_work;
  s = s < cap ? s : cap;
  s = s > 1 ? s : 1;
  return s < 64 ? s : 64;
}

// The keys lo .. hi-1 that any of the rows first .. last of batch row b sees, and the number of splits that take part.
struct MxSpan {
  int64_t start;
  int lo, hi, live;
};
__device__ __forceinline__ MxSpan mx_span(const MxAttnArgs& a, int b, int first_row, int last_row) {
  MxSpan s;
  s.start = mx_row_int(a.start_q, a.start_is_i64, static_cast<int64_t>(b) * a.start_stride);
  const int64_t far = 1ll << 40;                               // (beyond any slot; sums of it stay within 64 bits)
  s.start = s.start < -far ? -far : s.start > far ? far : s.start;
  const int q0 = first_row / a.group, q1 = last_row / a.group;
  int64_t hi = s.start + (q1 < a.n_q ? q1 : a.n_q - 1) + 1;
  hi = hi < 0 ? 0 : hi < a.c.n_slots ? hi : a.c.n_slots;
  int64_t lo = a.window > 0 ? s.start + q0 - a.window + 1 : 0;
  lo = lo < 0 ? 0 : lo < hi ? lo : hi;
  s.lo = static_cast<int>(lo);
  s.hi = static_cast<int>(hi);
  const int live = mx_attn_splits(a.fill, hi > lo ? s.hi - s.lo : 1, a.keys_shift);
  s.live = live < a.splits ? live : a.splits;
  return s;
}

// What the weighted sum of a row's values is multiplied with: the sink joins the denominator. Nothing at all to attend to -- no key and a
// sink of -infinity -- gives zeros.
__device__ __forceinline__ float mx_norm(const MxAttnArgs& a, int head, float m, float l) {
  const float sink = a.sinks ? static_cast<float>(a.sinks[head]) * kLog2e : 0.f;
  const float top = fmaxf(m, sink);
  if (top == -INFINITY) return l == l ? 0.f : l;
  const float f = __builtin_amdgcn_exp2f(m - top);
  return f / (l * f + __builtin_amdgcn_exp2f(sink - top));
}

// Rows of a workgroup: RT tiles of 16 of the rows r = query * G + head of a KV head. ONE: a single query of up to eight heads, which are
// held twice, once for each half of a block's keys.
template <int RT, bool ONE>
__global__ __launch_bounds__(kNW * 64) void mxfp4_attn_kernel(MxAttnArgs a) {
  constexpr int RB = ONE ? 8 : 16 * RT;
  __shared__ __align__(16) unsigned char vt[kNW * VTILE];
  __shared__ float s_m[kNW][16], s_l[kNW][16];
  static_assert(16 * AROW * 4 <= VTILE, "an accumulator fits a tile");
  static_assert(!ONE || RT == 1, "a single query is one tile");

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;

  // the splits are the slowest part of the index: those that a context does not need are the last
  unsigned id = blockIdx.x;
  const int kvh = id % a.n_kv_heads;
  id /= a.n_kv_heads;
  const int rg = id % a.row_groups;
  id /= a.row_groups;
  const int b = id % a.batch, split = id / a.batch;
  const int rows = a.n_q * a.group, row0 = rg * RB;
  const MxSpan sp = mx_span(a, b, row0, row0 + RB - 1);
  if (split >= sp.live) return;
  int chunk = (sp.hi - sp.lo + sp.live - 1) / sp.live;
  chunk = (chunk + 31) & ~31;
  const int s_lo = sp.lo + split * chunk < sp.hi ? sp.lo + split * chunk : sp.hi;
  const int s_hi = s_lo + chunk < sp.hi ? s_lo + chunk : sp.hi;
  const int nblk = (s_hi - s_lo + 31) >> 5;

  // ---- Q as the B operand of S^T = K . Q^T: lane (row r16, k slots 8 g + j)
  // ONE: the slots of g = 0, 1 are one key's two blocks of 32, those of g = 2, 3 the two of the key 16 places on. The columns 0 - 7 have
  // Q in the former and zeros in the latter, the columns 8 - 15 the reverse, so that they are the same heads over other keys, no
  // column is empty, and a lane's scores are four.
  bf16x8 qf[RT][ONE ? 4 : 2];
  int upper[RT], lower[RT];                                    // the keys that the lane's row sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int row = row0 + (ONE ? r16 & 7 : 16 * rt + r16);
    row = row < rows ? row : rows - 1;                         // (rows that are not there repeat the last one; never stored)
    const int i = row / a.group, head = kvh * a.group + row - i * a.group;
    const bf16* const qr = a.q + b * a.q_bs + i * a.q_ts + head * 64;
    const int64_t up = sp.start + i < a.c.n_slots - 1 ? sp.start + i : a.c.n_slots - 1, low = a.window > 0 ? sp.start + i - a.window + 1 : 0;
    upper[rt] = static_cast<int>(up > -1 ? up : -1);
    lower[rt] = static_cast<int>(low < 0 ? 0 : low < a.c.n_slots ? low : a.c.n_slots);
    if constexpr (ONE) {
      const bool mine = (g >> 1) == (r16 >> 3);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(qr + 32 * (g & 1) + 8 * st);
        qf[rt][st] = __builtin_bit_cast(bf16x8, mine ? w : u32x4{0u, 0u, 0u, 0u});
      }
    } else {
#pragma unroll
      for (int st = 0; st < 2; ++st) qf[rt][st] = *reinterpret_cast<const bf16x8*>(qr + 16 * g + 8 * st);
    }
  }

  const int64_t kv_off = b * a.c.bs + kvh * a.c.hs, sc_off = b * a.c.sbs + kvh * a.c.shs;
  const unsigned char *const kp = a.c.blocks[0] + kv_off, *const vp = a.c.blocks[1] + kv_off;
  const unsigned char *const ksp = a.c.scales[0] + sc_off, *const vsp = a.c.scales[1] + sc_off;
  const unsigned ts = static_cast<unsigned>(a.c.ts), sts = static_cast<unsigned>(a.c.sts);
  unsigned char* const vtile = vt + wave * VTILE;

  float m_run[RT], l_run[RT];                                  // of row r16 (the sum: this lane's share of it)
  f32x4 acc[RT][4];                                            // O: lane (d = 16 nb + r16, rows 4 g + i)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m_run[rt] = -INFINITY;
    l_run[rt] = 0.f;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[rt][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // A block's loads. Rows past the end are clamped to the last key, which is a visible one; their weights are zero.
  struct Block {
    u32x4 k, v;
    unsigned ks[2], vs;
  };
  auto load_block = [&](int blk, Block& w) __attribute__((always_inline)) {
    const int k0 = s_lo + 32 * blk;
    const unsigned last = s_hi - k0 - 1;
    const unsigned char *const kb = kp + static_cast<int64_t>(k0) * a.c.ts, *const vb = vp + static_cast<int64_t>(k0) * a.c.ts;
    const unsigned char *const ksb = ksp + static_cast<int64_t>(k0) * a.c.sts, *const vsb = vsp + static_cast<int64_t>(k0) * a.c.sts;
    auto held = [&](unsigned r) { return r < last ? r : last; };
    if constexpr (ONE) {
      const unsigned r = held(r16 + 16 * (g >> 1));
      w.k = *reinterpret_cast<const u32x4*>(kb + r * ts + 16 * (g & 1));
      w.ks[0] = ksb[r * sts + (g & 1)];
    } else {
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2) {
        const unsigned r = held(16 * kb2 + r16);
        const u32x2 two = *reinterpret_cast<const u32x2*>(kb + r * ts + 8 * g);
        w.k[2 * kb2] = two[0];
        w.k[2 * kb2 + 1] = two[1];
        w.ks[kb2] = ksb[r * sts + (g >> 1)];
      }
    }
    const unsigned r = held(lane >> 1);
    w.v = *reinterpret_cast<const u32x4*>(vb + r * ts + 16 * (lane & 1));
    w.vs = vsb[r * sts + (lane & 1)];
  };
  // keys up to `seen_hi` and from `seen_lo` on are seen by every row
  const int64_t first_at = sp.start + row0 / a.group, last_i = (row0 + RB - 1) / a.group;
  const int64_t last_low = a.window > 0 ? sp.start + (last_i < a.n_q ? last_i : a.n_q - 1) - a.window + 1 : 0;
  const int seen_hi = static_cast<int>(first_at < s_hi - 1 ? (first_at > -1 ? first_at : -1) : s_hi - 1);
  const int seen_lo = static_cast<int>(last_low < 0 ? 0 : last_low < a.c.n_slots ? last_low : a.c.n_slots);
  auto power = [](unsigned byte) { return __builtin_bit_cast(float, byte << 23); };

  Block cur;
  if (wave < nblk) load_block(wave, cur);
  for (int blk = wave; blk < nblk; blk += kNW) {
    const int k0 = s_lo + 32 * blk;
    // ---- S^T
    f32x4 st[RT][ONE ? 1 : 2];
    if constexpr (ONE) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_bf16x8(cur.k[t], power(cur.ks[0])), qf[0][t], s, 0, 0, 0);
      st[0][0] = s;
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const bf16x8 k0f = mx_bf16x8(cur.k[2 * kb], power(cur.ks[kb])), k1f = mx_bf16x8(cur.k[2 * kb + 1], power(cur.ks[kb]));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          f32x4 s = {0.f, 0.f, 0.f, 0.f};
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0f, qf[rt][0], s, 0, 0, 0);
          st[rt][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1f, qf[rt][1], s, 0, 0, 0);
        }
      }
    }
    // ---- V into the wavefront's tile, as bf16
    // A NaN that only some of the rows see may not reach the others as 0 x NaN: it is put aside as zeros and added behind (rare).
    unsigned long long bad = 0;
    unsigned vs = cur.vs;
    u32x4 vc = cur.v;
    if constexpr (!ONE) {
      bad = __builtin_amdgcn_ballot_w64(vs == 255u);
      if (bad != 0) {
        vc = vs == 255u ? u32x4{0u, 0u, 0u, 0u} : vc;
        vs = vs == 255u ? 0u : vs;
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) *reinterpret_cast<bf16x8*>(vtile + (lane >> 1) * VROW + (lane & 1) * 64 + t * 16) = mx_bf16x8(vc[t], power(vs));
    // The next block's loads go out before the rest of this one. Unconditional: the last round asks for its own block again.
    load_block(blk + kNW < nblk ? blk + kNW : blk, cur);

    // ---- online softmax: this lane holds keys k0 + 4 g + i of row r16 (ONE: 16 on in the columns 8 - 15), and 16 on
    bf16x8 pa[RT];                                             // A operand of P . V: k slot j <-> key 4 g + j (j < 4), 16 + 4 g + j - 4
    const bool masked = ONE ? k0 + 31 >= s_hi : k0 + 31 > seen_hi || k0 < seen_lo;     // (a single query sees all of its span)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      constexpr int NK = ONE ? 4 : 8;
      float sc[NK];
#pragma unroll
      for (int j = 0; j < NK; ++j) sc[j] = st[rt][j >> 2][j & 3];
      if (masked) {
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int key = k0 + 4 * g + (j & 3) + 16 * (ONE ? r16 >> 3 : j >> 2);
          sc[j] = key < s_hi && (ONE || (key <= upper[rt] && key >= lower[rt])) ? sc[j] : -INFINITY;
        }
      }
      float top = sc[0];
#pragma unroll
      for (int j = 1; j < NK; ++j) top = fmaxf(top, sc[j]);
      top = max_over_lane_bits_16_32(top) * a.scale_log2;
      const bool raise = top > m_run[rt] + kRaise;
      if (__any(raise)) {
        const float m_new = raise ? top : m_run[rt];
        const float alpha = raise ? __builtin_amdgcn_exp2f(m_run[rt] - m_new) : 1.f;
        m_run[rt] = m_new;
        l_run[rt] *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float al = __shfl(alpha, 4 * g + i, 64);
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) acc[rt][nb][i] *= al;
        }
      }
      const float ref = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
      bf16 p[NK];
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        const float e = __builtin_amdgcn_exp2f(fmaf(sc[j], a.scale_log2, -ref));
        p[j] = static_cast<bf16>(e);                           // the weights in bf16, as the matrix cores take them; their fp32 values are summed
        l_run[rt] += e;
      }
      if constexpr (ONE) {
        const bf16 z = static_cast<bf16>(0.f);
        const bool second = r16 >= 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pa[rt][j] = second ? z : p[j];
          pa[rt][4 + j] = second ? p[j] : z;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) pa[rt][j] = p[j];
      }
    }
    // ---- O += P . V: the B operand (lane: d = 16 nb + r16, eight keys) out of transposing reads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      i16x4 half[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)(vtile + (16 * u + 4 * g + (r16 >> 2)) * VROW + (16 * nb + 4 * (r16 & 3)) * 2));
      const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[rt], vf, acc[rt][nb], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (!ONE) {
      for (; bad != 0; bad &= bad - 1) {
        const int at = __builtin_ctzll(bad), key = k0 + (at >> 1);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t p = sp.start + (row0 + 16 * rt + 4 * g + i) / a.group;
            if (key < s_hi && key <= p && (a.window == 0 || key > p - a.window)) {
#pragma unroll
              for (int nb = 0; nb < 4; ++nb) acc[rt][nb][i] = (nb >> 1) == (at & 1) ? __builtin_nanf("") : acc[rt][nb][i];
            }
          }
      }
    }
  }

  // ---- the wavefronts meet, a tile of rows at a time
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt > 0) __syncthreads();
    const float l = sum_over_lane_bits_16_32(l_run[rt]);
    if (g == 0) {
      s_m[wave][r16] = m_run[rt];
      s_l[wave][r16] = l;
    }
    float* const mine = reinterpret_cast<float*>(vtile);       // (this wavefront is past its last read of the tile)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int nb = 0; nb < 4; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(4 * g + i) * AROW + 16 * nb + r16] = acc[rt][nb][i];
    __syncthreads();
    // thread -> (row, every TPR-th of its 64 values)
    constexpr int NR = ONE ? 8 : 16, TPR = kNW * 64 / NR, DPT = 64 / TPR;
    const int er = tid / TPR, ed = tid % TPR, row = row0 + 16 * rt + er;
    if (er >= NR || row >= rows) continue;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kNW; ++w)
#pragma unroll
      for (int t = er; t < 16; t += NR) m_all = fmaxf(m_all, s_m[w][t]);
    const float ref = m_all == -INFINITY ? 0.f : m_all;
    float l_all = 0.f, o[DPT] = {};
#pragma unroll
    for (int w = 0; w < kNW; ++w)
#pragma unroll
      for (int t = er; t < 16; t += NR) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][t] - ref);       // (0 for a wavefront that saw no key)
        l_all += s_l[w][t] * f;
        const float* const from = reinterpret_cast<const float*>(vt + w * VTILE) + t * AROW + ed;
#pragma unroll
        for (int j = 0; j < DPT; ++j) o[j] += from[TPR * j] * f;
      }
    const int i = row / a.group, head = kvh * a.group + row - i * a.group;
    if (a.splits > 1) {
      float* const p = a.part + (((static_cast<int64_t>(split) * a.batch + b) * a.n_q + i) * (a.n_kv_heads * a.group) + head) * PART;
#pragma unroll
      for (int j = 0; j < DPT; ++j) p[ed + TPR * j] = o[j];
      if (ed == 0) {
        p[64] = m_all;
        p[65] = l_all;
      }
      continue;
    }
    const float f = mx_norm(a, head, m_all, l_all);
    bf16* const to = a.out + b * a.out_bs + i * a.out_ts + head * 64;
#pragma unroll
    for (int j = 0; j < DPT; ++j) to[ed + TPR * j] = static_cast<bf16>(o[j] * f);
  }
}

// A wavefront per (batch row, query, head): the splits' records and the sink. Lane s has the (max, sum) of split s.
__global__ __launch_bounds__(64) void mxfp4_attn_reduce_kernel(MxAttnArgs a, int rows_per_group) {
  const int lane = threadIdx.x;
  const int n_heads = a.n_kv_heads * a.group;
  unsigned id = blockIdx.x;
  const int head = id % n_heads;
  id /= n_heads;
  const int i = id % a.n_q, b = id / a.n_q;
  const int kvh = head / a.group, row = i * a.group + head - kvh * a.group, row0 = row / rows_per_group * rows_per_group;
  const int64_t stride = static_cast<int64_t>(a.batch) * a.n_q * n_heads * PART;
  const float* const p0 = a.part + ((static_cast<int64_t>(b) * a.n_q + i) * n_heads + head) * PART;
  // requested before the start position is known; what splits that take no part have there is not used
  const float m_raw = lane < a.splits ? p0[lane * stride + 64] : -INFINITY, l_raw = lane < a.splits ? p0[lane * stride + 65] : 0.f;
  float v[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = p0[(u < a.splits ? u : a.splits - 1) * stride + lane];
  const int live = mx_span(a, b, row0, row0 + rows_per_group - 1).live;
  const float m_s = lane < live ? m_raw : -INFINITY;
  const float m_all = wave_max(m_s);
  const float f_s = __builtin_amdgcn_exp2f(m_s - (m_all == -INFINITY ? 0.f : m_all));
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
  const float f = mx_norm(a, head, m_all, l_all);
  a.out[b * a.out_bs + i * a.out_ts + static_cast<int64_t>(head) * 64 + lane] = static_cast<bf16>(o * f);
}

}  // namespace tllm

using namespace tllm;

namespace {
struct MxAttnPlan {
  bool one;
  int tiles, row_groups, splits, fill, keys_shift;
};
constexpr int kFill = 1024;           // workgroups that fill the CUs
constexpr int kKeysShift = 11;

MxAttnPlan mx_attn_plan(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window) {
  MxAttnPlan p;
  const int64_t rows = n_q * group;
  p.one = n_q == 1 && group <= 8;
  p.tiles = p.one || rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int rb = p.one ? 8 : 16 * p.tiles;
  p.row_groups = (int)((rows + rb - 1) / rb);
  const int64_t span = (int64_t)window + (rb + group - 1) / group;          // keys that a workgroup's queries can see together
  const int64_t ctx = window > 0 && span < n_slots ? span : n_slots;
  const int64_t units = batch * n_kv_heads * p.row_groups;
  p.fill = (int)((kFill + units - 1) / units);
  p.keys_shift = kKeysShift;
  p.splits = mx_attn_splits(p.fill, (int)(ctx > 0 ? ctx : 1), p.keys_shift);
  return p;
}

int64_t mx_attn_ctx(int64_t n_slots, int64_t hint) { return hint > 0 && hint < n_slots ? hint : n_slots; }
}  // namespace

extern "C" int tllm_mxfp4_attention_splits(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window, int64_t kv_len_hint) {
  if (batch < 1 || n_q < 1 || n_slots < 1 || n_kv_heads < 1 || group < 1 || window < 0) return 0;
  return mx_attn_plan(batch, n_q, mx_attn_ctx(n_slots, kv_len_hint), n_kv_heads, group, window).splits;
}

extern "C" int64_t tllm_mxfp4_attention_workspace_bytes(int64_t batch, int64_t n_q, int64_t n_slots, int n_kv_heads, int group, int window, int64_t kv_len_hint) {
  const int s = tllm_mxfp4_attention_splits(batch, n_q, n_slots, n_kv_heads, group, window, kv_len_hint);
  return s > 1 ? (int64_t)s * batch * n_q * n_kv_heads * group * PART * 4 : 0;
}

template <int RT, bool ONE>
static void launch(const MxAttnArgs& a, unsigned wgs, hipStream_t st) {
  hipLaunchKernelGGL((mxfp4_attn_kernel<RT, ONE>), dim3(wgs), dim3(kNW * 64), 0, st, a);
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
  a.keys_shift = p.keys_shift;
  a.scale_log2 = sm_scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.one) launch<1, true>(a, (unsigned)wgs, st);
  else if (p.tiles == 1) launch<1, false>(a, (unsigned)wgs, st);
  else if (p.tiles == 2) launch<2, false>(a, (unsigned)wgs, st);
  else launch<4, false>(a, (unsigned)wgs, st);
  const int rc = check_launch("mxfp4_attention");
  if (rc != TLLM_OK || p.splits == 1) return rc;
  hipLaunchKernelGGL(mxfp4_attn_reduce_kernel, dim3((unsigned)(batch * n_q * n_heads)), dim3(64), 0, st, a, p.one ? 8 : 16 * p.tiles);
  return check_launch("mxfp4_attention(reduce)");
}
