// A KV cache in MXFP4: keys and values quantised as they are written, and read back.
//
// The cache is codes [batch, slots, KV heads, head_dim / 32][16] and scale bytes [batch, slots, KV heads, head_dim / 32], once for keys and once
// for values, with strides: where a head's slots are next to each other (what ops.mxfp4_cache allocates), a head of 64 has 32 bytes of
// codes and two of scales per slot, and attention reads them as one stream. Values and scales are those of the quantisation of weights:
// per 32 values e = max(floor(log2 max|x|) - 2, -127), codes to the nearest e2m1 value of x 2^-e.
//
// A thread takes eight values (reading many, four times eight). A workgroup stays with one head: eight neighbours have a whole line of k or v
// (64 values of bf16), a wavefront 256 neighbouring bytes of the head's codes.
// Bound by the bytes, in a graph over several caches and outputs in turn: 8 rows of 4096 tokens of eight heads written in 21.0 us (85 MB, 4.05 TB/s; a
// large copy reaches 4.8), read in 15.5 (5.5; 13.1 into outputs that the chip's caches still hold); 8192 tokens 7.2 and 4.8; one token of eight rows 2.5
// and 2.6, a launch.
#include "mx_cache.h"
#include "mx_quantize.h"

namespace tllm {

// Of one head's `tokens` x `eights` eights of values, the one that place `i` is.
struct MxPlace {
  unsigned eights, shift;                 // head_dim / 8, its logarithm (32: it has none)
  __device__ __forceinline__ void split(unsigned i, unsigned* t, unsigned* c) const {
    *t = shift < 32 ? i >> shift : i / eights;
    *c = i - *t * eights;
  }
};

struct MxWriteArgs {
  const char* x[2];                       // k and v, [batch, tokens, heads, head_dim] with strides in bytes
  int64_t xs_batch[2], xs_head[2];
  unsigned xs_token[2];
  MxCache cache;
  const void* offset;
  const void* lengths;                    // or NULL
  int offset_is_i64, offset_stride, lengths_is_i64, lengths_stride;
  int64_t first;                          // the first of this launch's tokens
  MxPlace place;
  unsigned n;                             // eights of a head: tokens x eights
};

// The tokens of a launch are addressed with 32-bit offsets from a head's first one (the host sees to it that they are enough).
template <class T>
__global__ __launch_bounds__(256) void mxfp4_cache_write_kernel(MxWriteArgs a) {
  // (heads fastest: the workgroups that run at a time have whole tokens between them, which lie together in k, v and the outputs)
  const int64_t b = blockIdx.z, h = blockIdx.x >> 1;
  const int kv = blockIdx.x & 1;
  const unsigned i = blockIdx.y * 256u + threadIdx.x;
  unsigned t, c;
  a.place.split(i < a.n ? i : a.n - 1, &t, &c);
  Eight<T> e;
  e.load(a.x[kv] + b * a.xs_batch[kv] + h * a.xs_head[kv] + (t * a.xs_token[kv] + c * 8u * static_cast<unsigned>(sizeof(T))));
  // slots outside the cache and tokens behind the sequence's end are left as they are: the tokens from .. to - 1 are written
  const int64_t far = 1ll << 36;                                       // (beyond any slot and any token; its bytes stay within 64 bits)
  auto held = [&](int64_t x) { return x < -far ? -far : x > far ? far : x; };
  const int64_t slot0 = held(mx_row_int(a.offset, a.offset_is_i64, b * a.offset_stride)) + a.first;      // of the launch's first token
  int64_t to = a.cache.n_slots - slot0;
  if (a.lengths) {
    const int64_t length = held(mx_row_int(a.lengths, a.lengths_is_i64, b * a.lengths_stride)) - a.first;
    to = length < to ? length : to;
  }
  unsigned char* const codes_to = const_cast<unsigned char*>(a.cache.blocks[kv]) + b * a.cache.bs + h * a.cache.hs + slot0 * a.cache.ts;
  unsigned char* const scales_to = const_cast<unsigned char*>(a.cache.scales[kv]) + b * a.cache.sbs + h * a.cache.shs + slot0 * a.cache.sts;
  unsigned byte;
  const unsigned codes = mx_quantize8(e, &byte);
  if (i >= a.n || t < -slot0 || t >= to) return;
  *reinterpret_cast<unsigned*>(codes_to + (t * static_cast<unsigned>(a.cache.ts) + c * 4)) = codes;
  if ((c & 3) == 0) scales_to[t * static_cast<unsigned>(a.cache.sts) + (c >> 2)] = static_cast<unsigned char>(byte);
}

struct MxReadArgs {
  char* out[2];                           // k and v, [batch, tokens, heads, head_dim], strides in bytes
  int64_t out_batch, out_head;
  unsigned out_token;
  MxCache cache;
  int64_t first;                          // the first slot
  MxPlace place;
  unsigned n;
};

template <int U>
__global__ __launch_bounds__(256) void mxfp4_cache_read_kernel(MxReadArgs a) {
  const int64_t b = blockIdx.z, h = blockIdx.x >> 1;
  const int kv = blockIdx.x & 1;
  const unsigned i0 = blockIdx.y * (256u * U) + threadIdx.x;
  const unsigned char* const from = a.cache.blocks[kv] + b * a.cache.bs + h * a.cache.hs + a.first * a.cache.ts;
  const unsigned char* const sc = a.cache.scales[kv] + b * a.cache.sbs + h * a.cache.shs + a.first * a.cache.sts;
  unsigned codes[U], byte[U], t[U], c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned i = i0 + 256u * u;
    a.place.split(i < a.n ? i : a.n - 1, &t[u], &c[u]);
    codes[u] = *reinterpret_cast<const unsigned*>(from + (t[u] * static_cast<unsigned>(a.cache.ts) + c[u] * 4));
    byte[u] = sc[t[u] * static_cast<unsigned>(a.cache.sts) + (c[u] >> 2)];
  }
  char* const to = a.out[kv] + b * a.out_batch + h * a.out_head;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bf16x8 v = mx_bf16x8(codes[u], __builtin_bit_cast(float, byte[u] << 23));
    if (i0 + 256u * u < a.n) __builtin_nontemporal_store(v, reinterpret_cast<bf16x8*>(to + (t[u] * a.out_token + c[u] * 16)));
  }
}

int mx_cache_of(const TllmMxCache* c, const char* what, MxCache* out) {
  TLLM_REQUIRE(c != nullptr, TLLM_E_ARG, "%s: the cache is NULL", what);
  TLLM_REQUIRE(c->batch >= 0 && c->batch <= 65535 && c->n_slots >= 0 && c->n_slots < (1ll << 30) && c->n_kv_heads >= 1 && c->n_kv_heads <= 65535, TLLM_E_SHAPE,
               "%s: a cache of %lld x %lld slots x %d heads", what, (long long)c->batch, (long long)c->n_slots, c->n_kv_heads);
  TLLM_REQUIRE(c->head_dim >= 32 && c->head_dim % 32 == 0 && c->head_dim <= 1024, TLLM_E_SHAPE, "%s: head_dim %d, multiples of 32 up to 1024 are supported", what, c->head_dim);
  if (c->batch == 0 || c->n_slots == 0) return TLLM_OK;
  TLLM_REQUIRE(c->k_blocks && c->k_scales && c->v_blocks && c->v_scales, TLLM_E_ARG, "%s: the cache has a null pointer", what);
  TLLM_REQUIRE(aligned16(c->k_blocks) && aligned16(c->v_blocks) && c->batch_stride % 16 == 0 && c->slot_stride % 16 == 0 && c->head_stride % 16 == 0, TLLM_E_ALIGN,
               "%s: the cache's blocks must be 16-byte aligned", what);
  // (a block of 64 slots is addressed with 32-bit offsets)
  TLLM_REQUIRE(c->batch_stride >= 0 && c->head_stride >= 0 && c->scale_batch_stride >= 0 && c->scale_head_stride >= 0 && c->slot_stride >= 0 &&
                   c->slot_stride < (1ll << 24) && c->scale_slot_stride >= 0 && c->scale_slot_stride < (1ll << 24),
               TLLM_E_SHAPE, "%s: strides of %lld and %lld bytes between slots (up to 2^24 are supported)", what, (long long)c->slot_stride,
               (long long)c->scale_slot_stride);
  *out = MxCache{{static_cast<const unsigned char*>(c->k_blocks), static_cast<const unsigned char*>(c->v_blocks)},
                 {static_cast<const unsigned char*>(c->k_scales), static_cast<const unsigned char*>(c->v_scales)},
                 c->batch_stride, c->head_stride, c->slot_stride, c->scale_batch_stride, c->scale_head_stride, c->scale_slot_stride, (int)c->n_slots};
  return TLLM_OK;
}

}  // namespace tllm

using namespace tllm;

namespace {
MxPlace place_of(int eights) { return MxPlace{(unsigned)eights, (eights & (eights - 1)) == 0 ? (unsigned)__builtin_ctz(eights) : 32u}; }

// f(first token, tokens, first row, grid) for each launch: tokens whose places in a head and whose offsets, `stride` bytes from one to the next at
// most, 32 bits hold; rows that keep a grid below 2^32 threads.
template <class F>
int in_launches(int64_t batch, int64_t tokens, int heads, int eights, int per_thread, int64_t stride, F f) {
  int64_t most = (1ll << 23) / eights;                         // (at most 32768 workgroups of 256, of the 65535 that a grid's second dimension takes)
  const int64_t fits = (1ll << 22) / heads * 256 / eights;     // (heads are up to 65535: one token at least)
  most = most < fits ? most : fits;
  if (stride > 0 && most > (1ll << 31) / stride) most = (1ll << 31) / stride > 0 ? (1ll << 31) / stride : 1;
  for (int64_t t = 0; t < tokens; t += most) {
    const int64_t m = tokens - t < most ? tokens - t : most;
    const int64_t blocks = (m * eights + 256 * per_thread - 1) / (256 * per_thread);
    int64_t rows = (1ll << 23) / (2 * blocks * heads);
    rows = rows > 0 ? rows : 1;
    for (int64_t b = 0; b < batch; b += rows) {
      const dim3 grid(2 * (unsigned)heads, (unsigned)blocks, (unsigned)(batch - b < rows ? batch - b : rows));
      if (const int rc = f(t, m, b, grid); rc != TLLM_OK) return rc;
    }
  }
  return TLLM_OK;
}
}  // namespace

extern "C" int tllm_mxfp4_cache_write(const TllmMxCache* cache, const void* k, const void* v, int type, const int64_t* k_strides, const int64_t* v_strides,
                                      int64_t tokens, const void* offset, int offset_is_i64, int offset_per_row, const void* lengths, int lengths_is_i64,
                                      int lengths_per_row, void* stream) {
  MxWriteArgs a{};
  if (const int rc = mx_cache_of(cache, "mxfp4_cache_write", &a.cache); rc != TLLM_OK) return rc;
  TLLM_REQUIRE(type == TLLM_BF16 || type == TLLM_F16 || type == TLLM_F32, TLLM_E_ARG, "mxfp4_cache_write: type %d", type);
  TLLM_REQUIRE(tokens >= 0, TLLM_E_ARG, "mxfp4_cache_write: %lld tokens", (long long)tokens);
  if (tokens == 0 || cache->batch == 0 || cache->n_slots == 0) return TLLM_OK;
  TLLM_REQUIRE(k && v && offset && k_strides && v_strides, TLLM_E_ARG, "mxfp4_cache_write: null pointer");
  const int64_t size = type == TLLM_F32 ? 4 : 2;
  TLLM_REQUIRE(aligned16(k) && aligned16(v), TLLM_E_ALIGN, "mxfp4_cache_write: k and v must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    TLLM_REQUIRE(k_strides[i] * size % 16 == 0 && v_strides[i] * size % 16 == 0, TLLM_E_ALIGN, "mxfp4_cache_write: heads of k and v must be 16-byte aligned");
  const int heads = cache->n_kv_heads, eights = cache->head_dim / 8;
  TLLM_REQUIRE((cache->batch == 1 || (cache->batch_stride > 0 && cache->scale_batch_stride > 0)) && (heads == 1 || (cache->head_stride > 0 && cache->scale_head_stride > 0)) &&
                   (cache->n_slots == 1 || (cache->slot_stride > 0 && cache->scale_slot_stride > 0)),
               TLLM_E_ARG, "mxfp4_cache_write: the cache's rows share memory");
  int64_t stride = a.cache.ts > a.cache.sts ? a.cache.ts : a.cache.sts;
  for (int i = 0; i < 2; ++i) {
    const int64_t* const xs = i == 0 ? k_strides : v_strides;
    a.x[i] = static_cast<const char*>(i == 0 ? k : v);
    a.xs_batch[i] = xs[0] * size;
    a.xs_token[i] = (unsigned)(tokens > 1 ? xs[1] * size : 0);
    a.xs_head[i] = xs[2] * size;
    TLLM_REQUIRE(tokens == 1 || (xs[1] >= 0 && xs[1] < (1ll << 31) / size), TLLM_E_SHAPE, "mxfp4_cache_write: %lld values from token to token", (long long)xs[1]);
    stride = stride > a.xs_token[i] ? stride : a.xs_token[i];
  }
  a.offset = offset;
  a.offset_is_i64 = offset_is_i64;
  a.offset_stride = offset_per_row != 0;
  a.lengths = lengths;
  a.lengths_is_i64 = lengths_is_i64;
  a.lengths_stride = lengths_per_row != 0;
  a.place = place_of(eights);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const MxWriteArgs all = a;
  return in_launches(cache->batch, tokens, heads, eights, 1, stride, [&](int64_t t, int64_t m, int64_t b, dim3 grid) {
    MxWriteArgs w = all;
    w.first = t;
    w.n = (unsigned)(m * eights);
    for (int i = 0; i < 2; ++i) {
      w.x[i] = all.x[i] + b * all.xs_batch[i] + t * all.xs_token[i];
      w.cache.blocks[i] = all.cache.blocks[i] + b * all.cache.bs;
      w.cache.scales[i] = all.cache.scales[i] + b * all.cache.sbs;
    }
    w.offset = static_cast<const char*>(offset) + b * all.offset_stride * (offset_is_i64 ? 8 : 4);
    if (lengths) w.lengths = static_cast<const char*>(lengths) + b * all.lengths_stride * (lengths_is_i64 ? 8 : 4);
    if (type == TLLM_BF16) hipLaunchKernelGGL(mxfp4_cache_write_kernel<bf16>, grid, dim3(256), 0, st, w);
    else if (type == TLLM_F16) hipLaunchKernelGGL(mxfp4_cache_write_kernel<_Float16>, grid, dim3(256), 0, st, w);
    else hipLaunchKernelGGL(mxfp4_cache_write_kernel<float>, grid, dim3(256), 0, st, w);
    return check_launch("mxfp4_cache_write");
  });
}

extern "C" int tllm_mxfp4_cache_read_bf16(const TllmMxCache* cache, int64_t first, int64_t tokens, void* k_out, void* v_out, void* stream) {
  MxReadArgs a{};
  if (const int rc = mx_cache_of(cache, "mxfp4_cache_read", &a.cache); rc != TLLM_OK) return rc;
  TLLM_REQUIRE(first >= 0 && tokens >= 0 && first <= cache->n_slots && tokens <= cache->n_slots - first, TLLM_E_SHAPE,
               "mxfp4_cache_read: slots %lld .. %lld of %lld", (long long)first, (long long)(first + tokens), (long long)cache->n_slots);
  if (tokens == 0 || cache->batch == 0) return TLLM_OK;
  TLLM_REQUIRE(k_out && v_out, TLLM_E_ARG, "mxfp4_cache_read: null pointer");
  TLLM_REQUIRE(aligned16(k_out) && aligned16(v_out), TLLM_E_ALIGN, "mxfp4_cache_read: the outputs must be 16-byte aligned");
  const int heads = cache->n_kv_heads, eights = cache->head_dim / 8;
  a.out_head = 2 * cache->head_dim;
  a.out_token = (unsigned)(a.out_head * heads);
  a.out_batch = static_cast<int64_t>(a.out_token) * tokens;
  a.place = place_of(eights);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Four eights a thread, and stores that pass the caches by, where a head has more than a workgroup's worth: 8192 tokens of eight heads 4.8 us, one a
  // thread 6.4, ordinary stores 5.7; 8 x 4096 15.5, 16.6, 16.0.
  const bool many = tokens * eights > 1024;
  const int64_t stride = a.out_token > a.cache.ts ? (a.out_token > a.cache.sts ? a.out_token : a.cache.sts) : a.cache.ts > a.cache.sts ? a.cache.ts : a.cache.sts;
  const MxReadArgs all = a;
  return in_launches(cache->batch, tokens, heads, eights, many ? 4 : 1, stride, [&](int64_t t, int64_t m, int64_t b, dim3 grid) {
    MxReadArgs r = all;
    r.first = first + t;
    for (int i = 0; i < 2; ++i) {
      r.out[i] = static_cast<char*>(i == 0 ? k_out : v_out) + b * all.out_batch + t * all.out_token;
      r.cache.blocks[i] = all.cache.blocks[i] + b * all.cache.bs;
      r.cache.scales[i] = all.cache.scales[i] + b * all.cache.sbs;
    }
    r.n = (unsigned)(m * eights);
    if (many) hipLaunchKernelGGL(mxfp4_cache_read_kernel<4>, grid, dim3(256), 0, st, r);
    else hipLaunchKernelGGL(mxfp4_cache_read_kernel<1>, grid, dim3(256), 0, st, r);
    return check_launch("mxfp4_cache_read");
  });
}
