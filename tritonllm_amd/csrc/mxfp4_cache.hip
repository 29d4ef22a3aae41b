// A KV cache in MXFP4: keys and values quantised as they are written, and read back.
//
// The cache is codes [batch, slots, KV heads, head_dim / 32][16] and scale bytes [batch, slots, KV heads, head_dim / 32], once for keys and once
// for values, with strides: where a head's slots are next to each other (what ops.mxfp4_cache allocates), a head of 64 has 32 bytes of
// codes and two of scales per slot, and attention reads them as one stream. Values and scales are those of the quantisation of weights:
// per 32 values e = max(floor(log2 max|x|) - 2, -127), codes to the nearest e2m1 value of x 2^-e.
//
// A thread takes eight values. The order of the threads is (head, token, eight of the head's values), so that eight neighbours read a
// whole line of k or v (64 values of bf16) and a wavefront writes 256 neighbouring bytes of codes of a head. The bytes bound both kernels
// once there are a few MB of them.
#include "mx_cache.h"
#include "mx_quantize.h"

namespace tllm {

struct MxWriteArgs {
  const void* x[2];                       // k and v, [batch, tokens, heads, head_dim] with strides in elements
  int64_t xs_batch[2], xs_token[2], xs_head[2];
  MxCache cache;
  const void* offset;
  const void* lengths;                    // or NULL
  int offset_is_i64, offset_stride, lengths_is_i64, lengths_stride;
  int64_t first;                          // the first of this launch's tokens
  unsigned tokens, eights;                // its tokens; head_dim / 8
  unsigned n;                             // threads of one row: heads x tokens x eights
};

template <class T>
__global__ __launch_bounds__(256) void mxfp4_cache_write_kernel(MxWriteArgs a) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.n) return;
  const int64_t b = blockIdx.y;
  const int kv = blockIdx.z;
  const unsigned row = i / a.eights, c = i - row * a.eights, h = row / a.tokens;
  const int64_t t = a.first + (row - h * a.tokens);
  // slots outside the cache and tokens behind the sequence's end are left as they are (the four lanes of a block agree)
  if (a.lengths && t >= mx_row_int(a.lengths, a.lengths_is_i64, b * a.lengths_stride)) return;
  const int64_t slot = mx_row_int(a.offset, a.offset_is_i64, b * a.offset_stride) + t;
  if (slot < 0 || slot >= a.cache.n_slots) return;
  Eight<T> e;
  e.load(static_cast<const T*>(a.x[kv]) + b * a.xs_batch[kv] + t * a.xs_token[kv] + static_cast<int64_t>(h) * a.xs_head[kv] + c * 8);
  unsigned byte;
  const unsigned codes = mx_quantize8(e, &byte);
  unsigned char* const to = const_cast<unsigned char*>(a.cache.blocks[kv]) + b * a.cache.bs + static_cast<int64_t>(h) * a.cache.hs + slot * a.cache.ts;
  *reinterpret_cast<unsigned*>(to + c * 4) = codes;
  unsigned char* const sc = const_cast<unsigned char*>(a.cache.scales[kv]) + b * a.cache.sbs + static_cast<int64_t>(h) * a.cache.shs + slot * a.cache.sts;
  if ((c & 3) == 0) sc[c >> 2] = static_cast<unsigned char>(byte);
}

struct MxReadArgs {
  bf16* out[2];                           // k and v, [batch, tokens, heads, head_dim]
  int64_t out_batch, out_token, out_head; // strides in elements
  MxCache cache;
  int64_t first;                          // the first slot
  unsigned tokens, eights, n;
};

__global__ __launch_bounds__(256) void mxfp4_cache_read_kernel(MxReadArgs a) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.n) return;
  const int64_t b = blockIdx.y;
  const int kv = blockIdx.z;
  const unsigned row = i / a.eights, c = i - row * a.eights, h = row / a.tokens;
  const int64_t t = row - h * a.tokens, slot = a.first + t;
  const unsigned codes = *reinterpret_cast<const unsigned*>(a.cache.blocks[kv] + b * a.cache.bs + static_cast<int64_t>(h) * a.cache.hs + slot * a.cache.ts + c * 4);
  const unsigned byte = a.cache.scales[kv][b * a.cache.sbs + static_cast<int64_t>(h) * a.cache.shs + slot * a.cache.sts + (c >> 2)];
  *reinterpret_cast<bf16x8*>(a.out[kv] + b * a.out_batch + t * a.out_token + static_cast<int64_t>(h) * a.out_head + c * 8) =
      mx_bf16x8(codes, __builtin_bit_cast(float, byte << 23));
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

// Tokens of a launch: a grid holds fewer than 2^32 threads, keys' and values' rows of all of the batch together.
static int64_t tokens_per_launch(int64_t batch, int heads, int eights) {
  const int64_t per_token = 2 * batch * heads * eights;
  return per_token < (1ll << 30) ? (1ll << 30) / per_token : 1;
}

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
  TLLM_REQUIRE(2 * cache->batch * heads * eights < (1ll << 31), TLLM_E_SHAPE, "mxfp4_cache_write: %lld x %d heads of %d are too many", (long long)cache->batch, heads, cache->head_dim);
  TLLM_REQUIRE((cache->batch == 1 || (cache->batch_stride > 0 && cache->scale_batch_stride > 0)) && (heads == 1 || (cache->head_stride > 0 && cache->scale_head_stride > 0)) &&
                   (cache->n_slots == 1 || (cache->slot_stride > 0 && cache->scale_slot_stride > 0)),
               TLLM_E_ARG, "mxfp4_cache_write: the cache's rows share memory");
  a.x[0] = k;
  a.x[1] = v;
  for (int i = 0; i < 2; ++i) {
    const int64_t* const s = i == 0 ? k_strides : v_strides;
    a.xs_batch[i] = s[0];
    a.xs_token[i] = s[1];
    a.xs_head[i] = s[2];
  }
  a.offset = offset;
  a.offset_is_i64 = offset_is_i64;
  a.offset_stride = offset_per_row != 0;
  a.lengths = lengths;
  a.lengths_is_i64 = lengths_is_i64;
  a.lengths_stride = lengths_per_row != 0;
  a.eights = eights;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = tokens_per_launch(cache->batch, heads, eights);
  for (int64_t t = 0; t < tokens; t += most) {
    a.first = t;
    a.tokens = (unsigned)(tokens - t < most ? tokens - t : most);
    a.n = a.tokens * eights * heads;
    const dim3 grid((a.n + 255) / 256, (unsigned)cache->batch, 2);
    if (type == TLLM_BF16)
      hipLaunchKernelGGL(mxfp4_cache_write_kernel<bf16>, grid, dim3(256), 0, st, a);
    else if (type == TLLM_F16)
      hipLaunchKernelGGL(mxfp4_cache_write_kernel<_Float16>, grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL(mxfp4_cache_write_kernel<float>, grid, dim3(256), 0, st, a);
    if (const int rc = check_launch("mxfp4_cache_write"); rc != TLLM_OK) return rc;
  }
  return TLLM_OK;
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
  TLLM_REQUIRE(2 * cache->batch * heads * eights < (1ll << 31), TLLM_E_SHAPE, "mxfp4_cache_read: %lld x %d heads of %d are too many", (long long)cache->batch, heads, cache->head_dim);
  a.out_head = cache->head_dim;
  a.out_token = a.out_head * heads;
  a.out_batch = a.out_token * tokens;
  a.eights = eights;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = tokens_per_launch(cache->batch, heads, eights);
  for (int64_t t = 0; t < tokens; t += most) {
    a.first = first + t;
    a.tokens = (unsigned)(tokens - t < most ? tokens - t : most);
    a.n = a.tokens * eights * heads;
    a.out[0] = static_cast<bf16*>(k_out) + t * a.out_token;
    a.out[1] = static_cast<bf16*>(v_out) + t * a.out_token;
    hipLaunchKernelGGL(mxfp4_cache_read_kernel, dim3((a.n + 255) / 256, (unsigned)cache->batch, 2), dim3(256), 0, st, a);
    if (const int rc = check_launch("mxfp4_cache_read"); rc != TLLM_OK) return rc;
  }
  return TLLM_OK;
}
