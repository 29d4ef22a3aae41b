// Products with MXFP4 weights: the entry points, and the weighted sum over a token's experts.
#include "mx_common.h"

namespace tllm {

// out[t, n] = residual[t, n] + sum_j weights[t, j] pairs[t top + j, n], in the order of j, in fp32, rounded once. A thread takes V
// neighbours of a token, four where rows are whole fours; up to four experts' loads leave together. 2000 tokens of 2880 and four
// experts, 115 MB: 17.5 us, 6.6 TB/s (the pairs are in the Infinity Cache still; an element at a time 35). The pairs stay in fp32: as bf16
// they would be half the bytes, 8 us, and a second rounding in every result.
template <int V>
__global__ __launch_bounds__(256) void moe_combine_kernel(const float* __restrict__ pairs, const float* __restrict__ weights, const bf16* residual,
                                                          int64_t res_stride, bf16* out, int64_t out_stride, int n, int top, int per_row) {
  typedef __attribute__((__vector_size__(V * sizeof(float)))) float fv;
  typedef __attribute__((__vector_size__(V * sizeof(bf16)))) bf16 bv;
  const int64_t t = blockIdx.x / per_row;
  const int c = ((blockIdx.x % per_row) * 256 + threadIdx.x) * V;
  if (c >= n) return;
  float v[V] = {};
  if (residual) {
    const bv r = *reinterpret_cast<const bv*>(residual + t * res_stride + c);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = static_cast<float>(r[i]);
  }
  for (int j0 = 0; j0 < top; j0 += 4) {
    fv p[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = t * top + (j0 + j < top ? j0 + j : top - 1);
      p[j] = *reinterpret_cast<const fv*>(pairs + at * n + c);
      w[j] = weights[at];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j0 + j < top)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = fmaf(w[j], p[j][i], v[i]);
  }
  bv o;
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = static_cast<bf16>(v[i]);
  *reinterpret_cast<bv*>(out + t * out_stride + c) = o;
}

static int product(const MxArgs& a, int mode, bool a4, hipStream_t st) {
  if (a4) return mx_tiles4_take(a) ? mx_tiles4(a, st) : mx_stream(a, mode, true, st);
  return mx_tiles_take(a) ? mx_tiles(a, mode, st) : mx_stream(a, mode, false, st);
}

static int weight_ok(const char* what, const void* w, const void* ws, int64_t experts, int64_t k, int64_t n) {
  TLLM_REQUIRE(n >= 1 && k >= 32 && k % 32 == 0, TLLM_E_SHAPE, "%s: a weight of %lld x %lld values; rows of whole blocks of 32 are supported", what, (long long)n, (long long)k);
  // (a workgroup keeps the scale bytes of at least sixteen weight rows in LDS)
  TLLM_REQUIRE(k <= (1 << 18) && n <= (1 << 24), TLLM_E_SHAPE, "%s: a weight of %lld x %lld values is too large", what, (long long)n, (long long)k);
  TLLM_REQUIRE(experts >= 1, TLLM_E_ARG, "%s: %lld experts", what, (long long)experts);
  TLLM_REQUIRE(w && ws, TLLM_E_ARG, "%s: null pointer", what);
  TLLM_REQUIRE(aligned16(w) && aligned16(ws), TLLM_E_ALIGN, "%s: blocks and scales must be 16-byte aligned", what);
  return TLLM_OK;
}

// Bytes of x have 32-bit offsets: from its beginning where rows are gathered, from a tile's first row (of 128 at most) otherwise.
static int rows_ok(const char* what, const void* x, int64_t rows, int64_t pitch, int64_t row_bytes, bool gathered) {
  TLLM_REQUIRE(x, TLLM_E_ARG, "%s: null pointer", what);
  TLLM_REQUIRE(rows == 1 || pitch >= row_bytes, TLLM_E_ARG, "%s: rows of %lld bytes, %lld apart", what, (long long)row_bytes, (long long)pitch);
  TLLM_REQUIRE(aligned16(x) && (rows == 1 || pitch % 16 == 0), TLLM_E_ALIGN, "%s: rows of x must be 16-byte aligned", what);
  const int64_t together = gathered || rows < 128 ? rows : 128;
  TLLM_REQUIRE(together - 1 <= (int64_t)(MX_NONE - row_bytes) / (pitch > 0 ? pitch : 1), TLLM_E_SHAPE, "%s: %lld rows of x span 4 GiB or more", what,
               (long long)together);
  return TLLM_OK;
}

}  // namespace tllm

using namespace tllm;

#define TLLM_TRY(call)                 \
  do {                                 \
    const int rc_ = (call);            \
    if (rc_ != TLLM_OK) return rc_;    \
  } while (0)

extern "C" int tllm_mxfp4_linear_bf16(const void* x, const void* x_scales, int64_t x_row_stride, const void* w_blocks, const void* w_scales, const void* bias,
                                      void* out, int64_t out_row_stride, int64_t rows, int64_t in_dim, int64_t out_dim, void* stream) {
  TLLM_REQUIRE(rows >= 0 && rows < (1ll << 31), TLLM_E_ARG, "mxfp4_linear: %lld rows", (long long)rows);
  if (rows == 0) return TLLM_OK;
  TLLM_TRY(weight_ok("mxfp4_linear", w_blocks, w_scales, 1, in_dim, out_dim));
  const int64_t row_bytes = x_scales ? in_dim / 2 : in_dim * 2, pitch = x_scales ? row_bytes : x_row_stride * 2;
  TLLM_TRY(rows_ok("mxfp4_linear", x, rows, pitch, row_bytes, false));
  TLLM_REQUIRE(out, TLLM_E_ARG, "mxfp4_linear: null pointer");
  TLLM_REQUIRE(aligned16(x_scales), TLLM_E_ALIGN, "mxfp4_linear: x_scales must be 16-byte aligned");
  TLLM_REQUIRE(rows == 1 || out_row_stride >= out_dim, TLLM_E_ARG, "mxfp4_linear: out_row_stride %lld < %lld", (long long)out_row_stride, (long long)out_dim);
  MxArgs a{};
  a.x = x;
  a.x_scales = static_cast<const unsigned char*>(x_scales);
  a.x_pitch = pitch;
  a.w = static_cast<const unsigned char*>(w_blocks);
  a.w_scales = static_cast<const unsigned char*>(w_scales);
  a.bias = static_cast<const bf16*>(bias);
  a.out = out;
  a.out_stride = out_row_stride;
  a.rows = a.tokens = rows;
  a.experts = a.top = 1;
  a.n = static_cast<int>(out_dim);
  a.k = static_cast<int>(in_dim);
  return product(a, kMxLinear, x_scales != nullptr, static_cast<hipStream_t>(stream));
}

static int experts_args(const char* what, MxArgs* a, bool gathered, const void* x, int64_t x_row_stride, int64_t x_rows, const int32_t* order, const int32_t* offsets,
                        const void* w_blocks, const void* w_scales, const void* bias, int64_t tokens, int n_experts, int top, int64_t k, int64_t n) {
  TLLM_REQUIRE(top >= 1 && n_experts >= top, TLLM_E_SHAPE, "%s: top %d of %d experts", what, top, n_experts);
  TLLM_REQUIRE(tokens * top < (1ll << 31), TLLM_E_SHAPE, "%s: %lld tokens x %d are too many", what, (long long)tokens, top);
  TLLM_TRY(weight_ok(what, w_blocks, w_scales, n_experts, k, n));
  TLLM_TRY(rows_ok(what, x, x_rows, x_row_stride * 2, k * 2, gathered));
  TLLM_REQUIRE(order && offsets, TLLM_E_ARG, "%s: null pointer", what);
  a->x = x;
  a->x_pitch = x_row_stride * 2;
  a->w = static_cast<const unsigned char*>(w_blocks);
  a->w_scales = static_cast<const unsigned char*>(w_scales);
  a->bias = static_cast<const bf16*>(bias);
  a->order = order;
  a->offsets = offsets;
  a->rows = tokens * top;
  a->tokens = tokens;
  a->experts = n_experts;
  a->top = top;
  a->n = static_cast<int>(n);
  a->k = static_cast<int>(k);
  return TLLM_OK;
}

extern "C" int tllm_moe_mlp1_bf16(const void* x, int64_t x_row_stride, const int32_t* order, const int32_t* offsets, const void* w_blocks, const void* w_scales,
                                  const void* bias, void* h, int64_t h_row_stride, int64_t tokens, int n_experts, int top, int64_t hidden, int64_t inner,
                                  float alpha, float limit, int has_limit, void* stream) {
  TLLM_REQUIRE(tokens >= 0, TLLM_E_ARG, "moe_mlp1: tokens %lld", (long long)tokens);
  if (tokens == 0) return TLLM_OK;
  MxArgs a{};
  TLLM_TRY(experts_args("moe_mlp1", &a, true, x, x_row_stride, tokens, order, offsets, w_blocks, w_scales, bias, tokens, n_experts, top, hidden, 2 * inner));
  TLLM_REQUIRE(h && h_row_stride >= inner, TLLM_E_ARG, "moe_mlp1: null pointer, or h_row_stride %lld < %lld", (long long)h_row_stride, (long long)inner);
  TLLM_REQUIRE(!has_limit || limit >= 0.f, TLLM_E_ARG, "moe_mlp1: limit %g", (double)limit);
  a.out = h;
  a.out_stride = h_row_stride;
  a.alpha = alpha;
  a.limit = has_limit ? limit : __builtin_inff();
  return product(a, kMxSwiglu, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t tllm_moe_mlp2_workspace_bytes(int64_t tokens, int top, int64_t hidden) { return tokens > 0 && top > 0 && hidden > 0 ? tokens * top * hidden * 4 : 0; }

extern "C" int tllm_moe_mlp2_bf16(const void* h, int64_t h_row_stride, const int32_t* order, const int32_t* offsets, const float* weights, const void* w_blocks,
                                  const void* w_scales, const void* bias, const void* residual, int64_t res_row_stride, void* out, int64_t out_row_stride,
                                  void* workspace, int64_t workspace_bytes, int64_t tokens, int n_experts, int top, int64_t inner, int64_t hidden, void* stream) {
  TLLM_REQUIRE(tokens >= 0, TLLM_E_ARG, "moe_mlp2: tokens %lld", (long long)tokens);
  if (tokens == 0) return TLLM_OK;
  MxArgs a{};
  TLLM_TRY(experts_args("moe_mlp2", &a, false, h, h_row_stride, tokens * top, order, offsets, w_blocks, w_scales, bias, tokens, n_experts, top, inner, hidden));
  TLLM_REQUIRE(weights && out, TLLM_E_ARG, "moe_mlp2: null pointer");
  TLLM_REQUIRE(tokens == 1 || (out_row_stride >= hidden && (!residual || res_row_stride >= hidden)), TLLM_E_ARG, "moe_mlp2: rows of %lld values, %lld (residual %lld) apart",
               (long long)hidden, (long long)out_row_stride, (long long)res_row_stride);
  const int64_t need = tllm_moe_mlp2_workspace_bytes(tokens, top, hidden), per_row = (hidden + 255) / 256;
  TLLM_REQUIRE(tokens * per_row < (1ll << 24), TLLM_E_SHAPE, "moe_mlp2: %lld tokens of %lld values are too many", (long long)tokens, (long long)hidden);
  TLLM_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace), TLLM_E_ARG, "moe_mlp2: a 16-byte aligned workspace of %lld bytes is needed, got %lld",
               (long long)need, (long long)workspace_bytes);
  a.out = workspace;
  a.out_stride = hidden;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TLLM_TRY(product(a, kMxPairs, false, st));
  auto combine = [&](auto* kernel, int64_t per_row) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tokens * per_row)), dim3(256), 0, st, static_cast<const float*>(workspace), weights,
                       static_cast<const bf16*>(residual), res_row_stride, static_cast<bf16*>(out), out_row_stride, (int)hidden, top, (int)per_row);
  };
  auto fours = [](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 8 == 0 && stride % 4 == 0; };
  if (hidden % 4 == 0 && fours(out, out_row_stride) && (!residual || fours(residual, res_row_stride))) combine(moe_combine_kernel<4>, (hidden + 1023) / 1024);
  else combine(moe_combine_kernel<1>, per_row);
  return check_launch("moe_mlp2");
}
