// dcf_int8.cu — the product of 8-bit matrices with scales for each token and
// channel:
//   out[t][c] = (sum over k of a[t][k] * b[c][k]) * a_scale[t] * b_scale[c] + bias[c]
// Sums of whole numbers are exact in 32 bits (2^14 * 131071 < 2^31), in any
// order, so a sum may be split and joined freely.
#include "dcf_quant.cuh"

namespace dcf {

namespace {

struct Int8Args {
  const int8_t* a;
  const int8_t* b;
  const float* a_scale;  // null: the sums themselves
  const float* b_scale;
  const float* bias;
  void* out;
  int out_dtype;
  int tokens, channels, depth;
  int64_t as, bs, os;
};

__device__ __forceinline__ void put(const Int8Args& g, int64_t t, int64_t c, int sum) {
  const int64_t at = t * g.os + c;
  if (g.out_dtype == DCF_I32) {
    ((int*)g.out)[at] = sum;
    return;
  }
  float v = __fmul_rn(__fmul_rn((float)sum, g.a_scale[t]), g.b_scale[c]);
  if (g.bias) v = __fadd_rn(v, g.bias[c]);
  if (g.out_dtype == DCF_F32) ((float*)g.out)[at] = v;
  else if (g.out_dtype == DCF_F16) ((__half*)g.out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)g.out)[at] = __float2bfloat16_rn(v);
}

constexpr int kTile = 64, kDeep = 64;

// 64 x 64 results to a block of 256 threads, sixteen to a thread.
__global__ void __launch_bounds__(256) int8_tile_kernel(const Int8Args g) {
  __shared__ __align__(16) uint32_t a[kDeep / 4][kTile + 1], b[kDeep / 4][kTile + 1];
  pdl_begin();
  const int64_t tiles = ((int64_t)g.channels + kTile - 1) / kTile, total = tiles * (((int64_t)g.tokens + kTile - 1) / kTile);
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int64_t t0 = i / tiles * kTile, c0 = i % tiles * kTile;
    int sum[4][4] = {};
    for (int k0 = 0; k0 < g.depth; k0 += kDeep) {
      auto fill = [&](uint32_t (&to)[kDeep / 4][kTile + 1], const int8_t* from, int64_t row0, int rows, int64_t stride) {
        for (int w = threadIdx.x; w < kTile * kDeep / 4; w += 256) {
          const int r = w / (kDeep / 4), k = w % (kDeep / 4);
          uint32_t v = 0;
          for (int e = 0; e < 4; e++)
            if (row0 + r < rows && k0 + 4 * k + e < g.depth)
              v |= (uint32_t)(uint8_t)from[(row0 + r) * stride + k0 + 4 * k + e] << (8 * e);
          to[k][r] = v;
        }
      };
      __syncthreads();
      fill(a, g.a, t0, g.tokens, g.as);
      fill(b, g.b, c0, g.channels, g.bs);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kDeep / 4; k++)
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
          for (int n = 0; n < 4; n++) sum[m][n] = __dp4a((int)a[k][y + 16 * m], (int)b[k][x + 16 * n], sum[m][n]);
    }
    for (int m = 0; m < 4; m++)
      for (int n = 0; n < 4; n++)
        if (t0 + y + 16 * m < g.tokens && c0 + x + 16 * n < g.channels) put(g, t0 + y + 16 * m, c0 + x + 16 * n, sum[m][n]);
  }
}

// The workspace: tokens of a float type as whole numbers, and their scales.
struct Layout {
  int64_t stride;
  size_t q, scale, bytes;
};

Layout layout_of(const dcf_int8_desc& d) {
  Layout l = {};
  if (d.a_dtype == DCF_I8) return l;
  auto take = [&](size_t bytes) {
    const size_t at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  l.stride = (int64_t)((d.depth + 15) / 16 * 16);
  l.q = take((size_t)d.tokens * l.stride);
  l.scale = take((size_t)d.tokens * 4);
  return l;
}

}  // namespace

int int8_desc_check(const dcf_int8_desc* d) {
  auto bad = [](const char* m) { return record_error(DCF_EINVAL, m); };
  if (!d) return bad("null descriptor");
  const bool ints = d->a_dtype == DCF_I8;
  if (!ints && d->a_dtype != DCF_F16 && d->a_dtype != DCF_BF16 && d->a_dtype != DCF_F32)
    return bad("int8 matmul: a must be i8, f16, bf16 or f32");
  if (d->out_dtype != DCF_F16 && d->out_dtype != DCF_BF16 && d->out_dtype != DCF_F32 &&
      !(d->out_dtype == DCF_I32 && ints))
    return bad("int8 matmul: the result must be f16, bf16 or f32, or i32 of i8 tokens");
  const uint64_t most = (1ull << 31) - 65536;
  if (d->tokens > most || d->channels > most) return bad("int8 matmul: tokens and channels must be at most 2^31 - 65536");
  if (d->depth > DCF_INT8_MAX_DEPTH) return bad("int8 matmul: depth must be at most 131071");
  if (d->a_row_stride < 0 || d->b_row_stride < 0 || d->out_row_stride < 0) return bad("int8 matmul: negative stride");
  if (!d->tokens || !d->channels) return DCF_OK;
  const int64_t given[3] = {d->a_row_stride, d->b_row_stride, d->out_row_stride};
  const uint64_t rows[3] = {d->tokens, d->channels, d->tokens}, cols[3] = {d->depth, d->depth, d->channels};
  for (int k = 0; k < 3; k++) {
    const __int128 rs = given[k] ? given[k] : (int64_t)cols[k];
    if ((__int128)(rows[k] - 1) * rs + cols[k] > ((__int128)1 << 46)) return bad("int8 matmul: tensor too large");
    if (k == 2 && rows[k] > 1 && rs < (__int128)cols[k]) return bad("int8 matmul: strides make rows of the result overlap");
  }
  return DCF_OK;
}

size_t int8_workspace(const dcf_int8_desc& d) {
  if (!d.tokens || !d.channels) return 0;
  return layout_of(d).bytes;
}

int launch_int8_matmul(const dcf_int8_desc& d, const void* a, const float* a_scale, const int8_t* b,
                       const float* b_scale, const float* bias, void* out, void* ws, dcf_status* st, cudaStream_t s) {
  (void)st;
  Int8Args g;
  g.a = (const int8_t*)a;
  g.a_scale = a_scale;
  g.as = d.a_row_stride ? d.a_row_stride : (int64_t)d.depth;
  if (d.a_dtype != DCF_I8) {
    const Layout l = layout_of(d);
    int8_t* q = (int8_t*)ws + l.q;
    float* scale = (float*)((uint8_t*)ws + l.scale);
    const dcf_quant_desc tokens = {d.a_dtype, DCF_QUANT_ROWS, d.tokens, d.depth, g.as, l.stride};
    if (int rc = launch_quantize(tokens, a, q, scale, s)) return rc;
    g.a = q;
    g.a_scale = scale;
    g.as = l.stride;
  }
  g.b = b;
  g.b_scale = b_scale;
  g.bias = bias;
  g.out = out;
  g.out_dtype = (int)d.out_dtype;
  g.tokens = (int)d.tokens;
  g.channels = (int)d.channels;
  g.depth = (int)d.depth;
  g.bs = d.b_row_stride ? d.b_row_stride : (int64_t)d.depth;
  g.os = d.out_row_stride ? d.out_row_stride : (int64_t)d.channels;
  const int64_t total = (int64_t)((d.tokens + kTile - 1) / kTile) * (int64_t)((d.channels + kTile - 1) / kTile);
  return launch(int8_tile_kernel, dim3((unsigned)(total < (1 << 30) ? total : 1 << 30)), 256, 0, 1, s, g);
}

}  // namespace dcf
