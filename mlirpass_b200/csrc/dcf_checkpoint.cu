// dcf_checkpoint.cu — the gradient of a weight from a checkpoint of its
// layer's input:
//   out[c][k] = sum over runs r of scale[r][k] * (sum over t in r of grad[t][c] * q[t][k])
// A whole number of 8 bits is exact in f16 and bf16, so the products of the
// inner sum are exact in f32; the scale comes after it.
#include "dcf_quant.cuh"

namespace dcf {

namespace {

struct GradArgs {
  const void* grad;
  const int8_t* q;
  const float* scale;
  void* out;
  int out_dtype, add;
  int tokens, channels, depth;
  int64_t gs, qs, os;
};

__device__ __forceinline__ void put(const GradArgs& g, int64_t c, int64_t k, float v) {
  const int64_t at = c * g.os + k;
  if (g.out_dtype == DCF_F32) ((float*)g.out)[at] = g.add ? __fadd_rn(((float*)g.out)[at], v) : v;
  else if (g.out_dtype == DCF_F16) ((__half*)g.out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)g.out)[at] = __float2bfloat16_rn(v);
}

constexpr int kTile = 64, kDeep = 32;

// 64 channels x 64 k to a block of 256 threads, sixteen results to a thread.
template <class T> __global__ void __launch_bounds__(256) grad_tile_kernel(const GradArgs g) {
  __shared__ float a[kDeep][kTile], b[kDeep][kTile];
  pdl_begin();
  const int64_t tiles = ((int64_t)g.depth + kTile - 1) / kTile, total = tiles * (((int64_t)g.channels + kTile - 1) / kTile);
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int64_t c0 = i / tiles * kTile, k0 = i % tiles * kTile;
    float sum[4][4] = {};
    for (int64_t r0 = 0; r0 < g.tokens; r0 += kRun) {
      float part[4][4] = {};
      for (int64_t t0 = r0; t0 < r0 + kRun && t0 < g.tokens; t0 += kDeep) {
        __syncthreads();
        for (int w = threadIdx.x; w < kTile * kDeep; w += 256) {
          const int64_t t = t0 + w / kTile, c = c0 + w % kTile, k = k0 + w % kTile;
          a[w / kTile][w % kTile] =
              t < g.tokens && c < g.channels ? value_of<T>(bits_of((const T*)g.grad + t * g.gs + c)) : 0.0f;
          b[w / kTile][w % kTile] = t < g.tokens && k < g.depth ? (float)g.q[t * g.qs + k] : 0.0f;
        }
        __syncthreads();
#pragma unroll 8
        for (int t = 0; t < kDeep; t++)
#pragma unroll
          for (int m = 0; m < 4; m++)
#pragma unroll
            for (int n = 0; n < 4; n++) part[m][n] = __fmaf_rn(a[t][y + 16 * m], b[t][x + 16 * n], part[m][n]);
      }
      for (int n = 0; n < 4; n++) {
        const int64_t k = k0 + x + 16 * n;
        const float s = k < g.depth ? g.scale[r0 / kRun * g.depth + k] : 0.0f;
        for (int m = 0; m < 4; m++) sum[m][n] = __fmaf_rn(s, part[m][n], sum[m][n]);
      }
    }
    for (int m = 0; m < 4; m++)
      for (int n = 0; n < 4; n++)
        if (c0 + y + 16 * m < g.channels && k0 + x + 16 * n < g.depth) put(g, c0 + y + 16 * m, k0 + x + 16 * n, sum[m][n]);
  }
}

}  // namespace

int checkpoint_desc_check(const dcf_checkpoint_desc* d) {
  auto bad = [](const char* m) { return record_error(DCF_EINVAL, m); };
  if (!d) return bad("null descriptor");
  if (d->grad_dtype != DCF_F16 && d->grad_dtype != DCF_BF16) return bad("checkpoint grad: the gradient must be f16 or bf16");
  if (d->out_dtype != DCF_F32 && d->out_dtype != DCF_F16 && d->out_dtype != DCF_BF16)
    return bad("checkpoint grad: the result must be f32, f16 or bf16");
  if (d->reserved) return bad("checkpoint grad: reserved field is not 0");
  if (d->flags & ~DCF_CHECKPOINT_ACCUMULATE) return bad("checkpoint grad: unknown flag");
  if ((d->flags & DCF_CHECKPOINT_ACCUMULATE) && d->out_dtype != DCF_F32)
    return bad("checkpoint grad: only a f32 result accumulates");
  const uint64_t most = (1ull << 31) - 65536;
  if (d->tokens > most || d->channels > most || d->depth > most)
    return bad("checkpoint grad: tokens, channels and depth must be at most 2^31 - 65536");
  if (d->grad_row_stride < 0 || d->q_row_stride < 0 || d->out_row_stride < 0) return bad("checkpoint grad: negative stride");
  if (!d->channels || !d->depth) return DCF_OK;
  const int64_t given[3] = {d->grad_row_stride, d->q_row_stride, d->out_row_stride};
  const uint64_t rows[3] = {d->tokens, d->tokens, d->channels}, cols[3] = {d->channels, d->depth, d->depth};
  for (int k = 0; k < 3; k++) {
    if (!rows[k]) continue;
    const __int128 rs = given[k] ? given[k] : (int64_t)cols[k];
    if ((__int128)(rows[k] - 1) * rs + cols[k] > ((__int128)1 << 46)) return bad("checkpoint grad: tensor too large");
    if (k == 2 && rows[k] > 1 && rs < (__int128)cols[k])
      return bad("checkpoint grad: strides make rows of the result overlap");
  }
  return DCF_OK;
}

size_t checkpoint_workspace(const dcf_checkpoint_desc& d) {
  (void)d;
  return 0;
}

int launch_checkpoint_grad(const dcf_checkpoint_desc& d, const void* grad, const int8_t* q, const float* scale,
                           void* out, void* ws, dcf_status* st, cudaStream_t s) {
  (void)ws;
  (void)st;
  GradArgs g;
  g.grad = grad;
  g.q = q;
  g.scale = scale;
  g.out = out;
  g.out_dtype = (int)d.out_dtype;
  g.add = (d.flags & DCF_CHECKPOINT_ACCUMULATE) != 0;
  g.tokens = (int)d.tokens;
  g.channels = (int)d.channels;
  g.depth = (int)d.depth;
  g.gs = d.grad_row_stride ? d.grad_row_stride : (int64_t)d.channels;
  g.qs = d.q_row_stride ? d.q_row_stride : (int64_t)d.depth;
  g.os = d.out_row_stride ? d.out_row_stride : (int64_t)d.depth;
  const int64_t total = (int64_t)((d.channels + kTile - 1) / kTile) * (int64_t)((d.depth + kTile - 1) / kTile);
  const dim3 grid((unsigned)(total < (1 << 30) ? total : 1 << 30));
  return d.grad_dtype == DCF_F16 ? launch(grad_tile_kernel<__half>, grid, 256, 0, 1, s, g)
                                 : launch(grad_tile_kernel<__nv_bfloat16>, grid, 256, 0, 1, s, g);
}

}  // namespace dcf
