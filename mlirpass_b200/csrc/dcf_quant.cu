// dcf_quant.cu — matrices to 8-bit whole numbers with a scale for each row, or
// for each column of each run of 128 rows (a checkpoint of activations), and
// back.
//
// All four are bound by HBM: a value is read once, held in registers until the
// largest magnitude beside it is known, and its byte written; reading back is
// the same way round.  Some five instructions per value (dcf_quant.cuh) keep
// the arithmetic behind that.  Measured (bytes read and written over the
// kernel's time): 8192 x 4096 f32 by rows 32 us and back 28 us (5.3, 6.0 TB/s),
// bf16 by columns 20 us and back 17 us (4.9, 5.9 TB/s; one after the other they
// take 33 us, as what is read back is still in L2).
#include <math.h>

#include "dcf_quant.cuh"

namespace dcf {

namespace {

constexpr int kQuantThreads = 256;

struct QuantArgs {
  const void* in;
  int8_t* q;
  float* scale;
  int64_t rows;
  int cols;
  int64_t rs, qs;
};

// A row to TPR threads, which hold G groups of E values each; a longer row is
// read a second time (from L2).
template <class T, int E, int G, int TPR>
__global__ void __launch_bounds__(kQuantThreads) quant_rows_kernel(const QuantArgs a) {
  constexpr int kRows = kQuantThreads / TPR;
  __shared__ uint32_t keys[kQuantThreads / 32];
  pdl_begin();
  const int at = threadIdx.x % TPR, groups = (a.cols + E - 1) / E;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool there = r < a.rows;
    const T* in = (const T*)a.in + r * a.rs;
    Group<T, E> g[G];
    uint32_t key = 0;
    const int first = groups > TPR * G ? (groups - 1) / (TPR * G) * (TPR * G) : 0;  // of the part that stays in registers
    if (there) {
      for (int c = at; c < first; c += TPR) {
        Group<T, E> v;
        load_group(v, in + (int64_t)c * E, a.cols - c * E);
        key = group_key(v, key);
      }
#pragma unroll
      for (int j = 0; j < G; j++) {
        const int c = first + at + j * TPR;
        load_group(g[j], in + (int64_t)c * E, c < groups ? a.cols - c * E : 0);
      }
#pragma unroll
      for (int j = 0; j < G; j++) key = group_key(g[j], key);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = key_max<T>(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
    if (TPR > 32) {
      if (threadIdx.x % 32 == 0) keys[threadIdx.x / 32] = key;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kQuantThreads / 32; j++) key = key_max<T>(key, keys[j]);
      __syncthreads();
    }
    const Scale s(key_value<T>(key));
    if (!there) continue;
    if (at == 0) a.scale[r] = s.scale;
    int8_t* q = a.q + r * a.qs;
    auto write = [&](Group<T, E>& v, int c) {
      uint32_t w[kLevelWords<E>];
      quantise_group(v, s, w);
      store_levels<E>(q + (int64_t)c * E, w, a.cols - c * E);
    };
    for (int c = at; c < first; c += TPR) {
      Group<T, E> v;
      load_group(v, in + (int64_t)c * E, a.cols - c * E);
      write(v, c);
    }
#pragma unroll
    for (int j = 0; j < G; j++) {
      const int c = first + at + j * TPR;
      if (c < groups) write(g[j], c);
    }
  }
}

// Tiles of a run: kRun rows x (W groups of E columns).  Thread (x, y) holds
// group x of rows y, y + R, ...
template <class T, int E, int W> struct RunTile {
  static constexpr int kCols = E * W, kSteps = W * kRun / kQuantThreads, kRowStep = kQuantThreads / W;
};

template <class T, int E, int W>
__global__ void __launch_bounds__(kQuantThreads) quant_columns_kernel(const QuantArgs a) {
  using Tile = RunTile<T, E, W>;
  constexpr int S = Tile::kSteps, R = Tile::kRowStep, kWords = Group<T, E>::kWords;
  __shared__ uint32_t keys[R][W * kWords];  // of each row of threads
  __shared__ float factors[Tile::kCols];
  __shared__ uint32_t keeps[Tile::kCols];
  pdl_begin();
  const int x = threadIdx.x % W, y = threadIdx.x / W;
  const int64_t tiles = (a.cols + Tile::kCols - 1) / Tile::kCols, total = tiles * ((a.rows + kRun - 1) / kRun);
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int64_t run = t / tiles;
    const int col = (int)(t % tiles) * Tile::kCols, c = col + x * E, have = a.cols - c;
    const int rows = (int)(a.rows - run * kRun < kRun ? a.rows - run * kRun : kRun);
    const T* in = (const T*)a.in + run * kRun * a.rs + c;
    Group<T, E> g[S];
#pragma unroll
    for (int j = 0; j < S; j++) load_group(g[j], in + (y + j * R) * a.rs, y + j * R < rows ? have : 0);
    uint32_t key[kWords];
#pragma unroll
    for (int k = 0; k < kWords; k++) {
      key[k] = 0;
#pragma unroll
      for (int j = 0; j < S; j++) key[k] = key_max<T>(key[k], g[j].w[k] & kMagnitude<T>);
      keys[y][x * kWords + k] = key[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Tile::kCols; i += kQuantThreads) {
      constexpr int kPerWord = E * 1 / kWords;  // values of a word
      uint32_t m = 0;
#pragma unroll 8
      for (int j = 0; j < R; j++) {
        const uint32_t w = keys[j][i / kPerWord], v = kPerWord == 2 ? (i & 1 ? w >> 16 : w & 0xFFFF) : w;
        m = m > v ? m : v;
      }
      const Scale s(value_of<T>(m));
      factors[i] = s.factor;
      keeps[i] = s.keep;
      if (col + i < a.cols) a.scale[run * a.cols + col + i] = s.scale;
    }
    __syncthreads();
    float f[E];
    uint32_t keep[kWords];
#pragma unroll
    for (int e = 0; e < E; e++) f[e] = factors[x * E + e];
#pragma unroll
    for (int k = 0; k < kWords; k++) {
      if constexpr (kWords * 2 == E) keep[k] = __byte_perm(keeps[x * E + 2 * k], keeps[x * E + 2 * k + 1], 0x5410);
      else keep[k] = keeps[x * E + k];
    }
    int8_t* q = a.q + run * kRun * a.qs + c;
#pragma unroll
    for (int j = 0; j < S; j++) {
      if (y + j * R >= rows) break;
#pragma unroll
      for (int k = 0; k < kWords; k++) g[j].w[k] &= keep[k];
      uint32_t w[kLevelWords<E>];
      pack_levels<E>(w, [&](int e) { return level(group_value(g[j], e), f[e]); });
      store_levels<E>(q + (y + j * R) * a.qs, w, have);
    }
    __syncthreads();
  }
}

template <class T> __device__ __forceinline__ void store_value(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(v);
  else *p = __float2bfloat16_rn(v);
}

template <class T> __device__ __forceinline__ uint32_t two_values(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
  }
}

// Tiles as above, of the whole matrix.
template <class T, int E, int W, bool COLUMNS>
__global__ void __launch_bounds__(kQuantThreads) dequant_kernel(const QuantArgs a, T* out) {
  using Tile = RunTile<T, E, W>;
  constexpr int S = Tile::kSteps, R = Tile::kRowStep;
  pdl_begin();
  const int x = threadIdx.x % W, y = threadIdx.x / W;
  const int64_t tiles = (a.cols + Tile::kCols - 1) / Tile::kCols, total = tiles * ((a.rows + kRun - 1) / kRun);
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int64_t run = t / tiles;
    const int c = (int)(t % tiles) * Tile::kCols + x * E, have = a.cols - c;
    const int rows = (int)(a.rows - run * kRun < kRun ? a.rows - run * kRun : kRun);
    if (have <= 0) continue;
    const int8_t* q = a.q + run * kRun * a.qs + c;
    uint32_t w[S][kLevelWords<E>];
#pragma unroll
    for (int j = 0; j < S; j++) {
      const int8_t* p = q + (y + j * R) * a.qs;
      if (y + j * R >= rows) break;
      if (E == 1) {
        w[j][0] = *(const uint8_t*)p;
      } else if (have >= E) {
        if constexpr (E == 8) {
          const uint2 v = *(const uint2*)p;
          w[j][0] = v.x, w[j][E > 4] = v.y;
        } else if constexpr (E == 4) {
          w[j][0] = *(const uint32_t*)p;
        } else {
          w[j][0] = *(const uint16_t*)p;
        }
      } else {
#pragma unroll
        for (int k = 0; k < kLevelWords<E>; k++) w[j][k] = 0;
#pragma unroll
        for (int e = 0; e < E; e++)
          if (e < have) w[j][e >> 2] |= (uint32_t)(uint8_t)p[e] << ((e & 3) * 8);
      }
    }
    float s[E];
    if (COLUMNS) {
#pragma unroll
      for (int e = 0; e < E; e++) s[e] = e < have ? a.scale[run * a.cols + c + e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < S; j++) {
      const int row = y + j * R;
      if (row >= rows) break;
      if (!COLUMNS) {
        const float one = a.scale[run * kRun + row];
#pragma unroll
        for (int e = 0; e < E; e++) s[e] = one;
      }
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = __fmul_rn(s[e], byte_value(w[j][e >> 2] ^ 0x80808080u, e & 3));
      T* to = out + (run * kRun + row) * a.rs + c;
      if (E > 1 && have >= E) {
        if constexpr (E == 8)
          *(uint4*)to = make_uint4(two_values<T>(v[0], v[1]), two_values<T>(v[2], v[3]), two_values<T>(v[4], v[5]),
                                   two_values<T>(v[6], v[7]));
        else if constexpr (E == 4)
          *(float4*)to = make_float4(v[0], v[1], v[2], v[3]);
        else if constexpr (E == 2)
          *(uint32_t*)to = two_values<T>(v[0], v[1]);
      } else {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (e < have) store_value(to + e, v[e]);
      }
    }
  }
}

// A thread writes 16 bytes of a row.
__global__ void __launch_bounds__(kQuantThreads) pack_kernel(const uint8_t* from, int64_t stride, int64_t rows,
                                                             int64_t bytes, uint8_t* to, int64_t to_stride) {
  pdl_begin();
  const int64_t groups = (bytes + 15) / 16, all = groups * rows;
  for (int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kQuantThreads) {
    const int64_t r = i / groups, c = i % groups * 16;
    *(uint4*)(to + r * to_stride + c) = row_bytes(from + r * stride, c, bytes);
  }
}

unsigned blocks_of(int64_t n) { return (unsigned)(n < (1 << 30) ? n : 1 << 30); }

QuantArgs quant_args(const dcf_quant_desc& d, const void* in, int8_t* q, float* scale) {
  QuantArgs a;
  a.in = in;
  a.q = q;
  a.scale = scale;
  a.rows = (int64_t)d.rows;
  a.cols = (int)d.cols;
  a.rs = d.row_stride ? d.row_stride : (int64_t)d.cols;
  a.qs = d.q_row_stride ? d.q_row_stride : (int64_t)d.cols;
  return a;
}

// Whether rows of values and of whole numbers divide into whole vectors of E.
template <class T, int E> bool vectors(const QuantArgs& a, const void* values) {
  constexpr int kBytes = E * (int)sizeof(T);
  return (uintptr_t)values % kBytes == 0 && (uintptr_t)a.q % E == 0 &&
         (a.rows == 1 || (a.rs * (int64_t)sizeof(T) % kBytes == 0 && a.qs % E == 0));
}

// Rows to a warp while that keeps them in registers, then to a block that holds as little as
// it can: more blocks to an SM have more on its way (f32, 8192 x 4096: 38 us with room for twice the row, 32 us so).
template <class T, int E> int quantize_rows(const QuantArgs& a, cudaStream_t s) {
  constexpr int kUnit = E <= 2 ? 4 : 1;
  const int64_t groups = (a.cols + E - 1) / E;
  auto run = [&](auto kernel, int64_t blocks) { return launch(kernel, blocks_of(blocks), kQuantThreads, 0, 1, s, a); };
  if (groups <= 32 * 4 * kUnit)
    return run(quant_rows_kernel<T, E, 4 * kUnit, 32>, (a.rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32));
  if (groups <= kQuantThreads * 2 * kUnit) return run(quant_rows_kernel<T, E, 2 * kUnit, kQuantThreads>, a.rows);
  if (groups <= kQuantThreads * 4 * kUnit) return run(quant_rows_kernel<T, E, 4 * kUnit, kQuantThreads>, a.rows);
  return run(quant_rows_kernel<T, E, 8 * kUnit, kQuantThreads>, a.rows);
}

template <int E> constexpr int kWide = E == 1 ? 64 : E == 2 ? 32 : 16;  // groups of a tile's row

template <class T, int E, int W> int64_t run_tiles(const QuantArgs& a) {
  constexpr int kCols = RunTile<T, E, W>::kCols;
  return ((int64_t)a.cols + kCols - 1) / kCols * ((a.rows + kRun - 1) / kRun);
}

template <class T, int E> int quantize_t(const dcf_quant_desc& d, const QuantArgs& a, cudaStream_t s) {
  if (d.along == DCF_QUANT_ROWS) return quantize_rows<T, E>(a, s);
  return launch(quant_columns_kernel<T, E, kWide<E>>, blocks_of(run_tiles<T, E, kWide<E>>(a)), kQuantThreads, 0, 1, s, a);
}

template <class T, int E> int dequantize_t(const dcf_quant_desc& d, const QuantArgs& a, void* out, cudaStream_t s) {
  constexpr int W = kWide<E>;
  const unsigned blocks = blocks_of(run_tiles<T, E, W>(a));
  return d.along == DCF_QUANT_ROWS ? launch(dequant_kernel<T, E, W, false>, blocks, kQuantThreads, 0, 1, s, a, (T*)out)
                                   : launch(dequant_kernel<T, E, W, true>, blocks, kQuantThreads, 0, 1, s, a, (T*)out);
}

// Calls f<T, E>() of the type and of the widest vectors that rows divide into (16-bit values, rows of odd numbers
// of words: two at a time; 3728 x 3186 there and back 35 us by single values, 27 us so).
template <class F> int by_type(uint32_t dtype, const QuantArgs& a, const void* values, F f) {
  auto half = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (vectors<T, 8>(a, values)) return f(t, std::integral_constant<int, 8>());
    if (vectors<T, 2>(a, values)) return f(t, std::integral_constant<int, 2>());
    return f(t, std::integral_constant<int, 1>());
  };
  switch (dtype) {
    case DCF_F16: return half((__half*)0);
    case DCF_BF16: return half((__nv_bfloat16*)0);
    case DCF_F32: return vectors<float, 4>(a, values) ? f((float*)0, std::integral_constant<int, 4>())
                                                      : f((float*)0, std::integral_constant<int, 1>());
    default: return DCF_EUNSUPPORTED;
  }
}

}  // namespace

int launch_pack_rows(const void* from, int64_t stride, int64_t rows, int64_t bytes, void* to, int64_t to_stride,
                     cudaStream_t s) {
  const int64_t all = (bytes + 15) / 16 * rows;
  return launch(pack_kernel, blocks_of((all + kQuantThreads - 1) / kQuantThreads), kQuantThreads, 0, 1, s,
                (const uint8_t*)from, stride, rows, bytes, (uint8_t*)to, to_stride);
}

int quant_desc_check(const dcf_quant_desc* d, bool back) {
  auto bad = [](const char* m) { return record_error(DCF_EINVAL, m); };
  if (!d) return bad("null descriptor");
  if (d->dtype != DCF_F16 && d->dtype != DCF_BF16 && d->dtype != DCF_F32)
    return bad("quantize: dtype must be f16, bf16 or f32");
  if (d->along != DCF_QUANT_ROWS && d->along != DCF_QUANT_COLUMNS) return bad("quantize: along rows or columns");
  if (d->rows >= 1ull << 31 || d->cols > (1ull << 31) - 65536)
    return bad("quantize: rows must be below 2^31, cols at most 2^31 - 65536");
  if (d->row_stride < 0 || d->q_row_stride < 0) return bad("quantize: negative stride");
  if (!d->rows || !d->cols) return DCF_OK;
  for (int k = 0; k < 2; k++) {
    const int64_t given = k ? d->q_row_stride : d->row_stride;
    const __int128 rs = given ? given : (int64_t)d->cols;
    if ((__int128)(d->rows - 1) * rs + d->cols > ((__int128)1 << 46)) return bad("quantize: tensor too large");
    if (d->rows > 1 && rs < (__int128)d->cols && (k ? !back : back)) return bad("quantize: strides make rows of the result overlap");
  }
  return DCF_OK;
}

int launch_quantize(const dcf_quant_desc& d, const void* in, int8_t* q, float* scale, cudaStream_t s) {
  const QuantArgs a = quant_args(d, in, q, scale);
  return by_type(d.dtype, a, in, [&](auto* t, auto e) {
    return quantize_t<std::remove_pointer_t<decltype(t)>, decltype(e)::value>(d, a, s);
  });
}

int launch_dequantize(const dcf_quant_desc& d, const int8_t* q, const float* scale, void* out, cudaStream_t s) {
  const QuantArgs a = quant_args(d, nullptr, (int8_t*)q, (float*)scale);
  return by_type(d.dtype, a, out, [&](auto* t, auto e) {
    return dequantize_t<std::remove_pointer_t<decltype(t)>, decltype(e)::value>(d, a, out, s);
  });
}

}  // namespace dcf
