// dcf_orth.cu — Newton-Schulz orthogonalisation of dense matrices.
//
// With X (m x n, m <= n) scaled to Frobenius norm one, each step is
//     A = X X^T,   B = a I + b A + c A A,   X <- B X,
// three products on the tensor cores.  A step multiplies the smallest
// singular values by a (3.44 in the usual quintic), so five steps amplify what a
// rounding of X leaves in its null space by several hundred: operands of 11
// bits show as 4 % in a matrix of low rank.  Operands are therefore exact splits:
// a value v scaled by a power of two is kept as two fp16 planes, hi = fp16(v)
// and lo = fp16(v - hi), 22 bits or more, and a product is
//     hi hi + hi lo + lo hi
// accumulated in fp32 in TMEM (the dropped lo lo is 2^-22 of it).  The result
// is closer to 64-bit arithmetic than products of fp32 values are, at three
// fp16 products instead of fp32 arithmetic on the CUDA cores.
//
// Scales are powers of two from bounds the host computes: singular values of
// X are in [0, 1] at the start, a step maps s to |a s + b s^3 + c s^5|, and
// no element of X, A = X X^T or B exceeds the largest singular value of its matrix.
// So no plane overflows, whatever the data.
//
// A and A A are symmetric: only tiles that touch the upper triangle are
// computed, and their elements written to both sides.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <mutex>

#include "dcf_kernels.cuh"

namespace dcf {

namespace {

constexpr int kBM = 128, kBK = 64;      // tile rows; k extent of a stage: one 128-byte swizzle row
constexpr int kGemmThreads = 192;       // warp 0 loads, warp 1 multiplies, warps 2-5 write out

// ------------------------------------------------------- PTX wrappers

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory descriptor of a K-major operand tile with the 128-byte
// swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// -------------------------------------------------------------- planes

// One operand as the tensor map and the epilogue see it: per matrix two
// planes (hi, lo) of `rows` rows of `ld` fp16 values.
struct Planes {
  __half* p;
  int rows, ld;
  __device__ __forceinline__ __half* row(uint32_t z, int plane, int r) const {
    return p + ((size_t)(2 * z + plane) * rows + r) * ld;
  }
};

__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(__fsub_rn(v, __half2float(hi)));
}

// What the epilogue of a product does with its accumulators.
enum Mode {
  GRAM,   // A = X X^T: planes, both triangles
  POLY,   // B = a I + b A + c A A: planes, both triangles
  APPLY,  // X <- B X: planes of X and of X^T
  FINAL   // the result, in the caller's type and orientation
};

struct GemmArgs {
  int m, n, k;            // rows, columns, length of the product
  int tiles_m, tiles_n;   // tiles of kBM x BN
  int tiles;              // per matrix (of the upper triangle for GRAM, POLY)
  float alpha, beta, diag;  // v = alpha acc [+ beta A + diag I]
  Planes to, to_t, from;  // results; POLY: A
  void* out;
  int out_dtype, transposed;
  int64_t out_rs, out_bs;
  dcf_status* st;
};

__device__ __forceinline__ void store_typed(void* out, int64_t at, int dtype, float v) {
  if (dtype == DCF_F32) ((float*)out)[at] = v;
  else if (dtype == DCF_F16) ((__half*)out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)out)[at] = __float2bfloat16_rn(v);
}

template <int BN, int STAGES> struct GemmSmem {
  static constexpr int kA = kBM * kBK * 2, kB = BN * kBK * 2;  // one plane of one stage
  static constexpr int kStage = 2 * (kA + kB);
  static constexpr int kBytes = STAGES * kStage + 1024 + (2 * STAGES + 1) * 8 + 16;
};

// One kBM x BN tile of D = P Q^T per CTA, P and Q given as two fp16 planes each,
// K-major.  A stage holds 64 columns of all four planes, which three products
// share: hi hi, hi lo and lo hi.
template <int BN, int STAGES, Mode MODE>
__global__ void __launch_bounds__(kGemmThreads) orth_gemm_kernel(const __grid_constant__ CUtensorMap map_p,
                                                                 const __grid_constant__ CUtensorMap map_q,
                                                                 const __grid_constant__ GemmArgs g) {
  using L = GemmSmem<BN, STAGES>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(base + STAGES * L::kStage);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_at = (uint32_t*)(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const uint32_t z = blockIdx.x / (uint32_t)g.tiles;
  int tile = (int)(blockIdx.x % (uint32_t)g.tiles);
  int tm, tn;
  if (MODE == GRAM || MODE == POLY) {
    // Row tm keeps the tiles that reach the diagonal or lie right of it.
    for (tm = 0;; tm++) {
      const int first = tm * kBM / BN, count = g.tiles_n - first;
      if (tile < count) {
        tn = first + tile;
        break;
      }
      tile -= count;
    }
  } else {
    tm = tile % g.tiles_m;
    tn = tile / g.tiles_m;
  }
  const int row0 = tm * kBM, col0 = tn * BN;
  const int blocks = (g.k + kBK - 1) / kBK;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_at)), "r"(BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)tmem_at;

  bool fail = false;
  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < blocks; i++) {
        const int s = i % STAGES;
        if (i >= STAGES && !mbar_wait_bounded(&empty[s], (unsigned)((i / STAGES - 1) & 1))) {
          fail = true;
          break;
        }
        const uint32_t at = smem_addr(base + s * L::kStage);
        mbar_expect_tx(&full[s], L::kStage);
        for (int p = 0; p < 2; p++) {
          tma_load_3d(at + p * L::kA, &map_p, i * kBK, row0, (int)(2 * z + p), &full[s]);
          for (int r = 0; r < BN; r += 128)
            tma_load_3d(at + 2 * L::kA + p * L::kB + r * kBK * 2, &map_q, i * kBK, col0 + r, (int)(2 * z + p), &full[s]);
        }
        issued = i + 1;
      }
      // Give up only with no copy of ours left in flight.
      if (fail)
        for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; i++)
          mbar_wait_bounded(&full[i % STAGES], (unsigned)((i / STAGES) & 1));
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
      for (int i = 0; i < blocks; i++) {
        const int s = i % STAGES;
        if (!mbar_wait_bounded(&full[s], (unsigned)((i / STAGES) & 1))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = smem_addr(base + s * L::kStage);
        const uint64_t ph = smem_desc(at), pl = smem_desc(at + L::kA);
        const uint64_t qh = smem_desc(at + 2 * L::kA), ql = smem_desc(at + 2 * L::kA + L::kB);
#pragma unroll
        for (int j = 0; j < kBK / 16; j++) {  // 16 columns: 32 bytes on
          mma_f16(tmem, ph + 2 * j, qh + 2 * j, idesc, (i | j) != 0);
          mma_f16(tmem, ph + 2 * j, ql + 2 * j, idesc, 1);
          mma_f16(tmem, pl + 2 * j, qh + 2 * j, idesc, 1);
        }
        mma_commit(&empty[s]);
      }
      mma_commit(done);
    }
  } else {
    fail = __any_sync(0xFFFFFFFFu, !mbar_wait_bounded(done, 0));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int part = warp & 3;  // the 32 TMEM lanes this warp may read
    const int r = row0 + part * 32 + lane;
    for (int c = 0; c < BN && !fail; c += 32) {
      const int c0 = col0 + c;
      if (c0 >= g.n) break;
      uint32_t acc[32];
      tmem_load32(tmem + ((uint32_t)(part * 32) << 16) + c, acc);
      if (MODE == FINAL) {
        for (int j = 0; j < 32; j++) {
          const int cc = c0 + j;
          if (r < g.m && cc < g.n) {
            const int64_t at = (int64_t)z * g.out_bs + (g.transposed ? (int64_t)cc * g.out_rs + r : (int64_t)r * g.out_rs + cc);
            store_typed(g.out, at, g.out_dtype, __fmul_rn(g.alpha, __uint_as_float(acc[j])));
          }
        }
        continue;
      }
      constexpr bool sym = MODE == GRAM || MODE == POLY;
      if (sym && c0 + 31 < row0 + part * 32) continue;  // below the diagonal: written by its mirror image
      __half hi[32], lo[32];
#pragma unroll
      for (int j = 0; j < 32; j++) {
        float v = __fmul_rn(g.alpha, __uint_as_float(acc[j]));
        if (MODE == POLY) {
          const int cc = c0 + j;
          if (r < g.m && cc < g.n) {
            const float x = __fadd_rn(__half2float(g.from.row(z, 0, r)[cc]), __half2float(g.from.row(z, 1, r)[cc]));
            v = __fmaf_rn(g.beta, x, v);
            if (r == cc) v = __fadd_rn(v, g.diag);
          }
        }
        split(v, hi[j], lo[j]);
      }
      if (r < g.m) {
        __half* h = g.to.row(z, 0, r) + c0;
        __half* l = g.to.row(z, 1, r) + c0;
        if (!sym || c0 >= r) {  // rows are padded to 64 columns, so whole chunks fit
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            *(uint4*)(h + j) = *(const uint4*)(hi + j);
            *(uint4*)(l + j) = *(const uint4*)(lo + j);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++)
            if (c0 + j >= r) {
              h[j] = hi[j];
              l[j] = lo[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 32; j++) {
          const int cc = c0 + j;
          if (cc < g.n && (!sym || cc > r)) {
            g.to_t.row(z, 0, cc)[r] = hi[j];
            g.to_t.row(z, 1, cc)[r] = lo[j];
          }
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  if (fail) atomicExch(&g.st->error, 1u);
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(BN) : "memory");
  }
}

// ------------------------------------------------------- norm and split

struct MatArgs {
  const void* in;
  int dtype;
  int rows, cols;        // as the caller has them
  int64_t rs, bs;
};

__device__ __forceinline__ float load_typed(const void* p, int dtype, int64_t at) {
  if (dtype == DCF_F32) return ((const float*)p)[at];
  if (dtype == DCF_F16) return __half2float(((const __half*)p)[at]);
  return __bfloat162float(((const __nv_bfloat16*)p)[at]);
}

constexpr int kNormThreads = 256;

// Sums of squares in 64 bits (a f32 element's square can pass 32), one part
// per block.
__global__ void __launch_bounds__(kNormThreads) orth_norm_kernel(const __grid_constant__ MatArgs a, double* part) {
  const uint32_t z = blockIdx.y;
  double s = 0;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t at = (int64_t)z * a.bs + (int64_t)r * a.rs;
    for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
      const double v = load_typed(a.in, a.dtype, at + c);
      s = __fma_rn(v, v, s);
    }
  }
  __shared__ double sh[kNormThreads / 32];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; w++) s += sh[w];
    part[(size_t)z * gridDim.x + blockIdx.x] = s;
  }
}

// X = G / (norm + eps), 64 x 64 elements per block, into the planes of X and
// of its transpose; or, with no steps to take, straight to the result.
__global__ void __launch_bounds__(256) orth_split_kernel(const __grid_constant__ MatArgs a, const double* part,
                                                         int parts, double eps, double scale, Planes x, Planes xt,
                                                         int transposed, void* out, int out_dtype, int64_t out_rs,
                                                         int64_t out_bs) {
  __shared__ float tile[64][65];
  __shared__ double factor;
  const uint32_t z = blockIdx.z;
  if (threadIdx.x < 32) {
    double s = 0;
    for (int i = threadIdx.x; i < parts; i += 32) s += part[(size_t)z * parts + i];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (threadIdx.x == 0) factor = scale / (sqrt(s) + eps);
  }
  __syncthreads();
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int r = r0 + i / 64, c = c0 + i % 64;
    float v = 0;
    if (r < a.rows && c < a.cols) {
      v = (float)((double)load_typed(a.in, a.dtype, (int64_t)z * a.bs + (int64_t)r * a.rs + c) * factor);
      if (out) store_typed(out, (int64_t)z * out_bs + (int64_t)r * out_rs + c, out_dtype, v);
    }
    tile[i / 64][i % 64] = v;
  }
  if (out) return;
  __syncthreads();
  const Planes& same = transposed ? xt : x;    // rows as the caller has them
  const Planes& other = transposed ? x : xt;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int u = i / 64, v = i % 64;
    __half hi, lo;
    if (r0 + u < a.rows && c0 + v < a.cols) {
      split(tile[u][v], hi, lo);
      same.row(z, 0, r0 + u)[c0 + v] = hi;
      same.row(z, 1, r0 + u)[c0 + v] = lo;
    }
    if (c0 + u < a.cols && r0 + v < a.rows) {
      split(tile[v][u], hi, lo);
      other.row(z, 0, c0 + u)[r0 + v] = hi;
      other.row(z, 1, c0 + u)[r0 + v] = lo;
    }
  }
}

// ---------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiled)p;
    cudaGetLastError();
  });
  return fn;
}

// Boxes of 64 columns x 128 rows of one plane; what lies beyond the matrix
// reads as zero.
bool encode(CUtensorMap* map, const Planes& x, int cols, uint64_t batch) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)x.rows, 2 * batch};
  const cuuint64_t strides[2] = {(cuuint64_t)x.ld * 2, (cuuint64_t)x.ld * 2 * (cuuint64_t)x.rows};
  const cuuint32_t box[3] = {kBK, 128, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, x.p, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int round64(uint64_t v) { return (int)((v + 63) / 64 * 64); }

// Bounds of one step on [0, s]: the largest |a s + b s^3 + c s^5| and
// |a + b s^2 + c s^4|, from the ends and the points where the derivative is
// zero.
void step_bounds(const double* k, double s, double* x, double* q) {
  const double a = k[0], b = k[1], c = k[2], t1 = s * s;
  auto at = [&](double t) {
    if (!(t >= 0 && t <= t1)) return;
    const double f = fabs(a + t * (b + t * c));
    if (f > *q) *q = f;
    if (f * sqrt(t) > *x) *x = f * sqrt(t);
  };
  *x = *q = 0;
  at(0);
  at(t1);
  if (c != 0) at(-b / (2 * c));
  // a + 3 b t + 5 c t^2 = 0
  if (c == 0) {
    if (b != 0) at(-a / (3 * b));
  } else {
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      at((-3 * b + sqrt(d)) / (10 * c));
      at((-3 * b - sqrt(d)) / (10 * c));
    }
  }
}

// The power of two that brings a bound to at most 2^13: a factor 8 below
// fp16's largest value, for what rounding adds.
int scale_of(double bound) {
  int e;
  frexp(bound > 1e-30 ? bound : 1e-30, &e);  // bound < 2^e
  return 13 - e;
}

constexpr double kMostSingular = 64;

struct Layout {
  Planes x, xt[2], a, b;
  double* part;
  int parts;
  size_t bytes;
};

Layout layout_of(const dcf_orth_desc& d, void* ws) {
  Layout l;
  const bool t = d.rows > d.cols;
  const int m = (int)(t ? d.cols : d.rows), n = (int)(t ? d.rows : d.cols);
  uint8_t* at = (uint8_t*)ws;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = at + off;
    off += (bytes + 255) / 256 * 256;
    return p;
  };
  auto planes = [&](int rows, int cols) {
    const int ld = round64((uint64_t)cols);
    return Planes{(__half*)take((size_t)d.batch * 2 * rows * ld * 2), rows, ld};
  };
  l.parts = (int)(d.rows < 256 ? d.rows : 256);
  l.part = (double*)take(d.batch * l.parts * 8);
  if (d.steps) {
    l.x = planes(m, n);
    l.xt[0] = planes(n, m);
    l.xt[1] = planes(n, m);
    l.a = planes(m, m);
    l.b = planes(m, m);
  } else {
    l.x = l.xt[0] = l.xt[1] = l.a = l.b = Planes{nullptr, 0, 0};
  }
  l.bytes = off;
  return l;
}

template <int BN, int STAGES, Mode MODE>
int gemm(const CUtensorMap& p, const CUtensorMap& q, GemmArgs g, uint64_t batch, cudaStream_t s) {
  using L = GemmSmem<BN, STAGES>;
  g.tiles_m = (g.m + kBM - 1) / kBM;
  g.tiles_n = (g.n + BN - 1) / BN;
  g.tiles = 0;
  if (MODE == GRAM || MODE == POLY)
    for (int t = 0; t < g.tiles_m; t++) g.tiles += g.tiles_n - t * kBM / BN;
  else
    g.tiles = g.tiles_m * g.tiles_n;
  auto kernel = orth_gemm_kernel<BN, STAGES, MODE>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess)
    return DCF_ECUDA;
  kernel<<<(unsigned)(g.tiles * batch), kGemmThreads, L::kBytes, s>>>(p, q, g);
  note_launch();
  return cudaPeekAtLastError() == cudaSuccess ? DCF_OK : DCF_ECUDA;
}

}  // namespace

int orth_desc_check(const dcf_orth_desc* d) {
  auto bad = [](const char* m) { return record_error(DCF_EINVAL, m); };
  if (!d) return bad("null descriptor");
  for (uint32_t t : {d->dtype, d->out_dtype})
    if (t != DCF_F16 && t != DCF_BF16 && t != DCF_F32) return bad("orthogonalize: dtype must be f16, bf16 or f32");
  if (d->reserved) return bad("orthogonalize: reserved field is not 0");
  if (d->steps > DCF_ORTH_MAX_STEPS) return bad("orthogonalize: too many steps");
  if (d->rows > 65536 || d->cols > 65536) return bad("orthogonalize: rows and cols must be at most 65536");
  if (d->batch > 65535) return bad("orthogonalize: at most 65535 matrices");
  if (!(d->eps >= 0) || !(d->eps < INFINITY)) return bad("orthogonalize: eps must be finite and not negative");
  if (d->row_stride < 0 || d->batch_stride < 0 || d->out_row_stride < 0 || d->out_batch_stride < 0)
    return bad("orthogonalize: negative stride");
  double s = 1;
  for (uint32_t i = 0; i < d->steps; i++) {
    for (int j = 0; j < 3; j++)
      if (!(fabs(d->coef[i][j]) <= 1e4)) return bad("orthogonalize: coefficient out of range");
    double q;
    step_bounds(d->coef[i], s, &s, &q);
    if (!(s <= kMostSingular)) return bad("orthogonalize: the coefficients let singular values grow past 64");
  }
  if (!d->batch || !d->rows || !d->cols) return DCF_OK;
  const uint64_t m = d->rows < d->cols ? d->rows : d->cols, n = d->rows < d->cols ? d->cols : d->rows;
  if ((__int128)d->batch * ((m + 127) / 128) * ((n + 127) / 128) >= (1ll << 31))
    return bad("orthogonalize: too many tiles");
  for (int k = 0; k < 2; k++) {
    const int64_t r = k ? d->out_row_stride : d->row_stride, b = k ? d->out_batch_stride : d->batch_stride;
    const __int128 rs = r ? r : (int64_t)d->cols, bs = b ? b : (__int128)d->rows * rs;
    const __int128 one = (__int128)(d->rows - 1) * rs + d->cols;
    if (one + (__int128)(d->batch - 1) * bs > ((__int128)1 << 46)) return bad("orthogonalize: tensor too large");
    if (k && ((d->rows > 1 && rs < (__int128)d->cols) || (d->batch > 1 && bs < one)))
      return bad("orthogonalize: output strides make rows overlap");
  }
  return DCF_OK;
}

size_t orth_workspace(const dcf_orth_desc& d) {
  if (!d.batch || !d.rows || !d.cols) return 0;
  return layout_of(d, nullptr).bytes;
}

int launch_orthogonalize(const dcf_orth_desc& d, const void* in, void* out, void* ws, dcf_status* st, cudaStream_t s) {
  const Layout l = layout_of(d, ws);
  const int t = d.rows > d.cols;
  const int m = (int)(t ? d.cols : d.rows), n = (int)(t ? d.rows : d.cols);
  MatArgs a;
  a.in = in;
  a.dtype = (int)d.dtype;
  a.rows = (int)d.rows;
  a.cols = (int)d.cols;
  a.rs = d.row_stride ? d.row_stride : (int64_t)d.cols;
  a.bs = d.batch_stride ? d.batch_stride : (int64_t)d.rows * a.rs;
  const int64_t out_rs = d.out_row_stride ? d.out_row_stride : (int64_t)d.cols;
  const int64_t out_bs = d.out_batch_stride ? d.out_batch_stride : (int64_t)d.rows * out_rs;
  orth_norm_kernel<<<dim3((unsigned)l.parts, (unsigned)d.batch), kNormThreads, 0, s>>>(a, l.part);
  note_launch();
  int sx = d.steps ? scale_of(1) : 0;
  const dim3 blocks((unsigned)((d.cols + 63) / 64), (unsigned)((d.rows + 63) / 64), (unsigned)d.batch);
  orth_split_kernel<<<blocks, 256, 0, s>>>(a, l.part, l.parts, d.eps, ldexp(1.0, sx), l.x, l.xt[0], t,
                                           d.steps ? nullptr : out, (int)d.out_dtype, out_rs, out_bs);
  note_launch();
  if (cudaPeekAtLastError() != cudaSuccess) return DCF_ECUDA;
  if (!d.steps) return DCF_OK;

  if (!encoder()) return DCF_EUNSUPPORTED;
  CUtensorMap mx, mxt[2], ma, mb;
  if (!encode(&mx, l.x, n, d.batch) || !encode(&mxt[0], l.xt[0], m, d.batch) || !encode(&mxt[1], l.xt[1], m, d.batch) ||
      !encode(&ma, l.a, m, d.batch) || !encode(&mb, l.b, m, d.batch))
    return DCF_ECUDA;
  double bound = 1;
  for (uint32_t i = 0; i < d.steps; i++) {
    const double* k = d.coef[i];
    double next, q;
    step_bounds(k, bound, &next, &q);
    const int sa = scale_of(bound * bound), sb = scale_of(q);
    GemmArgs g = {};
    g.st = st;
    g.m = g.n = m;
    g.k = n;
    g.alpha = (float)ldexp(1.0, sa - 2 * sx);
    g.to = g.to_t = l.a;
    int rc = gemm<128, 3, GRAM>(mx, mx, g, d.batch, s);
    if (rc) return rc;
    g.k = m;
    g.alpha = (float)ldexp(k[2], sb - 2 * sa);
    g.beta = (float)ldexp(k[1], sb - sa);
    g.diag = (float)ldexp(k[0], sb);
    g.from = l.a;
    g.to = g.to_t = l.b;
    if ((rc = gemm<128, 3, POLY>(ma, ma, g, d.batch, s))) return rc;
    const int sn = scale_of(next);
    g.n = n;
    g.beta = g.diag = 0;
    if (i + 1 < d.steps) {
      g.alpha = (float)ldexp(1.0, sn - sb - sx);
      g.to = l.x;
      g.to_t = l.xt[(i + 1) & 1];
      if ((rc = gemm<128, 3, APPLY>(mb, mxt[i & 1], g, d.batch, s))) return rc;
    } else {
      g.alpha = (float)ldexp(1.0, -sb - sx);
      g.out = out;
      g.out_dtype = (int)d.out_dtype;
      g.transposed = t;
      g.out_rs = out_rs;
      g.out_bs = out_bs;
      if ((rc = gemm<128, 3, FINAL>(mb, mxt[i & 1], g, d.batch, s))) return rc;
    }
    bound = next;
    sx = sn;
  }
  return DCF_OK;
}

}  // namespace dcf
