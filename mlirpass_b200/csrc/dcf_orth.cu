// dcf_orth.cu — Newton-Schulz orthogonalisation of dense matrices.
//
// With X (m x n, m <= n) scaled to Frobenius norm one, each step is
//     A = X X^T,   B = a I + b A + c A A,   X <- B X,
// three products on the tensor cores.  A step multiplies the smallest
// singular values by a (3.44 in the usual quintic), so five steps amplify what a
// rounding of X leaves in its null space by several hundred: operands of 11
// bits show as 4 % in a matrix of low rank.  Operands are therefore exact splits:
// a value v scaled by a power of two is kept as two fp16 planes, hi = fp16(v)
// and lo = fp16(v - hi): 22 bits, or, of what lies far below the scale, half of
// fp16's smallest step, 2^-25 beside a bound of 2^13.  A product is
//     hi hi + hi lo + lo hi
// (the dropped lo lo is 2^-22 of it).  The tensor core truncates as it
// accumulates, which over a long k costs more than the split does: TMEM sums
// short runs of k (32 to 128, see sums_of) and fp32 registers, which round, add
// the runs.  Five steps end about as near to
// 64-bit arithmetic as with products of fp32 values (f32, 8 to 1200 rows, one to sixteen
// times as many columns: 0.3 to 1.6 times their error, the more at few rows; 8192 x 2048: 2.8e-6
// here, 5.4e-6 there), at three fp16 products instead of fp32 arithmetic on the CUDA cores.
//
// Scales are powers of two from bounds: singular values of
// X are in [0, 1] at the start, a step maps s to |a s + b s^3 + c s^5|, and
// no element of X, A = X X^T or B exceeds the largest singular value of its matrix.
// So no plane overflows, whatever the data.  The host computes the bounds; a matrix whose
// norm eps exceeds starts from norm / (norm + eps) instead of 1, and its scales are
// made on the device (set_factors): planes scaled for 1 would lose what fp16 has no
// exponents for (norm 1e-12 beside an eps of 1e-7: 4e-4 of X).
//
// A and A A are symmetric: only tiles that touch the upper triangle are
// computed, and their elements written to both sides.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "dcf_tensor.cuh"

namespace dcf {

namespace {

constexpr int kSide = 128, kBK = 64;  // rows of an operand a CTA loads; k extent of a stage: one 128-byte swizzle row
constexpr int kPlane = kSide * kBK * 2;  // bytes of one plane of one operand in a stage
constexpr int kStage = 4 * kPlane;       // P hi, P lo, Q hi, Q lo
constexpr int kOrthStages = 3;
constexpr int kOutWarps = 8;             // warps that add up and write out
constexpr int kGemmThreads = 128 + 32 * kOutWarps;  // warp 0 loads, warp 1 multiplies, 2 and 3 lend their registers
constexpr int kTile = 2 * kSide;         // a pair's tile: 256 x 256
constexpr int kTmem = 2 * kTile;         // TMEM columns: two sums
constexpr int kBlock = 32 * 32;          // values an out warp writes at a time: 32 rows x 32 columns
constexpr int kBuffer = 4096;            // bytes through which an out warp reorders 32 rows
constexpr int kGemmSmem = kOrthStages * kStage + kOutWarps * kBuffer + 256 + 1024;

// ------------------------------------------------------- PTX wrappers

// Into this CTA's memory; the bytes are reported to a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Shared-memory descriptor of one plane of an operand with the 128-byte
// swizzle: groups of eight 128-byte rows lie 1024 bytes apart.  A K-major
// plane has a row of 64 k for each of 128 rows of the operand; one whose rows
// run along the operand (MN) has two blocks of 64 of these, 8192 bytes apart,
// with a row for each of 64 k.
template <bool MN> __device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((MN ? 512ull : 1ull) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// From one 16-k slice to the next: 32 bytes along a row, or 16 rows.
template <bool MN> constexpr uint32_t kSlice = (MN ? 2048 : 32) >> 4;

// -------------------------------------------------------------- planes

// What a step's products are multiplied by on their way out, powers of two included.
struct alignas(16) Factors {
  float gram;       // A = gram acc
  float b2, b1, b0; // B = b2 acc + b1 A + b0 I
  float apply;      // X = apply acc
};

// From which set_factors makes a matrix's factors; `usual` are those of a bound of 1.
struct Scaling {
  int steps;
  double eps;
  double coef[DCF_ORTH_MAX_STEPS][3];
  double bound[DCF_ORTH_MAX_STEPS + 1];  // of X's singular values before each step and after the last
  double largest[DCF_ORTH_MAX_STEPS];    // of B's
  Factors usual[DCF_ORTH_MAX_STEPS];
};

// The power of two that brings a bound to at most 2^13: a factor 8 below
// fp16's largest value, for what rounding adds.  2^132 at most: what then falls off
// fp16's smallest value is below fp32's, too.
__host__ __device__ inline int scale_of(double bound) {
  int e;
  frexp(bound > 0x1p-120 ? bound : 0x1p-120, &e);  // bound < 2^e
  return 13 - e;
}

// The factors of every step where singular values start in [0, s].
__host__ __device__ inline void set_factors(const Scaling& k, double s, Factors* out) {
  int sx = scale_of(s);
  for (int i = 0; i < k.steps; i++) {
    const double a = k.coef[i][0], b = k.coef[i][1], c = k.coef[i][2], t = s * s;
    const double q = fmin(k.largest[i], fabs(a) + t * (fabs(b) + t * fabs(c)));
    s = fmin(k.bound[i + 1], s * q);
    const bool last = i + 1 == k.steps;
    const int sa = scale_of(t), sn = last ? 0 : scale_of(s);
    int sb = scale_of(q);
    if (last && sb > 149 - sx) sb = 149 - sx;  // the factor stays a fp32 value; the result is below 2^-120
    out[i].gram = (float)ldexp(1.0, sa - 2 * sx);
    out[i].b2 = (float)ldexp(c, sb - 2 * sa);
    out[i].b1 = (float)ldexp(b, sb - sa);
    out[i].b0 = (float)ldexp(a, sb);
    out[i].apply = (float)ldexp(1.0, sn - sb - sx);
    sx = sn;
  }
}

// The bound to start from, given a matrix's norm: 1 unless eps exceeds the norm.
__host__ __device__ inline double start_of(double norm, double eps) {
  const double s = norm / (norm + eps);
  return s < 0.5 ? s : 1;
}

// One operand as the tensor map and the epilogue see it: per matrix two
// planes (hi, lo) of `rows` rows of `ld` fp16 values.
struct Planes {
  __half* p;
  int rows, ld;
  __device__ __forceinline__ __half* row(uint32_t z, int plane, int r) const {
    return p + ((size_t)(2 * z + plane) * rows + r) * ld;
  }
};

// What becomes of a product.
enum Mode {
  GRAM,   // A = X X^T: planes, both triangles
  POLY,   // B = a I + b A + c A A: planes, both triangles
  APPLY,  // X <- B X: planes
  FINAL,  // the result, in the caller's type
  PART    // of a symmetric product cut along k: fp32 sums to be joined
};

struct GemmArgs {
  int m, n, k;              // rows, columns, length of the product
  int tile_n;               // 256 or 128: columns of a tile of 256 rows
  int tiles_m, tiles_n;
  int tiles;                // per matrix (of a symmetric product: of the upper triangle)
  int total;                // work items: tiles of the batch, times splits
  int splits, split_k;      // PART: parts of k, stages of each
  int sum;                  // stages that TMEM sums before registers do; 0: half a stage
  const Factors* factors;   // of this step, the first matrix's; `steps` on the next one's
  int steps;
  Planes to, from;          // result; POLY: A
  float* part;              // PART
  void* out;
  int out_dtype, vectors;   // vectors: rows of out start on 16-byte boundaries
  int64_t out_rs, out_bs;
  dcf_status* st;
};

__device__ __forceinline__ void store_typed(void* out, int64_t at, int dtype, float v) {
  if (dtype == DCF_F32) ((float*)out)[at] = v;
  else if (dtype == DCF_F16) ((__half*)out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)out)[at] = __float2bfloat16_rn(v);
}

// Two values split at once: the his in one word, the los in another.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(__fsub_rn(a, f.x), __fsub_rn(b, f.y));
  hi = *(const uint32_t*)&h;
  lo = *(const uint32_t*)&l;
}

// Where a work item lies.
struct Tile {
  uint32_t z;
  int row0, col0;
  __device__ __forceinline__ Tile(const GemmArgs& g, int t, bool symmetric) {
    z = (uint32_t)(t / g.tiles);
    int tile = t - (int)z * g.tiles, tm, tn;
    if (symmetric) {
      const int per = kTile / g.tile_n;  // row tm keeps the tiles that reach the diagonal or lie right of it
      for (tm = 0; tile >= g.tiles_n - tm * per; tm++) tile -= g.tiles_n - tm * per;
      tn = tm * per + tile;
    } else {
      tm = tile % g.tiles_m;
      tn = tile / g.tiles_m;
    }
    row0 = tm * kTile;
    col0 = tn * g.tile_n;
  }
};

// A block of 32 rows x 32 columns on its way out: from rows in lanes, through
// 4 KB of shared memory, to eight columns of a row, or eight rows of a column,
// in each lane.  Groups of four rows are exchanged so that none of the three
// has bank conflicts.  (One block at a time on purpose: unrolled over a
// warp's 128 columns the code ran once per tile, and fetching it took 15 us.)
__device__ __forceinline__ uint32_t place(int col, int row) {
  return (uint32_t)(col * 32 + ((((row >> 2) ^ (col & 7) ^ ((col >> 2) & 6)) << 2) | (row & 3)));
}

__device__ __forceinline__ void block_in(float* buf, const float* v, int lane) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; j++) buf[place(j, lane)] = v[j];
  __syncwarp();
}

// Eight values as his and los.
__device__ __forceinline__ void split8(const float (&v)[8], uint4& hi, uint4& lo) {
  split2(v[0], v[1], hi.x, lo.x);
  split2(v[2], v[3], hi.y, lo.y);
  split2(v[4], v[5], hi.z, lo.z);
  split2(v[6], v[7], hi.w, lo.w);
}

// Those of eight 16-bit values with from <= index < to.
__device__ __forceinline__ void put_some(uint16_t* at, const uint4& v, int from, int to) {
  const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j >= from && j < to) at[j] = (uint16_t)(e[j >> 1] >> ((j & 1) * 16));
}

// Eight values of a row of the result, of which `have` (or all) are there, in
// the caller's type; `at` in elements.
__device__ __forceinline__ void put_row8(void* out, int dtype, int vectors, int64_t at, int have, const float (&v)[8]) {
  if (have <= 0) return;
  if (dtype == DCF_F32) {
    float* to = (float*)out + at;
    if (vectors && have >= 8) {
      *(float4*)to = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < have) to[e] = v[e];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (dtype == DCF_F16) {
      const __half2 p = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
      w[e] = *(const uint32_t*)&p;
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
      w[e] = *(const uint32_t*)&p;
    }
  }
  const uint4 x = make_uint4(w[0], w[1], w[2], w[3]);
  uint16_t* to = (uint16_t*)out + at;
  if (vectors && have >= 8) *(uint4*)to = x;
  else put_some(to, x, 0, have);
}

// Writes the block at row r0, column c0 of the result in the caller's type.
__device__ __forceinline__ void write_final(const GemmArgs& g, const Factors& f, uint32_t z, int r0, int c0, const float* buf,
                                            int lane) {
  if (!g.vectors) {  // element by element, a row at a time
    const int64_t at = (int64_t)z * g.out_bs + (int64_t)r0 * g.out_rs + c0 + lane;
    const int rows = c0 + lane < g.n ? min(32, g.m - r0) : 0;
    auto each = [&](auto* out, auto cast) {
      out += at;
#pragma unroll 8
      for (int row = 0; row < 32; row++, out += g.out_rs)
        if (row < rows) *out = cast(__fmul_rn(f.apply, buf[place(lane, row)]));
    };
    if (g.out_dtype == DCF_F32) each((float*)g.out, [](float v) { return v; });
    else if (g.out_dtype == DCF_F16) each((__half*)g.out, [](float v) { return __float2half_rn(v); });
    else each((__nv_bfloat16*)g.out, [](float v) { return __float2bfloat16_rn(v); });
    return;
  }
  const int o = (lane & 3) * 8, c = c0 + o;
#pragma unroll 1
  for (int row = lane >> 2; row < 32 && r0 + row < g.m; row += 8) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = __fmul_rn(f.apply, buf[place(o + e, row)]);
    put_row8(g.out, g.out_dtype, g.vectors, (int64_t)z * g.out_bs + (int64_t)(r0 + row) * g.out_rs + c, g.n - c, v);
  }
}

// The same as planes.  Of a symmetric matrix, blocks right of the diagonal are
// written with their mirror image, and one on it (blocks lie on multiples of
// 32) takes its lower half from its upper.
template <Mode MODE>
__device__ __forceinline__ void write_planes(const GemmArgs& g, const Factors& f, uint32_t z, int r0, int c0, float* buf,
                                             int lane) {
  constexpr bool sym = MODE == GRAM || MODE == POLY;
  const float alpha = MODE == GRAM ? f.gram : MODE == POLY ? f.b2 : f.apply;
  const bool on = sym && c0 == r0;
  const int o = (lane & 3) * 8, c = c0 + o;
  const size_t plane = (size_t)g.to.rows * g.to.ld;
#pragma unroll 4
  for (int row = lane >> 2; row < 32 && r0 + row < g.m; row += 8) {
    const int r = r0 + row;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = __fmul_rn(alpha, buf[on && o + e < row ? place(row, o + e) : place(o + e, row)]);
    if (MODE == POLY) {
      const __half* from = g.from.row(z, 0, r) + c;
      const uint4 x = *(const uint4*)from, y = *(const uint4*)(from + plane);
      const __half2* h = (const __half2*)&x;
      const __half2* l = (const __half2*)&y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 p = __half22float2(h[e]), q = __half22float2(l[e]);
        v[2 * e] = __fmaf_rn(f.b1, __fadd_rn(p.x, q.x), v[2 * e]);
        v[2 * e + 1] = __fmaf_rn(f.b1, __fadd_rn(p.y, q.y), v[2 * e + 1]);
      }
      if (on) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (o + e == row) v[e] = __fadd_rn(v[e], f.b0);
      }
    }
    if (sym && !on) {  // for the mirror image
#pragma unroll
      for (int e = 0; e < 8; e++) buf[place(o + e, row)] = v[e];
    }
    uint4 hi, lo;
    split8(v, hi, lo);
    __half* to = g.to.row(z, 0, r) + c;  // rows are padded to 64 columns: whole vectors fit
    *(uint4*)to = hi;
    *(uint4*)(to + plane) = lo;
  }
  if (!sym || on) return;
  __syncwarp();
  const int r = r0 + o;  // eight rows of one column
  if (r >= g.m) return;
#pragma unroll 4
  for (int col = lane >> 2; col < 32 && c0 + col < g.n; col += 8) {
    const float4 x = *(const float4*)&buf[place(col, o)], y = *(const float4*)&buf[place(col, o + 4)];
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    uint4 hi, lo;
    split8(v, hi, lo);
    __half* to = g.to.row(z, 0, c0 + col) + r;
    *(uint4*)to = hi;
    *(uint4*)(to + plane) = lo;
  }
}

// Values of PART: per item and block, [column][row].
__device__ __forceinline__ float* part_block(const GemmArgs& g, int64_t item, int block) {
  return g.part + (item * (kTile / 32 * (g.tile_n / 32)) + block) * kBlock;
}

// D = P Q^T in tiles of 256 x 256 (256 x 128 where these are few), P and Q given as two fp16 planes each; P_MN,
// Q_MN: its memory has rows of k and runs along the operand, so that no
// operand is ever written transposed.
//
// Persistent pairs of CTAs; each CTA loads 128 rows of P and of Q and keeps the
// result of its rows of P with all of Q: 64 KB of loads feed 12 instructions of
// 128 cycles (one CTA by itself with 128 x 128 tiles waits for its loads and
// for shared memory: twice the time per product, measured).  Warp 0 keeps a ring
// of stages full, 64 columns of all four planes, which three products share.
// One thread of the first CTA issues these for both; the second CTA reports
// its full stages to it.  Eight warps add up and write out.
//
// The tensor core truncates as it accumulates, a bias of some 2^-25 per
// instruction: 1e-4 in the result over k = 8192.  So TMEM sums `sum` stages
// only (the two small products of a stage first, then the large one), in two
// buffers in turn, and the eight warps add the sums in registers, rounding to
// nearest; sums_of says how many stages.
template <Mode MODE, bool P_MN, bool Q_MN, int TN>
__global__ void __launch_bounds__(kGemmThreads, 1) orth_gemm_kernel(const __grid_constant__ CUtensorMap map_p,
                                                                    const __grid_constant__ CUtensorMap map_q,
                                                                    const GemmArgs args) {
  constexpr int kMine = TN / 2;  // columns of one out warp
  const GemmArgs g = args;  // a reference to the parameter itself would be read through memory
  constexpr bool symmetric = MODE == GRAM || MODE == POLY || MODE == PART;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + (-smem_addr(smem_raw) & 1023);  // (a cast through an integer would make every access generic)
  uint8_t* buffers = base + kOrthStages * kStage;
  uint64_t* full = (uint64_t*)(buffers + kOutWarps * kBuffer);  // the first CTA's counts what both have loaded
  uint64_t* empty = full + kOrthStages;
  uint64_t* sum_full = empty + kOrthStages;
  uint64_t* sum_empty = sum_full + 2;     // the first CTA's
  uint32_t* tmem_at = (uint32_t*)(sum_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int first = (int)(blockIdx.x / 2), step = (int)(gridDim.x / 2);
  uint32_t full0;  // the first CTA's
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(full0) : "r"(smem_addr(full)));
  const int all = (g.k + kBK - 1) / kBK;
  // The stages of a work item.
  auto begin_of = [&](int t) { return MODE == PART ? t % g.splits * g.split_k : 0; };
  auto count_of = [&](int t) { return MODE == PART ? min(g.split_k, all - begin_of(t)) : all; };
  auto tile_of = [&](int t) { return Tile(g, MODE == PART ? t / g.splits : t, symmetric); };

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kOrthStages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sum_full[b], 1);
      mbar_init(&sum_empty[b], 2 * kOutWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_at)), "r"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)tmem_at;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_p) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_q) : "memory");
  }
  pdl_begin();

  bool fail = false;
  if (warp < 4) shrink_registers();
  if (warp == 0) {
    if (lane == 0) {
      int64_t i = 0;  // stages so far
      for (int t = first; t < g.total && !fail; t += step) {
        const Tile at = tile_of(t);
        const int row = at.row0 + (int)rank * kSide, col = at.col0 + (int)rank * (TN / 2), z = (int)(2 * at.z);
        const int b0 = begin_of(t), blocks = count_of(t);
        for (int b = 0; b < blocks; b++, i++) {
          const int s = (int)(i % kOrthStages);
          if (i >= kOrthStages && !mbar_wait_bounded(&empty[s], (unsigned)((i / kOrthStages - 1) & 1))) {
            fail = true;
            break;
          }
          const uint32_t to = smem_addr(base + s * kStage);
          const uint32_t bar = full0 + s * 8;
          if (!rank) mbar_expect_tx(&full[s], 2 * 2 * (kSide + TN / 2) * kBK * 2);
#pragma unroll
          for (int half = 0; half < 2; half++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
              const uint32_t at = to + p * kPlane + half * (kPlane / 2);
              const int r = row + half * 64, c = col + half * 64, k = (b0 + b) * kBK;
              pair_load_3d(at, &map_p, P_MN ? r : k, P_MN ? k : r, z + p, bar);
              if (half * 128 < TN) pair_load_3d(at + 2 * kPlane, &map_q, Q_MN ? c : k, Q_MN ? k : c, z + p, bar);
            }
        }
      }
      // Leave only with no copy of ours and no arrival for us left in flight.
      for (int64_t j = i > kOrthStages ? i - kOrthStages : 0; j < i; j++) {
        const unsigned turn = (unsigned)((j / kOrthStages) & 1);
        if (!rank && !mbar_wait_bounded(&full[j % kOrthStages], turn)) fail = true;
        if (!fail && !mbar_wait_bounded(&empty[j % kOrthStages], turn)) fail = true;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && !rank) {
      const uint32_t idesc = (1u << 4) | ((uint32_t)P_MN << 15) | ((uint32_t)Q_MN << 16) |
                             ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
      int64_t i = 0, u = 0;  // stages and sums so far
      for (int t = first; t < g.total && !fail; t += step) {
        const int blocks = count_of(t);
        int in_sum = 0;
        for (int b = 0; b < blocks; b++, i++) {
          const int s = (int)(i % kOrthStages), d = (int)(u & 1);
          const unsigned turn = (unsigned)((i / kOrthStages) & 1);
          if (!mbar_wait_bounded(&full[s], turn) ||
              (in_sum == 0 && u >= 2 && !pair_wait(&sum_empty[d], (unsigned)((u / 2 - 1) & 1)))) {
            fail = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t at = smem_addr(base + s * kStage), to = tmem + d * kTile;
          const uint64_t ph = smem_desc<P_MN>(at), pl = smem_desc<P_MN>(at + kPlane);
          const uint64_t qh = smem_desc<Q_MN>(at + 2 * kPlane), ql = smem_desc<Q_MN>(at + 3 * kPlane);
          constexpr uint32_t ps = kSlice<P_MN>, qs = kSlice<Q_MN>;
          auto products = [&](uint32_t to, uint32_t from, uint32_t end, int in_sum) {
#pragma unroll
            for (uint32_t j = 0; j < kBK / 16; j++)
              if (j >= from && j < end) {
                pair_mma(to, ph + ps * j, ql + qs * j, idesc, in_sum | (int)(j - from));
                pair_mma(to, pl + ps * j, qh + qs * j, idesc, 1);
              }
#pragma unroll
            for (uint32_t j = 0; j < kBK / 16; j++)
              if (j >= from && j < end) pair_mma(to, ph + ps * j, qh + qs * j, idesc, 1);
          };
          if (g.sum == 0) {  // two sums of half a stage: one here, one below
            products(to, 0, kBK / 32, 0);
            pair_commit(&sum_full[d]);
            u++;
            if (u >= 2 && !pair_wait(&sum_empty[u & 1], (unsigned)((u / 2 - 1) & 1))) {
              fail = true;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            products(tmem + (uint32_t)(u & 1) * kTile, kBK / 32, kBK / 16, 0);
          } else {
            products(to, 0, kBK / 16, in_sum);
          }
          pair_commit(&empty[s]);
          if (++in_sum >= g.sum || b == blocks - 1) {
            pair_commit(&sum_full[u & 1]);
            u++;
            in_sum = 0;
          }
        }
      }
    }
  } else if (warp >= 4) {
    grow_registers();
    const int part = warp & 3;               // the 32 TMEM lanes this warp may read
    const int col = (warp - 4) / 4 * kMine;  // and the half of the columns it takes
    float* buf = (float*)(buffers + (warp - 4) * kBuffer);
    const uint32_t lanes = tmem + ((uint32_t)(part * 32) << 16) + col;
    int64_t u = 0;  // sums so far
    for (int t = first; t < g.total && !fail; t += step) {
      const Tile at = tile_of(t);
      Factors f = {};
      if (MODE != PART) f = g.factors[(size_t)at.z * g.steps];
      const int sums = g.sum ? (count_of(t) + g.sum - 1) / g.sum : 2 * count_of(t);
      float acc[kMine];
#pragma unroll
      for (int j = 0; j < kMine; j++) acc[j] = 0;
      for (int b = 0; b < sums; b++, u++) {
        const int d = (int)(u & 1);
        if (__any_sync(0xFFFFFFFFu, !mbar_wait_bounded(&sum_full[d], (unsigned)((u >> 1) & 1)))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t x[2][32];  // one part is added while the next arrives
        tmem_load32(lanes + d * kTile, x[0]);
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          tmem_wait(x[c / 32 & 1]);
          if (c + 32 < kMine) {
            tmem_load32(lanes + d * kTile + c + 32, x[(c / 32 + 1) & 1]);
          } else {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) arrive_first<false>(&sum_empty[d]);
          }
#pragma unroll
          for (int j = 0; j < 32; j++) acc[c + j] = __fadd_rn(acc[c + j], __uint_as_float(x[c / 32 & 1][j]));
        }
      }
      if (fail) break;
      const int row = (int)rank * kSide + part * 32, r0 = at.row0 + row;
#pragma unroll 1
      for (int c = 0; c < kMine; c += 32) {
        const int c0 = at.col0 + col + c;
        // beyond the matrix, or below the diagonal: written by its mirror image
        if (r0 < g.m && c0 < g.n && !(symmetric && c0 + 31 < r0)) {
          if (MODE == PART) {
            float* p = part_block(g, t, row / 32 * (TN / 32) + (col + c) / 32) + lane;
#pragma unroll
            for (int j = 0; j < 32; j++) p[j * 32] = acc[j];
          } else {
            block_in(buf, acc, lane);
            if (MODE == FINAL) write_final(g, f, at.z, r0, c0, buf, lane);
            else write_planes<MODE>(g, f, at.z, r0, c0, buf, lane);
          }
        }
#pragma unroll
        for (int j = 0; j < kMine - 32; j++) acc[j] = acc[j + 32];
      }
    }
  }
  if (fail) atomicExch(&g.st->error, 1u);
  __syncthreads();
  pair_sync();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
  }
}

// Joins the parts of a symmetric product, always in the same order; a warp
// takes a block.
constexpr int kJoinWarps = 1;  // (four to a block: 255 us instead of 206 at 256 x 2500, three steps)
template <Mode MODE>
__global__ void __launch_bounds__(32 * kJoinWarps) orth_join_kernel(const GemmArgs args) {
  const GemmArgs g = args;
  __shared__ __align__(16) float buffers[kJoinWarps][kBlock];
  pdl_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wide = g.tile_n / 32, blocks = kTile / 32 * wide;
  const int64_t id = (int64_t)blockIdx.x * kJoinWarps + warp, item = id / blocks;
  const int block = (int)(id % blocks);
  if (item >= g.total) return;
  const Tile at(g, (int)item, true);
  const int r0 = at.row0 + block / wide * 32, c0 = at.col0 + block % wide * 32;
  if (r0 >= g.m || c0 >= g.n || c0 + 31 < r0) return;
  const Factors f = g.factors[(size_t)at.z * g.steps];
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; j++) v[j] = 0;
#pragma unroll 4
  for (int s = 0; s < g.splits; s++) {
    const float* p = part_block(g, item * g.splits + s, block) + lane;
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = __fadd_rn(v[j], p[j * 32]);
  }
  block_in(buffers[warp], v, lane);
  write_planes<MODE>(g, f, at.z, r0, c0, buffers[warp], lane);
}

// ------------------------------------------------------- norm and split

struct MatArgs {
  const void* in;
  int dtype;
  int rows, cols;
  int64_t rs, bs;
  int vectors;           // rows start on 16-byte boundaries
};

// Eight columns of a row from column c (a multiple of 8) on, zeros behind the
// row; with `vectors`, whole ones are read as 16-byte vectors.
__device__ __forceinline__ void load_row8(const MatArgs& a, uint32_t z, int r, int c, float (&v)[8]) {
  const int64_t at = (int64_t)z * a.bs + (int64_t)r * a.rs + c;
  if (a.vectors && c + 8 <= a.cols) {
    if (a.dtype == DCF_F32) {
      const float4 x = *(const float4*)((const float*)a.in + at), y = *(const float4*)((const float*)a.in + at + 4);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
      const uint4 x = *(const uint4*)((const uint16_t*)a.in + at);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const unsigned short b = (unsigned short)(w[j >> 1] >> ((j & 1) * 16));
        v[j] = a.dtype == DCF_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    v[j] = 0;
    if (c + j >= a.cols) continue;
    if (a.dtype == DCF_F32) v[j] = ((const float*)a.in)[at + j];
    else if (a.dtype == DCF_F16) v[j] = __half2float(((const __half*)a.in)[at + j]);
    else v[j] = __bfloat162float(((const __nv_bfloat16*)a.in)[at + j]);
  }
}

// scale / (norm + eps); 0 for a matrix of zeros, which stays one however small eps is.
__device__ __forceinline__ double factor_of(double norm, double eps, double scale) {
  return norm == 0 && eps > 0 ? 0 : scale / (norm + eps);
}

constexpr int kNormThreads = 256;

// Sums of squares in 64 bits (a f32 element's square can pass 32), one part
// per block.
__global__ void __launch_bounds__(kNormThreads) orth_norm_kernel(const __grid_constant__ MatArgs a, double* part) {
  pdl_begin();
  const uint32_t z = blockIdx.y, groups = (uint32_t)(a.cols + 7) / 8;
  const uint64_t total = (uint64_t)groups * a.rows;
  double s = 0;
  for (uint64_t i = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x; i < total; i += (uint64_t)gridDim.x * kNormThreads) {
    float v[8];
    load_row8(a, z, (int)(i / groups), (int)(i % groups) * 8, v);
#pragma unroll
    for (int j = 0; j < 8; j++) s = __fma_rn((double)v[j], (double)v[j], s);
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

// X = G / (norm + eps) into its planes and the matrix's factors beside them, or, with
// no steps to take, straight to the result.  A thread takes eight columns of a row.
__global__ void __launch_bounds__(kNormThreads) orth_split_kernel(const __grid_constant__ MatArgs a,
                                                                  const __grid_constant__ Scaling k, const double* part,
                                                                  int parts, Planes x, Factors* factors, void* out,
                                                                  int out_dtype, int64_t out_rs, int64_t out_bs) {
  __shared__ double factor;
  pdl_begin();
  const uint32_t z = blockIdx.y;
  if (threadIdx.x < 32) {
    double s = 0;
    for (int i = threadIdx.x; i < parts; i += 32) s += part[(size_t)z * parts + i];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    const double norm = sqrt(s), start = start_of(norm, k.eps);
    if (threadIdx.x == 0) factor = factor_of(norm, k.eps, k.steps ? ldexp(1.0, scale_of(start)) : 1.0);
    if (blockIdx.x == 0 && threadIdx.x < k.steps) {
      Factors* to = factors + (size_t)z * k.steps;
      if (start == 1) to[threadIdx.x] = k.usual[threadIdx.x];
      else if (threadIdx.x == 0) set_factors(k, start, to);
    }
  }
  __syncthreads();
  const double f = factor;
  const uint32_t groups = (uint32_t)(a.cols + 7) / 8;
  const uint64_t total = (uint64_t)groups * a.rows;
  for (uint64_t i = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x; i < total; i += (uint64_t)gridDim.x * kNormThreads) {
    const int r = (int)(i / groups), c = (int)(i % groups) * 8;
    float v[8];
    load_row8(a, z, r, c, v);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)((double)v[j] * f);
    if (out) {
      for (int j = 0; j < 8 && c + j < a.cols; j++)
        store_typed(out, (int64_t)z * out_bs + (int64_t)r * out_rs + c + j, out_dtype, v[j]);
    } else {
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; j++) split2(v[2 * j], v[2 * j + 1], h[j], l[j]);
      *(uint4*)(x.row(z, 0, r) + c) = make_uint4(h[0], h[1], h[2], h[3]);  // rows are padded to 64 columns
      *(uint4*)(x.row(z, 1, r) + c) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  }
}

// ------------------------------------------------ matrices of few rows

// The whole iteration of a matrix with min(rows, cols) <= 128 in one launch.  A
// cluster of CTAs keeps X in shared memory, cut along its longer side, as the
// two planes that the products read; a step's three products then read nothing
// else:
//   - each CTA multiplies its slice into a part of A (TMEM); the parts are
//     added over the cluster, every CTA a share of the rows, and the sums written to
//     all;
//   - each CTA makes B from A by itself and multiplies it with its slice.
// What bounds it is latency: three products of 24 to 48 instructions, three
// passes over 128 x 128 accumulators and, in a cluster, three barriers per step.  The
// separate products of orth_gemm_kernel took 17 launches of 8 to 28 us
// (96 x 96: 157 us, 32 x 128 x 1000: 300 us).
//
// Shared memory has 64 columns of a plane as rows of 128 bytes with the
// 128-byte swizzle.  The same bytes are a K-major operand (its 64 columns along k)
// and an MN-major one (its rows along k), so that X serves X X^T and B X as
// it lies, whichever of its sides is the longer.
constexpr int kFewThreads = 512, kFewSlice = 256, kFewCluster = 8;
constexpr int kFewPlane = 128 * 128 * 2;       // a plane of A or B
constexpr int kFewTmem = 512;
constexpr int kFewLeast = 120 << 10;           // shared memory that keeps a second CTA off the SM and its TMEM

struct FewArgs {
  MatArgs in;
  void* out;
  int out_dtype, vectors;
  int64_t out_rs, out_bs;
  int tall;                 // rows > cols: X^T is what lies in memory
  int slice;                // of the longer side per CTA: a multiple of 64 (128 where tall)
  Scaling k;
  dcf_status* st;
};

__device__ __forceinline__ void one_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void one_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

// One operand of a product: descriptors of its first 16 k in both planes, and
// how far on the next 16 and the next 64 are.
struct Operand {
  uint64_t hi, lo;
  uint32_t step, chunk, mn;
};

__device__ __forceinline__ Operand k_major(uint32_t at, uint32_t plane, uint32_t block) {  // blocks of 64 k
  return {smem_desc<false>(at), smem_desc<false>(at + plane), 32 >> 4, block >> 4, 0};
}

__device__ __forceinline__ Operand mn_major(uint32_t at, uint32_t plane, uint32_t block) {  // blocks of 64 along the operand
  const uint64_t far = ((uint64_t)(block >> 4) << 16) - (1ull << 16);
  return {smem_desc<false>(at) + far, smem_desc<false>(at + plane) + far, 2048 >> 4, 4 * (2048 >> 4), 1};
}

// Every PER slices of 16 k have an accumulator of their own, `pitch` columns after
// the last, and the small products come first, while its sum is small: the tensor
// core truncates.  Four slices, and two in A A (from 64 bits, f32 at
// 79 x 249: 1.4e-6; with four 1.9e-6, with two in all products 1.3e-6 but 14 us of 38
// more at 96 x 96; plain fp32 products 1.1e-6).  Of few rows most of A's and B's k is
// zero and left out, and the accumulators it would take halve the runs: up to 80 rows one
// slice in A A, up to 64 two in B X (60 x 1000: 3.3e-6 -> 2.3e-6, plain fp32 products 2.0e-6;
// 8 x 60 x 60: 30 -> 28 us).
template <int PER>
__device__ __forceinline__ void one_product(uint32_t d, int pitch, const Operand& p, const Operand& q, int n, int from,
                                            int to) {
  const uint32_t idesc =
      (1u << 4) | (p.mn << 15) | (q.mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
#pragma unroll 1
  for (int s = from; s < to; s += PER, d += pitch) {  // a run of slices lies in one chunk of 64 k
    const uint32_t po = (uint32_t)(s >> 2) * p.chunk + (uint32_t)(s & 3) * p.step;
    const uint32_t qo = (uint32_t)(s >> 2) * q.chunk + (uint32_t)(s & 3) * q.step;
    const uint64_t ph = p.hi + po, pl = p.lo + po, qh = q.hi + qo, ql = q.lo + qo;
#pragma unroll
    for (uint32_t k = 0; k < PER; k++) {
      one_mma(d, ph + k * p.step, ql + k * q.step, idesc, k);
      one_mma(d, pl + k * p.step, qh + k * q.step, idesc, 1);
    }
#pragma unroll
    for (uint32_t k = 0; k < PER; k++) one_mma(d, ph + k * p.step, qh + k * q.step, idesc, 1);
  }
}

// 32 columns of a product: its accumulators' sum.
__device__ __forceinline__ void product_of(uint32_t addr, int pitch, int chunks, float (&v)[32]) {
  uint32_t x[32];
  tmem_load32(addr, x);
  tmem_wait(x);
#pragma unroll
  for (int j = 0; j < 32; j++) v[j] = __uint_as_float(x[j]);
#pragma unroll 1
  for (int c = 1; c < chunks; c++) {
    addr += pitch;
    tmem_load32(addr, x);
    tmem_wait(x);
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = __fadd_rn(v[j], __uint_as_float(x[j]));
  }
}

// Eight values of a row to their place in both planes.
__device__ __forceinline__ uint32_t few_offset(int row, int col, uint32_t block) {
  return (uint32_t)(col >> 6) * block + (uint32_t)row * 128 + (uint32_t)((((col & 63) >> 3) ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint32_t remote(uint32_t local, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync(int ctas) {
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
}

__global__ void __launch_bounds__(kFewThreads, 1) orth_few_kernel(const __grid_constant__ FewArgs g) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + (-smem_addr(smem_raw) & 1023);  // (a cast through an integer would make every access generic)
  __shared__ uint64_t done;
  __shared__ uint32_t tmem_at;
  __shared__ double sums[kFewThreads / 32], own;
  __shared__ Factors factors[DCF_ORTH_MAX_STEPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int ctas, rank;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t z = blockIdx.x / (uint32_t)ctas;
  // X's slice as it lies in memory: wide 128 rows x slice columns, tall slice rows x 128.
  const int rows = g.tall ? g.slice : 128, cols = g.tall ? 128 : g.slice;
  const int row0 = g.tall ? rank * g.slice : 0, col0 = g.tall ? 0 : rank * g.slice;
  const int m = g.tall ? g.in.cols : g.in.rows;
  const uint32_t block = (uint32_t)rows * 128, plane = (uint32_t)rows * (uint32_t)cols * 2;
  uint8_t* ab = base + 2 * plane;       // A, then B: two planes; the parts of A before that
  const uint32_t x_at = smem_addr(base), ab_at = smem_addr(ab);

  if (threadIdx.x == 0) {
    mbar_init(&done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(kFewTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)&tmem_at;
  pdl_begin();

  // The norm, in 64 bits: of the slice, then of the cluster's.
  const int groups = cols / 8;
  double s = 0;
#pragma unroll 2
  for (int i = threadIdx.x; i < rows * groups; i += kFewThreads) {
    const int r = row0 + i / groups, c = col0 + i % groups * 8;
    if (r >= g.in.rows || c >= g.in.cols) continue;
    float v[8];
    load_row8(g.in, z, r, c, v);
#pragma unroll
    for (int j = 0; j < 8; j++) s = __fma_rn((double)v[j], (double)v[j], s);
  }
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (lane == 0) sums[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kFewThreads / 32; w++) s += sums[w];
    own = s;
  }
  cluster_sync(ctas);
  double norm = 0;
  for (int k = 0; k < ctas; k++) {
    double part;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(part) : "r"(remote(smem_addr(&own), k)) : "memory");
    norm += part;
  }
  norm = sqrt(norm);
  const double start = start_of(norm, g.k.eps), factor = factor_of(norm, g.k.eps, ldexp(1.0, scale_of(start)));
  if (start == 1) {
    if (threadIdx.x < g.k.steps) factors[threadIdx.x] = g.k.usual[threadIdx.x];
  } else if (threadIdx.x == 0) {
    set_factors(g.k, start, factors);
  }
  for (int i = threadIdx.x; i < rows * groups; i += kFewThreads) {
    const int lr = i / groups, lc = i % groups * 8, r = row0 + lr, c = col0 + lc;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r < g.in.rows && c < g.in.cols) {
      load_row8(g.in, z, r, c, v);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = c + j < g.in.cols ? (float)((double)v[j] * factor) : 0;
    }
    uint4 hi, lo;
    split8(v, hi, lo);
    uint8_t* at = base + few_offset(lr, lc, block);
    *(uint4*)at = hi;
    *(uint4*)(at + plane) = lo;
  }

  const Operand x_mn = mn_major(x_at, plane, block), ab_k = k_major(ab_at, kFewPlane, 128 * 128);
  const Operand x_gram = g.tall ? x_mn : k_major(x_at, plane, block);
  const int part = warp & 3, quarter = warp >> 2, row = part * 32 + lane;  // TMEM lanes; columns
  const uint32_t lanes = tmem + ((uint32_t)(part * 32) << 16);
  // A A: columns, and slices of 16 k that are not all zero.
  const int square = m > 64 && m <= 80 ? 96 : 128, slices = m <= 64 ? 4 : m <= 80 ? 5 : 8;
  bool fail = false;
  unsigned phase = 0;
  auto before = [&]() {  // shared memory written so far is what the products read
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  auto after = [&]() {
    if (!mbar_wait_bounded(&done, phase)) fail = true;
    phase ^= 1;
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };

  for (int step = 0; step < g.k.steps; step++) {
    before();
    if (threadIdx.x == 0) {
      one_product<4>(tmem, 128, x_gram, x_gram, 128, 0, g.slice / 16);
      one_commit(&done);
    }
    after();
    const int c = quarter * 32;
    float sum[32];  // this thread's row, 32 columns
    product_of(lanes + c, 128, g.slice / 64, sum);
    const float fa = factors[step].gram;
    if (ctas == 1) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __fmul_rn(fa, sum[8 * k + j]);
        uint4 hi, lo;
        split8(v, hi, lo);
        uint8_t* at = ab + few_offset(row, c + 8 * k, 128 * 128);
        *(uint4*)at = hi;
        *(uint4*)(at + kFewPlane) = lo;
      }
    } else {
      // Parts as rows of 512 bytes, their 16-byte chunks exchanged by row.
#pragma unroll
      for (int k = 0; k < 8; k++)
        *(float4*)(ab + row * 512 + (((c >> 2) + k) ^ (row & 7)) * 16) =
            make_float4(sum[4 * k], sum[4 * k + 1], sum[4 * k + 2], sum[4 * k + 3]);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      cluster_sync(ctas);
      // Rows rank * 128 / ctas on, eight columns at a time: 16 values a thread at most.
      const int share = 128 / ctas, items = share * 16;
      float v[2][8];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int i = u * kFewThreads + (int)threadIdx.x;
        if (i >= items) break;
        const int r = rank * share + i / 16, c4 = i % 16 * 2;
        const uint32_t at0 = ab_at + (uint32_t)(r * 512 + (c4 ^ (r & 7)) * 16);
        const uint32_t at1 = ab_at + (uint32_t)(r * 512 + ((c4 + 1) ^ (r & 7)) * 16);
#pragma unroll
        for (int j = 0; j < 8; j++) v[u][j] = 0;
        for (int k = 0; k < ctas; k += 4) {  // eight loads in flight
          float4 p[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            p[e] = make_float4(0, 0, 0, 0);
            if (k + (e >> 1) < ctas)
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(p[e].x), "=f"(p[e].y), "=f"(p[e].z), "=f"(p[e].w)
                           : "r"(remote(e & 1 ? at1 : at0, k + (e >> 1))));
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            v[u][4 * (e & 1)] = __fadd_rn(v[u][4 * (e & 1)], p[e].x);
            v[u][4 * (e & 1) + 1] = __fadd_rn(v[u][4 * (e & 1) + 1], p[e].y);
            v[u][4 * (e & 1) + 2] = __fadd_rn(v[u][4 * (e & 1) + 2], p[e].z);
            v[u][4 * (e & 1) + 3] = __fadd_rn(v[u][4 * (e & 1) + 3], p[e].w);
          }
        }
      }
      cluster_sync(ctas);  // everyone has read: the parts may be overwritten
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int i = u * kFewThreads + (int)threadIdx.x;
        if (i >= items) break;
        const int r = rank * share + i / 16, c = i % 16 * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) v[u][j] = __fmul_rn(fa, v[u][j]);
        uint4 hi, lo;
        split8(v[u], hi, lo);
        const uint32_t at = ab_at + few_offset(r, c, 128 * 128);
        for (int k = 0; k < ctas; k++) {
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(remote(at, k)), "r"(hi.x), "r"(hi.y),
                       "r"(hi.z), "r"(hi.w)
                       : "memory");
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(remote(at + kFewPlane, k)), "r"(lo.x),
                       "r"(lo.y), "r"(lo.z), "r"(lo.w)
                       : "memory");
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      cluster_sync(ctas);
    }
    before();
    if (threadIdx.x == 0) {
      if (m <= 80) one_product<1>(tmem, square, ab_k, ab_k, square, 0, slices);
      else one_product<2>(tmem, square, ab_k, ab_k, square, 0, slices);
      one_commit(&done);
    }
    after();
    const float fb2 = factors[step].b2, fb1 = factors[step].b1, fb0 = factors[step].b0;
    {
      float x[32];
      if (c < square) {
        product_of(lanes + c, square, m <= 80 ? slices : slices / 2, x);
      } else {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = 0;
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        uint8_t* at = ab + few_offset(row, c + 8 * k, 128 * 128);
        const uint4 ah = *(const uint4*)at, al = *(const uint4*)(at + kFewPlane);
        const __half2* h = (const __half2*)&ah;
        const __half2* l = (const __half2*)&al;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float2 p = __half22float2(h[j]), q = __half22float2(l[j]);
          v[2 * j] = __fmaf_rn(fb1, __fadd_rn(p.x, q.x), __fmul_rn(fb2, x[8 * k + 2 * j]));
          v[2 * j + 1] = __fmaf_rn(fb1, __fadd_rn(p.y, q.y), __fmul_rn(fb2, x[8 * k + 2 * j + 1]));
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (c + 8 * k + j == row && row < m) v[j] = __fadd_rn(v[j], fb0);
        uint4 hi, lo;
        split8(v, hi, lo);
        *(uint4*)at = hi;
        *(uint4*)(at + kFewPlane) = lo;
      }
    }
    before();
    if (threadIdx.x == 0) {
      auto apply = [&](auto product, int to) {
        if (g.tall)
          for (int b = 0; b < g.slice / 128; b++)
            product(tmem + b * 128, g.slice, k_major(x_at + (uint32_t)b * 128 * 128, plane, block), ab_k, 128, 0, to);
        else
          product(tmem, g.slice, ab_k, x_mn, g.slice, 0, to);
      };
      if (m <= 64) apply(one_product<2>, 4);
      else apply(one_product<4>, 8);
      one_commit(&done);
    }
    after();
    // The accumulators: wide 128 rows x slice columns, tall slice / 128 blocks of
    // 128 x 128 beside each other.
    const float fx = factors[step].apply;
#pragma unroll 1
    for (int at_col = quarter * 32; at_col < g.slice; at_col += 128) {
      const int lr = g.tall ? (at_col & ~127) + row : row, lc = g.tall ? at_col & 127 : at_col;
      float x[32];
      product_of(lanes + at_col, g.slice, 2, x);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __fmul_rn(fx, x[8 * k + j]);
        if (step + 1 < g.k.steps) {
          uint4 hi, lo;
          split8(v, hi, lo);
          uint8_t* at = base + few_offset(lr, lc + 8 * k, block);
          *(uint4*)at = hi;
          *(uint4*)(at + plane) = lo;
        } else if (row0 + lr < g.in.rows) {
          const int64_t at = (int64_t)z * g.out_bs + (int64_t)(row0 + lr) * g.out_rs + col0 + lc + 8 * k;
          put_row8(g.out, g.out_dtype, g.vectors, at, g.in.cols - (col0 + lc + 8 * k), v);
        }
      }
    }
  }
  if (fail) atomicExch(&g.st->error, 1u);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync(ctas);  // no one leaves while its shared memory may be read
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kFewTmem) : "memory");
  }
}

// ---------------------------------------------------------------- host

// Boxes of 64 columns x 64 rows of one plane; what lies beyond the matrix
// reads as zero.
bool encode(CUtensorMap* map, const Planes& x, int cols, uint64_t batch) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)x.rows, 2 * batch};
  const cuuint64_t strides[2] = {(cuuint64_t)x.ld * 2, (cuuint64_t)x.ld * 2 * (cuuint64_t)x.rows};
  const cuuint32_t box[3] = {64, 64, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, x.p, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int round64(uint64_t v) { return (int)((v + 63) / 64 * 64); }

// Bounds of one step on [0, s]: the largest |a s + b s^3 + c s^5| and
// |a + b s^2 + c s^4|, from the ends and the points where the derivative is
// zero, in t = s^2.  (The roots of a + 3 b t + 5 c t^2 in the form without
// cancellation: a c that is nearly 0 puts one far away and leaves the other at
// -a / 3 b.  A coefficient of 0 gives infinities or NaN, which lie outside.)
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
  at(-b / (2 * c));
  const double d = 9 * b * b - 20 * a * c;
  if (d >= 0) {
    const double w = -(3 * b + copysign(sqrt(d), b)) / 2;
    at(w / (5 * c));
    at(a / w);
  }
}

Scaling scaling_of(const dcf_orth_desc& d) {
  Scaling k = {};
  k.steps = (int)d.steps;
  k.eps = d.eps;
  k.bound[0] = 1;
  for (int i = 0; i < k.steps; i++) {
    for (int j = 0; j < 3; j++) k.coef[i][j] = d.coef[i][j];
    step_bounds(k.coef[i], k.bound[i], &k.bound[i + 1], &k.largest[i]);
  }
  set_factors(k, 1, k.usual);
  return k;
}

constexpr double kMostSingular = 64;

// Stages of 64 k that TMEM sums before registers do, 0 for half a stage: few
// enough for the result to be as near to 64 bits as with products of fp32 values.
//
// f32 results: every stage (8192 x 2048: 2.8e-6; two stages 6e-6, fp32 products
// 5.4e-6), and every half stage in A A, whose truncation the next step amplifies, of up to
// 1024 rows, where fp32 products are nearer (258 x 131, six steps: 3.6e-6 with whole
// stages, 2.4e-6 with half ones, fp32 products 2.1e-6).
//
// 16-bit results hide less than that: the share of them that is not the 64-bit value
// rounded is proportional to the error before the rounding.  Up to 768 rows as for
// f32 (bf16 258 x 131, six steps: 0.21 % of the results, with two stages 0.58 %, fp32 products
// 0.17 %; 520 x 530: two stages 0.33 %, fp32 products 0.20 %), above two stages (4096 x 4096:
// 0.25 % and 3.6 ms, with 16 1.8 % and 3.4 ms, fp32 products 0.33 %), up to 1024 rows one in A A
// (1024 x 4096: 0.16 %, with two 0.23 % and 1 us less, with 16 1.6 % and 11 us less of 438, fp32
// products 0.27 %; 770 x 1540: with two 1.8 times as many as fp32 products).
int sums_of(const dcf_orth_desc& d, int m, bool square) {
  const bool f32 = d.out_dtype == DCF_F32;
  if (square && m <= 1024) return f32 || m <= 768 ? 0 : 1;
  return f32 || m <= 768 ? 1 : 2;
}

// Pairs of SMs on a B200: not asked of the device, as a workspace's size needs none and
// the parts of a sum are then the same everywhere.  Any number runs the persistent grids.
constexpr int kPairs = 74;

// Blocks of the norm's sum: 32 KB of a f32 matrix each, 256 at most.
int norm_parts(const dcf_orth_desc& d) {
  const uint64_t p = (d.rows * d.cols + 8191) / 8192;
  return (int)(p < 256 ? p : 256);
}

// How a product is laid out: columns of a tile, and for a symmetric one the
// parts into which its k is cut, `stages` stages each.
struct Cut {
  int tile_n, splits, stages;
};

int64_t upper_tiles(int m, int tile_n) {
  const int64_t tm = (m + kTile - 1) / kTile, tn = (m + tile_n - 1) / tile_n;
  return tm * tn - tm * (tm - 1) / 2 * (kTile / tile_n);
}

// In units of a stage of a 256 x 256 tile (0.85 us): every round of tiles costs its
// stages (those of a 256 x 128 tile 0.65 each: its loads bound it), a launch some 16
// to start and to write both triangles, 11 with the smaller tile; cut along k, which keeps
// pairs of SMs busy that would have no tile, some 10 (8) to write parts and 12 to join them.
Cut cut_of(int m, uint64_t batch, int stages) {
  Cut best = {256, 1, stages};
  double least = 1e300;
  for (int tile_n : {256, 128}) {
    const int64_t tiles = upper_tiles(m, tile_n) * (int64_t)batch;
    const double stage = tile_n == 256 ? 1 : 0.65;
    const double whole = (double)((tiles + kPairs - 1) / kPairs) * stages * stage + (tile_n == 256 ? 16 : 11);
    if (whole < least) {
      least = whole;
      best = {tile_n, 1, stages};
    }
    for (int s = 2; s <= stages && tiles * s <= kPairs; s++) {
      const int each = (stages + s - 1) / s, parts = (stages + each - 1) / each;
      const double cost = each * stage + (tile_n == 256 ? 22 : 20);
      if (cost < least) {
        least = cost;
        best = {tile_n, parts, each};
      }
    }
  }
  return best;
}

// The workspace: X twice (a step reads one and writes the other), A, B, and
// the parts of A or B.
struct Layout {
  Planes x[2], a, b;
  float* sums;
  Cut gram, poly;
  double* part;
  int parts;
  Factors* factors;
  size_t bytes;
};

Layout layout_of(const dcf_orth_desc& d, void* ws) {
  Layout l;
  const int m = (int)(d.rows < d.cols ? d.rows : d.cols);
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
  l.parts = norm_parts(d);
  l.part = (double*)take(d.batch * l.parts * 8);
  l.factors = d.steps ? (Factors*)take(d.batch * d.steps * sizeof(Factors)) : nullptr;
  l.x[0] = l.x[1] = l.a = l.b = Planes{nullptr, 0, 0};
  if (d.steps) {
    l.x[0] = planes((int)d.rows, (int)d.cols);
    l.a = planes(m, m);
    l.b = planes(m, m);
  }
  if (d.steps > 1) l.x[1] = planes((int)d.rows, (int)d.cols);
  const int n = (int)(d.rows < d.cols ? d.cols : d.rows);
  l.gram = cut_of(m, d.batch, (n + kBK - 1) / kBK);
  l.poly = cut_of(m, d.batch, (m + kBK - 1) / kBK);
  size_t sums = 0;
  for (const Cut& c : {l.gram, l.poly})
    if (c.splits > 1) {
      const size_t bytes = (size_t)upper_tiles(m, c.tile_n) * d.batch * c.splits * kTile * c.tile_n * 4;
      if (bytes > sums) sums = bytes;
    }
  l.sums = d.steps && sums ? (float*)take(sums) : nullptr;
  l.bytes = off;
  return l;
}

// CTAs of a cluster that take a matrix of few rows at once, 0 where it does not
// fit: the longer side is at most 8 x 256.  As few as hold it: more of them have
// less to multiply, but joining their parts of A costs a step 7 us, and a product
// of 256 k 2 us (128 x 256: 48 us with two, 35 us with one, 3 steps).
int few_ctas(const dcf_orth_desc& d) {
  const uint64_t m = d.rows < d.cols ? d.rows : d.cols, n = d.rows < d.cols ? d.cols : d.rows;
  if (!d.steps || m > 128 || n > kFewSlice * kFewCluster) return 0;
  int c = 1;
  while ((uint64_t)c * kFewSlice < n) c *= 2;
  return c;
}

int launch_few(const dcf_orth_desc& d, const MatArgs& in, void* out, int64_t out_rs, int64_t out_bs, int vectors,
               dcf_status* st, cudaStream_t s) {
  const int ctas = few_ctas(d);
  FewArgs g = {};
  g.in = in;
  g.out = out;
  g.out_dtype = (int)d.out_dtype;
  g.vectors = vectors;
  g.out_rs = out_rs;
  g.out_bs = out_bs;
  g.tall = d.rows > d.cols;
  const int n = (int)(g.tall ? d.rows : d.cols), unit = g.tall ? 128 : 64;
  g.slice = ((n + ctas - 1) / ctas + unit - 1) / unit * unit;
  g.k = scaling_of(d);
  g.st = st;
  int smem = 2 * (128 * g.slice * 2) + 2 * kFewPlane + 1024;
  if (smem < kFewLeast) smem = kFewLeast;
  if (!prepare_smem((const void*)orth_few_kernel, 2 * (128 * kFewSlice * 2) + 2 * kFewPlane + 1024)) return DCF_ECUDA;
  return launch(orth_few_kernel, dim3((unsigned)(d.batch * ctas)), kFewThreads, smem, ctas, s, g);
}

template <Mode MODE, bool P_MN, bool Q_MN>
int gemm_run(const CUtensorMap& p, const CUtensorMap& q, const GemmArgs& g, cudaStream_t s) {
  auto kernel = g.tile_n == 256 ? orth_gemm_kernel<MODE, P_MN, Q_MN, 256> : orth_gemm_kernel<MODE, P_MN, Q_MN, 128>;
  if (!prepare_smem((const void*)kernel, kGemmSmem)) return DCF_ECUDA;
  const unsigned pairs = (unsigned)(g.total < kPairs ? g.total : kPairs);
  return launch(kernel, dim3(2 * pairs), kGemmThreads, kGemmSmem, 2, s, p, q, g);
}

template <Mode MODE, bool P_MN, bool Q_MN>
int gemm(const CUtensorMap& p, const CUtensorMap& q, GemmArgs g, uint64_t batch, cudaStream_t s) {
  g.tiles_m = (g.m + kTile - 1) / kTile;
  // Narrower tiles where they leave no pair a second one: less to write for each.
  g.tile_n = (uint64_t)g.tiles_m * ((g.n + 127) / 128) * batch <= (uint64_t)kPairs ? 128 : 256;
  g.tiles_n = (g.n + g.tile_n - 1) / g.tile_n;
  g.tiles = g.tiles_m * g.tiles_n;
  g.total = (int)(g.tiles * batch);
  return gemm_run<MODE, P_MN, Q_MN>(p, q, g, s);
}

// A symmetric product, cut along k where that pays.
template <Mode MODE, bool MN>
int gemm_symmetric(const CUtensorMap& x, GemmArgs g, const Cut& cut, uint64_t batch, cudaStream_t s) {
  g.tile_n = cut.tile_n;
  g.tiles_m = (g.m + kTile - 1) / kTile;
  g.tiles_n = (g.m + g.tile_n - 1) / g.tile_n;
  g.tiles = (int)upper_tiles(g.m, g.tile_n);
  g.total = (int)(g.tiles * batch);
  g.splits = cut.splits;
  g.split_k = cut.stages;
  if (cut.splits == 1) return gemm_run<MODE, MN, MN>(x, x, g, s);
  GemmArgs parts = g;
  parts.total *= cut.splits;
  if (int rc = gemm_run<PART, MN, MN>(x, x, parts, s)) return rc;
  const int64_t warps = (int64_t)g.total * (kTile / 32 * (g.tile_n / 32));
  const unsigned blocks = (unsigned)((warps + kJoinWarps - 1) / kJoinWarps);
  return launch(orth_join_kernel<MODE>, dim3(blocks), 32 * kJoinWarps, 0, 1, s, g);
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
    // below, powers of two that scale what is kept leave the range of fp32
    if (!(q >= 1e-30) || !(s >= 1e-30)) return bad("orthogonalize: the coefficients leave nothing");
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
  if (!d.batch || !d.rows || !d.cols || few_ctas(d)) return 0;
  return layout_of(d, nullptr).bytes;
}

int launch_orthogonalize(const dcf_orth_desc& d, const void* in, void* out, void* ws, dcf_status* st, cudaStream_t s) {
  const Layout l = layout_of(d, ws);
  const int rows = (int)d.rows, cols = (int)d.cols;
  const bool tall = rows > cols;  // then the memory is X^T, and X <- B X is X^T <- X^T B
  const int m = tall ? cols : rows, n = tall ? rows : cols;
  MatArgs a;
  a.in = in;
  a.dtype = (int)d.dtype;
  a.rows = rows;
  a.cols = cols;
  a.rs = d.row_stride ? d.row_stride : (int64_t)d.cols;
  a.bs = d.batch_stride ? d.batch_stride : (int64_t)d.rows * a.rs;
  auto vectors = [](const void* p, int64_t rs, int64_t bs, size_t es) {
    return (uintptr_t)p % 16 == 0 && (rs * es) % 16 == 0 && (bs * es) % 16 == 0;
  };
  a.vectors = vectors(in, a.rs, a.bs, dtype_size(a.dtype));
  const int64_t out_rs = d.out_row_stride ? d.out_row_stride : (int64_t)d.cols;
  const int64_t out_bs = d.out_batch_stride ? d.out_batch_stride : (int64_t)d.rows * out_rs;
  const int whole = vectors(out, out_rs, out_bs, dtype_size((int)d.out_dtype));
  if (few_ctas(d)) return launch_few(d, a, out, out_rs, out_bs, whole, st, s);
  int rc = launch(orth_norm_kernel, dim3((unsigned)l.parts, (unsigned)d.batch), kNormThreads, 0, 1, s, a, l.part);
  if (rc) return rc;
  const uint64_t groups = (d.cols + 7) / 8 * d.rows, blocks = (groups + kNormThreads - 1) / kNormThreads;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)d.batch);
  rc = launch(orth_split_kernel, grid, kNormThreads, 0, 1, s, a, scaling_of(d),
              (const double*)l.part, l.parts, l.x[0], l.factors, d.steps ? (void*)nullptr : out,
              (int)d.out_dtype, out_rs, out_bs);
  if (rc) return rc;
  if (!d.steps) return DCF_OK;

  if (!encoder()) return DCF_EUNSUPPORTED;
  CUtensorMap mx[2], ma, mb;
  if (!encode(&mx[0], l.x[0], cols, d.batch) || !encode(&ma, l.a, m, d.batch) || !encode(&mb, l.b, m, d.batch) ||
      (d.steps > 1 && !encode(&mx[1], l.x[1], cols, d.batch)))
    return DCF_ECUDA;
  for (uint32_t i = 0; i < d.steps; i++) {
    const CUtensorMap& x = mx[i & 1];
    GemmArgs g = {};
    g.st = st;
    g.sum = sums_of(d, m, false);
    g.part = l.sums;
    g.m = g.n = m;
    g.k = n;
    g.factors = l.factors + i;
    g.steps = (int)d.steps;
    g.to = l.a;
    rc = tall ? gemm_symmetric<GRAM, true>(x, g, l.gram, d.batch, s) : gemm_symmetric<GRAM, false>(x, g, l.gram, d.batch, s);
    if (rc) return rc;
    g.k = m;
    g.from = l.a;
    g.to = l.b;
    g.sum = sums_of(d, m, true);
    if ((rc = gemm_symmetric<POLY, false>(ma, g, l.poly, d.batch, s))) return rc;
    g.sum = sums_of(d, m, false);
    g.m = rows;
    g.n = cols;
    if (i + 1 < d.steps) {
      g.to = l.x[(i + 1) & 1];
      rc = tall ? gemm<APPLY, false, false>(x, mb, g, d.batch, s) : gemm<APPLY, false, true>(mb, x, g, d.batch, s);
    } else {
      g.out = out;
      g.out_dtype = (int)d.out_dtype;
      g.vectors = whole;
      g.out_rs = out_rs;
      g.out_bs = out_bs;
      rc = tall ? gemm<FINAL, false, false>(x, mb, g, d.batch, s) : gemm<FINAL, false, true>(mb, x, g, d.batch, s);
    }
    if (rc) return rc;
  }
  return DCF_OK;
}

}  // namespace dcf
