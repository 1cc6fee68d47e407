// dcf_checkpoint.cu — the gradient of a weight from a checkpoint of its
// layer's input:
//   out[c][k] = sum over runs r of scale[r][k] * (sum over t in r of grad[t][c] * q[t][k])
// A whole number of 8 bits is exact in f16 and bf16, so the tensor cores
// multiply it by the gradient as it is, and the products are exact in f32.  A
// run's scale comes after its sum: TMEM sums the 128 tokens of a run, and
// registers multiply that by the scale and add it, rounding to nearest.  (The
// tensor core truncates as it accumulates; longer sums in TMEM would be further
// from 64 bits than fp32 products are.)
//
// Whole numbers become 16-bit values in a pass of their own (three bytes of
// memory each, two of them in the workspace: 20 us of 8192 x 4096).  Made on their way into each
// tile instead, by eight warps between the copy and the product, the gradient of 4096
// channels took 270 us against 220 (bursts): every tile makes them again, and copying,
// reading and writing them in shared memory takes a quarter of what its banks
// move, which the operands of the products need.
//
// What bounds it: at 8192 x 4096 x 4096 the products take 340000 cycles of which
// the tensor cores are active in 68 %; 256 tiles on 74 pairs of CTAs are 3.5 rounds of work
// in 4.  With the 16-bit values 210 us in a burst, 240 us in a long run at the power
// limit (SM at 1.65 GHz; 278 us with inputs that change).
// Registers that spilt in the one thread that issues products cost more than
// anything else measured here (317 us): it waits for each, and the tensor core
// has no more than two products in hand.
#include "dcf_quant.cuh"

namespace dcf {

namespace {

constexpr int kSide = 128;                // k of a CTA
constexpr int kTileM = 2 * kSide;         // of a pair
constexpr int kOutWarps = 8;
constexpr int kGemmThreads = 128 + 32 * kOutWarps;  // warp 0 loads, warp 1 multiplies, 2 and 3 lend their registers
constexpr int kPairs = 74;                // of SMs on a B200; any number runs the persistent grid

// A stage is a run: 128 tokens of 128 k and of TN / 2 channels in two bytes each, in
// blocks of 64 that have a 128-byte row for each token.
constexpr int kBlockBytes = kRun * 128;
template <int TN> constexpr int kStage = (kSide + TN / 2) * kRun * 2;
template <int TN> constexpr int kStages = TN == 256 ? 3 : 4;
template <int TN> constexpr int kSmem = kStages<TN> * kStage<TN> + 256 + 1024;

struct GradArgs {
  const float* scale;
  void* out;
  int out_dtype, add;
  int pairs;               // two neighbours of a row of a 16-bit result make an aligned word
  int vectors;             // four neighbours of a row make an aligned vector
  int channels, depth;
  int skip;                // columns of the gradient's map before its first channel
  int64_t os;
  int runs, tiles_m;       // tiles along k
  int splits, split_runs;  // parts of the runs, runs of each
  int total;               // tiles times splits
  float* part;             // sums of the parts, where there is more than one
  uint32_t idesc;
  dcf_status* st;
};

// The low half of an operand's descriptor, whose memory runs along it: blocks of 64
// lie kBlockBytes apart.  The high half says that groups of eight tokens lie
// 1024 bytes apart, and the 128-byte swizzle.  (In halves because the thread that issues
// has few registers, and waits for none.)
__device__ __forceinline__ uint32_t block_desc(uint32_t addr) {
  return ((addr >> 4) & 0x3FFF) | (uint32_t)(kBlockBytes >> 4) << 16;
}
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);

__device__ __forceinline__ void pair_mma_low(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// Two of a word's signed bytes (the low ones of its halves) in a 16-bit type.
template <class T> __device__ __forceinline__ uint32_t to_halves(uint32_t h) {
  if constexpr (std::is_same<T, __half>::value) {
    // a byte, its sign turned, under the exponent of 1024: 1024 + 128 + q
    const uint32_t m = (h ^ 0x00800080u) | 0x64006400u, c = 0x64806480u;
    const __half2 r = __hsub2(*(const __half2*)&m, *(const __half2*)&c);
    return *(const uint32_t*)&r;
  } else {
    // seven bits under the exponent of 128, less 128 or, beside the sign, 256
    const uint32_t m = (h & 0x007F007Fu) | 0x43004300u, c = (h & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&m, *(const __nv_bfloat162*)&c);
    return *(const uint32_t*)&r;
  }
}

template <class T> __device__ __forceinline__ uint4 to_eight(uint32_t a, uint32_t b) {
  return make_uint4(to_halves<T>(__byte_perm(a, 0, 0x4140)), to_halves<T>(__byte_perm(a, 0, 0x4342)),
                    to_halves<T>(__byte_perm(b, 0, 0x4140)), to_halves<T>(__byte_perm(b, 0, 0x4342)));
}

__device__ __forceinline__ void put(const GradArgs& g, int64_t c, int64_t k, float v) {
  const int64_t at = c * g.os + k;
  if (g.out_dtype == DCF_F32) ((float*)g.out)[at] = g.add ? __fadd_rn(((float*)g.out)[at], v) : v;
  else if (g.out_dtype == DCF_F16) ((__half*)g.out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)g.out)[at] = __float2bfloat16_rn(v);
}

// 16 columns (channels from c0 on) of 32 k, a k in each lane.
__device__ __forceinline__ void write_block(const GradArgs& g, const float* v, int c0, int k) {
  if (g.out_dtype == DCF_F32) {
    if (k >= g.depth) return;
    float* out = (float*)g.out + (int64_t)c0 * g.os + k;
    float old[16];
#pragma unroll
    for (int j = 0; j < 16; j++) old[j] = g.add && c0 + j >= 0 && c0 + j < g.channels ? out[j * g.os] : 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++, out += g.os)
      if (c0 + j >= 0 && c0 + j < g.channels) *out = g.add ? __fadd_rn(old[j], v[j]) : v[j];
  } else if (g.pairs) {
    // Lanes trade: an even one writes its channel for two k, an odd one the next channel.
    const int odd = threadIdx.x & 1;
    uint16_t* out = (uint16_t*)g.out + (int64_t)(c0 + odd) * g.os + (k & ~1);
    const bool both = (k | 1) < g.depth, one = (k & ~1) < g.depth, half = g.out_dtype == DCF_F16;
#pragma unroll
    for (int j = 0; j < 16; j += 2, out += 2 * g.os) {
      const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1);
      const float lo = odd ? got : v[j], hi = odd ? v[j + 1] : got;
      uint32_t w;
      if (half) {
        const __half2 h = __floats2half2_rn(lo, hi);
        w = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        w = *(const uint32_t*)&h;
      }
      const int c = c0 + j + odd;
      if (c >= 0 && c < g.channels) {
        if (both) *(uint32_t*)out = w;
        else if (one) *out = (uint16_t)w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (c0 + j >= 0 && c0 + j < g.channels && k < g.depth) put(g, c0 + j, k, v[j]);
  }
}

// Sums of a part: [column of the tile][k of the tile].
template <int TN> __device__ __forceinline__ float* part_of(const GradArgs& g, int item) {
  return g.part + (int64_t)item * (kTileM * TN);
}

// D = q^T grad of each run in tiles of 256 k x TN channels by persistent pairs
// of CTAs, each with 128 k and half of the channels.  Warp 0 loads; one thread
// of the first CTA issues the eight products of a run for both; eight warps
// take a run's sums out of one of two buffers of TMEM while the other is
// filled.  k lies in the lanes: a lane needs one scale a run, and a warp writes
// neighbours of a row.
template <int TN>
__global__ void __launch_bounds__(kGemmThreads, 1) grad_kernel(const __grid_constant__ CUtensorMap map_q,
                                                               const __grid_constant__ CUtensorMap map_g,
                                                               const GradArgs args) {
  const GradArgs g = args;  // a reference to the parameter itself would be read through memory
  constexpr int S = kStages<TN>, kMine = TN / 2;  // columns of one out warp
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + (-smem_addr(smem_raw) & 1023);
  uint64_t* full = (uint64_t*)(base + S * kStage<TN>);  // the first CTA's counts what both have
  uint64_t* empty = full + S;
  uint64_t* sum_full = empty + S;
  uint64_t* sum_empty = sum_full + 2;  // the first CTA's
  uint32_t* tmem_at = (uint32_t*)(sum_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int first = (int)(blockIdx.x / 2), step = (int)(gridDim.x / 2);
  const uint32_t stage0 = smem_addr(base);
  uint32_t full0;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(full0) : "r"(smem_addr(full)));
  auto begin_of = [&](int t) { return t % g.splits * g.split_runs; };
  auto count_of = [&](int t) { return min(g.split_runs, g.runs - begin_of(t)); };

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < S; s++) {
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
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_at)), "r"(2 * TN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *(volatile uint32_t*)tmem_at;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_g) : "memory");
  }
  pdl_begin();

  bool fail = false;
  if (warp < 4) shrink_registers();
  if (warp == 0) {
    if (lane == 0) {
      Ring<S> at;
      int used = 0;  // stages filled, S at most
      for (int t = first; t < g.total && !fail; t += step) {
        const int tile = t / g.splits;
        const int row = (tile % g.tiles_m) * kTileM + (int)rank * kSide;
        const int col = tile / g.tiles_m * TN + (int)rank * (TN / 2);
        const int r0 = begin_of(t), count = count_of(t);
        for (int r = 0; r < count; r++, at.next()) {
          if (!mbar_wait_parked(&empty[at.s], at.turn ^ 1)) {
            fail = true;
            break;
          }
          const uint32_t to = stage0 + at.s * kStage<TN>, bar = full0 + at.s * 8;
          const int token = (r0 + r) * kRun;
          if (!rank) mbar_expect_tx(&full[at.s], 2 * kStage<TN>);
          pair_load_2d(to, &map_q, row, token, bar);
          pair_load_2d(to + kBlockBytes, &map_q, row + 64, token, bar);
          pair_load_2d(to + 2 * kBlockBytes, &map_g, col, token, bar);
          if (TN == 256) pair_load_2d(to + 3 * kBlockBytes, &map_g, col + 64, token, bar);
          used += used < S;
        }
      }
      // Leave only with no copy of ours and no arrival for us left in flight.
      for (; used > 0; used--) {
        const Ring<S> last = at.back(used);
        if (!rank && !mbar_wait_parked(&full[last.s], last.turn)) fail = true;
        if (!fail && !mbar_wait_parked(&empty[last.s], last.turn)) fail = true;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && !rank) {
      // The tensor core has one or two products in hand at most, so a look at a barrier after the last one (160
      // cycles) leaves it without: whether the next run is there is asked before this one's last products.
      const uint32_t desc = block_desc(stage0);
      Ring<S> at;
      Ring<2> sum;
      int left = 0;  // runs of this pair
      for (int t = first; t < g.total; t += step) left += count_of(t);
      bool room = false, there = false;
      for (; left > 0; left--) {
        if ((!room && !pair_wait_parked(&sum_empty[sum.s], sum.turn ^ 1)) || (!there && !mbar_wait_parked(&full[at.s], at.turn))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t pq = desc + (uint32_t)(at.s * (kStage<TN> >> 4)), pg = pq + (kSide * kRun * 2 >> 4);
        uint64_t* const done = &empty[at.s];
        uint64_t* const summed = &sum_full[sum.s];
        const uint32_t to = tmem + sum.s * TN;
        at.next();
        sum.next();
#pragma unroll
        for (int j = 0; j < kRun / 16; j++) {
          pair_mma_low(to, pq + j * (2048 >> 4), pg + j * (2048 >> 4), g.idesc, j);
          if (j == 3) room = pair_test(&sum_empty[sum.s], sum.turn ^ 1);
          if (j == 5) there = mbar_test(&full[at.s], at.turn);
        }
        pair_commit(summed);
        pair_commit(done);
      }
    }
  } else if (warp >= 4) {
    grow_registers();
    const int part = warp & 3;               // the 32 TMEM lanes this warp may read
    const int col = (warp - 4) / 4 * kMine;  // and the half of the columns it takes
    const uint32_t lanes = tmem + ((uint32_t)(part * 32) << 16) + col;
    Ring<2> sum;
    for (int t = first; t < g.total && !fail; t += step) {
      const int tile = t / g.splits;
      const int row = (int)rank * kSide + part * 32 + lane;  // of the tile
      const int k = tile % g.tiles_m * kTileM + row, c0 = tile / g.tiles_m * TN + col - g.skip;
      const int r0 = begin_of(t), count = count_of(t);
      const float* scale = g.scale + (int64_t)r0 * g.depth + k;
      float s = k < g.depth ? *scale : 0.0f;
      uint64_t acc[kMine / 2];  // two columns each
#pragma unroll
      for (int j = 0; j < kMine / 2; j++) acc[j] = 0;
      for (int r = 0; r < count; r++, sum.next()) {
        scale += g.depth;
        const float then = k < g.depth && r + 1 < count ? *scale : 0.0f;
        if (__any_sync(0xFFFFFFFFu, !mbar_wait_parked(&sum_full[sum.s], sum.turn))) {
          fail = true;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t x[2][16];  // one part is added while the next arrives
        tmem_load16(lanes + sum.s * TN, x[0]);
#pragma unroll
        for (int c = 0; c < kMine; c += 16) {
          uint32_t(&y)[16] = x[c / 16 & 1];
          tmem_wait(y);
          if (c + 16 < kMine) {
            tmem_load16(lanes + sum.s * TN + c + 16, x[(c / 16 + 1) & 1]);
          } else {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) arrive_first<false>(&sum_empty[sum.s]);
          }
#pragma unroll
          for (int j = 0; j < 16; j += 2)
            acc[(c + j) / 2] = fma2(two(s, s), two(__uint_as_float(y[j]), __uint_as_float(y[j + 1])), acc[(c + j) / 2]);
        }
        s = then;
      }
      if (fail) break;
      // The products wait while a tile is written, so the usual ways out are straight: sums of parts, and whole
      // tiles (17000 cycles a tile by the general way below).
      const bool inside = c0 >= 0 && c0 + kMine <= g.channels && k - lane + 32 <= g.depth;
      if (g.splits > 1) {
        float* p = part_of<TN>(g, t) + (int64_t)col * kTileM + row;
#pragma unroll
        for (int j = 0; j < kMine / 2; j++) {
          const float2 f = apart(acc[j]);
          p[2 * j * kTileM] = f.x;
          p[(2 * j + 1) * kTileM] = f.y;
        }
        continue;
      }
      if (inside && g.out_dtype == DCF_F32) {
        float* p = (float*)g.out + (int64_t)c0 * g.os + k;
        if (g.add) {
#pragma unroll
          for (int c = 0; c < kMine; c += 16) {  // what is there is read sixteen at a time
            float old[16];
#pragma unroll
            for (int j = 0; j < 16; j++) old[j] = p[j * g.os];
#pragma unroll
            for (int j = 0; j < 16; j += 2, p += 2 * g.os) {
              const float2 f = apart(acc[(c + j) / 2]);
              p[0] = __fadd_rn(old[j], f.x);
              p[g.os] = __fadd_rn(old[j + 1], f.y);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kMine / 2; j++, p += 2 * g.os) {
            const float2 f = apart(acc[j]);
            p[0] = f.x;
            p[g.os] = f.y;
          }
        }
        continue;
      }
      if (inside && g.pairs) {
        // As in write_block, every lane with both of its k.
        const int odd = lane & 1;
        uint16_t* p = (uint16_t*)g.out + (int64_t)(c0 + odd) * g.os + (k & ~1);
        auto each = [&](auto cast) {
#pragma unroll
          for (int j = 0; j < kMine / 2; j++, p += 2 * g.os) {
            const float2 f = apart(acc[j]);
            const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? f.x : f.y, 1);
            const auto h = cast(odd ? got : f.x, odd ? f.y : got);
            *(uint32_t*)p = *(const uint32_t*)&h;
          }
        };
        if (g.out_dtype == DCF_F16) each([](float a, float b) { return __floats2half2_rn(a, b); });
        else each([](float a, float b) { return __floats2bfloat162_rn(a, b); });
        continue;
      }
#pragma unroll 1
      for (int c = 0; c < kMine; c += 16) {
        if (c0 + c < g.channels) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 f = apart(acc[j / 2]);
            v[j] = f.x, v[j + 1] = f.y;
          }
          write_block(g, v, c0 + c, k);
        }
#pragma unroll
        for (int j = 0; j < kMine / 2 - 8; j++) acc[j] = acc[j + 8];
      }
    }
  }
  if (fail) atomicExch(&g.st->error, 1u);
  __syncthreads();
  pair_sync();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TN) : "memory");
  }
}

// Joins the parts of each sum, always in the same order; a thread takes four
// neighbouring k of a channel, a block 512.  Also what writes the gradient of no tokens, whose
// sums have no parts.
constexpr int kJoinThreads = 128;
__global__ void __launch_bounds__(kJoinThreads) grad_join_kernel(const __grid_constant__ GradArgs g, int tile_n) {
  pdl_begin();
  const int across = (g.depth + 4 * kJoinThreads - 1) / (4 * kJoinThreads);
  const int64_t all = (int64_t)across * g.channels;
  for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const int c = (int)(i / across), k = ((int)(i - (int64_t)c * across) * kJoinThreads + (int)threadIdx.x) * 4;
    if (k >= g.depth) continue;
    float4 sum = make_float4(0, 0, 0, 0);
    if (g.splits) {
      const int col = c + g.skip, tile = col / tile_n * g.tiles_m + k / kTileM;
      const int64_t size = (int64_t)kTileM * tile_n;
      const float* p = g.part + tile * g.splits * size + (int64_t)(col % tile_n) * kTileM + k % kTileM;
#pragma unroll 4
      for (int s = 0; s < g.splits; s++, p += size) {
        const float4 v = *(const float4*)p;
        sum = make_float4(__fadd_rn(sum.x, v.x), __fadd_rn(sum.y, v.y), __fadd_rn(sum.z, v.z), __fadd_rn(sum.w, v.w));
      }
    }
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
    if (g.vectors && k + 4 <= g.depth && !g.add) {
      const int64_t at = (int64_t)c * g.os + k;
      if (g.out_dtype == DCF_F32) {
        *(float4*)((float*)g.out + at) = sum;
      } else if (g.out_dtype == DCF_F16) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *(uint2*)((__half*)g.out + at) = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
      } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *(uint2*)((__nv_bfloat16*)g.out + at) = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (k + e < g.depth) put(g, c, k + e, v[e]);
    }
  }
}

// What the products read, in rows of whole vectors: whole numbers as values of T, and, in a second row of
// blocks, a gradient whose rows no tensor map describes.  A thread makes sixteen values, or copies sixteen
// bytes; 2^wide threads take a row.
constexpr int kOperandThreads = 256;
struct Rows {
  const uint8_t* from;
  int64_t stride, bytes;  // in bytes
  uint8_t* to;
  int64_t to_stride;
  int wide;
};
template <class T>
__global__ void __launch_bounds__(kOperandThreads) operands_kernel(const __grid_constant__ Rows levels,
                                                                   const __grid_constant__ Rows grad, int64_t rows) {
  pdl_begin();
  const bool copy = blockIdx.y;
  const int64_t stride = copy ? grad.stride : levels.stride, bytes = copy ? grad.bytes : levels.bytes;
  const int64_t to_stride = copy ? grad.to_stride : levels.to_stride;
  const uint8_t* from = copy ? grad.from : levels.from;
  uint8_t* to = copy ? grad.to : levels.to;
  const int wide = copy ? grad.wide : levels.wide, first = threadIdx.x & ((1 << wide) - 1);
  const int64_t step = (int64_t)gridDim.x * (kOperandThreads >> wide);
  for (int64_t r = (int64_t)blockIdx.x * (kOperandThreads >> wide) + (threadIdx.x >> wide); r < rows; r += step) {
    const uint8_t* row = from + r * stride;
    for (int64_t c = (int64_t)first * 16; c < bytes; c += (int64_t)16 << wide) {
      const uint4 v = row_bytes(row, c, bytes);
      if (copy) {
        *(uint4*)(to + r * to_stride + c) = v;
      } else {
        uint4* out = (uint4*)(to + r * to_stride + 2 * c);
        out[0] = to_eight<T>(v.x, v.y);
        out[1] = to_eight<T>(v.z, v.w);
      }
    }
  }
}

// ---------------------------------------------------------------- host

// An operand as boxes of 64 columns x 128 tokens.
bool encode_operand(CUtensorMap* map, const void* p, bool bf16, int64_t cols, int64_t tokens, int64_t stride) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)tokens};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t boxes[2] = {64, kRun};
  const cuuint32_t estr[2] = {1, 1};
  return encoder()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)p, dims,
                   strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t stride_of(int64_t given, uint64_t cols) { return given ? given : (int64_t)cols; }

// How a gradient is laid out: channels of a tile, and the parts into which its
// runs are cut.
struct Cut {
  int tile_n;
  int64_t tiles_m, tiles;
  int splits, runs;        // runs of a part
};

// In units of a run of a 256 x 256 tile (0.6 us): every round of tiles costs its runs (those of a 256 x 128 tile 0.65
// each: shared memory bounds it) and some five to start and to write; parts cost six more to join.  (8192 x 512 x 512:
// 20.7 us with 256 channels a tile, 17.2 us with 128; 8192 x 1024 x 4096: 71 and 96 us.)
Cut cut_of(const dcf_checkpoint_desc& d, int skip) {
  const int runs = (int)((d.tokens + kRun - 1) / kRun);
  Cut best = {};
  double least = 1e300;
  for (int tn : {128, 256}) {
    const int64_t tm = ((int64_t)d.depth + kTileM - 1) / kTileM;
    const int64_t tiles = tm * (((int64_t)d.channels + skip + tn - 1) / tn);
    const double run = tn == 256 ? 1 : 0.65;
    for (int s = 1; s == 1 || (s <= runs && tiles * s <= kPairs); s++) {
      const int each = (runs + s - 1) / s, parts = each ? (runs + each - 1) / each : 1;
      const double rounds = (double)((tiles * parts + kPairs - 1) / kPairs);
      const double cost = rounds * (each + 5) * run + (parts > 1 ? 6 : 0);
      if (cost < least) {
        least = cost;
        best = {tn, tm, tiles, parts, each};
      }
    }
  }
  return best;
}

// The workspace: whole numbers as 16-bit values, a copy of a gradient whose stride no tensor map takes,
// and the parts of sums.
struct Layout {
  Cut cut;
  bool copy;
  int64_t stride, level_stride;  // of the copies, in elements
  size_t levels, grad, part, bytes;
};

Layout layout_of(const dcf_checkpoint_desc& d, int skip) {
  Layout l = {};
  auto take = [&](size_t bytes) {
    const size_t at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  l.cut = cut_of(d, skip);
  const int64_t gs = stride_of(d.grad_row_stride, d.channels);
  l.copy = d.tokens > 1 && (gs % 8 || gs < (int64_t)d.channels || gs >= 1ll << 38);
  l.stride = (int64_t)((d.channels + 7) / 8 * 8);
  l.level_stride = (int64_t)((d.depth + 15) / 16 * 16);
  l.levels = take((size_t)d.tokens * l.level_stride * 2);
  l.grad = take(l.copy ? (size_t)d.tokens * l.stride * 2 : 0);
  l.part = take(l.cut.splits > 1 ? (size_t)l.cut.tiles * l.cut.splits * kTileM * l.cut.tile_n * 4 : 0);
  return l;
}

template <int TN> int run(const CUtensorMap& map_q, const CUtensorMap& map_g, const GradArgs& g, cudaStream_t s) {
  if (!prepare_smem((const void*)grad_kernel<TN>, kSmem<TN>)) return DCF_ECUDA;
  const unsigned pairs = (unsigned)(g.total < kPairs ? g.total : kPairs);
  return launch(grad_kernel<TN>, dim3(2 * pairs), kGemmThreads, kSmem<TN>, 2, s, map_q, map_g, g);
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
  if ((d->channels / 128 + 2) * (d->depth / kTileM + 1) >= 1ull << 30) return bad("checkpoint grad: too many tiles");
  return DCF_OK;
}

size_t checkpoint_workspace(const dcf_checkpoint_desc& d) {
  if (!d.tokens || !d.channels || !d.depth) return 0;
  // The gradient may start 0 to 7 elements into a vector: as many tiles as with none, or as with seven.
  const Layout none = layout_of(d, 0), most = layout_of(d, 7);
  return none.copy || none.bytes > most.bytes ? none.bytes : most.bytes;
}

int launch_checkpoint_grad(const dcf_checkpoint_desc& d, const void* grad, const int8_t* q, const float* scale,
                           void* out, void* ws, dcf_status* st, cudaStream_t s) {
  GradArgs g = {};
  g.scale = scale;
  g.out = out;
  g.out_dtype = (int)d.out_dtype;
  g.add = (d.flags & DCF_CHECKPOINT_ACCUMULATE) != 0;
  g.channels = (int)d.channels;
  g.depth = (int)d.depth;
  g.os = stride_of(d.out_row_stride, d.depth);
  g.pairs = (uintptr_t)out % 4 == 0 && (d.channels == 1 || g.os % 2 == 0);
  const int four = 4 * (int)dtype_size(g.out_dtype);
  g.vectors = (uintptr_t)out % four == 0 && (d.channels == 1 || g.os % 4 == 0);
  g.st = st;
  int tile_n = 0;
  if (d.tokens) {
    Layout l = layout_of(d, 0);
    int64_t gs = d.tokens > 1 ? stride_of(d.grad_row_stride, d.channels) : l.stride + 8;
    int rc;
    auto rows_of = [](const void* from, int64_t stride, int64_t bytes, void* to, int64_t to_stride) {
      Rows r = {(const uint8_t*)from, stride, bytes, (uint8_t*)to, to_stride, 0};
      while (r.wide < 8 && (16ll << r.wide) < bytes) r.wide++;
      return r;
    };
    const Rows copy = rows_of(grad, gs * 2, (int64_t)d.channels * 2, (uint8_t*)ws + l.grad, l.stride * 2);
    const bool copied = l.copy;
    if (copied) {
      grad = copy.to;
      gs = l.stride;
    }
    // A map starts on a 16-byte boundary; the columns before the first channel are left out again.
    g.skip = (int)((uintptr_t)grad % 16 / 2);
    if (g.skip) l = layout_of(d, g.skip);
    const bool bf16 = d.grad_dtype == DCF_BF16;
    if (!encoder()) return DCF_EUNSUPPORTED;
    const int64_t rows = (int64_t)d.tokens, cols = (int64_t)d.depth;
    const Rows levels = rows_of(q, stride_of(d.q_row_stride, d.depth), cols, (uint8_t*)ws + l.levels, l.level_stride * 2);
    const int across = kOperandThreads >> (copied && copy.wide > levels.wide ? copy.wide : levels.wide);
    const int64_t blocks = (rows + across - 1) / across;
    const dim3 grid((unsigned)(blocks < (1 << 30) ? blocks : 1 << 30), copied ? 2 : 1);
    rc = bf16 ? launch(operands_kernel<__nv_bfloat16>, grid, kOperandThreads, 0, 1, s, levels, copy, rows)
              : launch(operands_kernel<__half>, grid, kOperandThreads, 0, 1, s, levels, copy, rows);
    if (rc) return rc;
    CUtensorMap map_q, map_g;
    tile_n = l.cut.tile_n;
    if (!encode_operand(&map_q, levels.to, bf16, cols, rows, l.level_stride) ||
        !encode_operand(&map_g, (const uint8_t*)grad - g.skip * 2, bf16, (int64_t)d.channels + g.skip, rows, gs))
      return DCF_ECUDA;
    g.runs = (int)((d.tokens + kRun - 1) / kRun);
    g.tiles_m = (int)l.cut.tiles_m;
    g.splits = l.cut.splits;
    g.split_runs = l.cut.runs;
    g.total = (int)(l.cut.tiles * l.cut.splits);
    g.part = (float*)((uint8_t*)ws + l.part);
    g.idesc = (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 15) | (1u << 16) | ((uint32_t)(tile_n >> 3) << 17) |
              ((uint32_t)(kTileM >> 4) << 24);
    rc = tile_n == 256 ? run<256>(map_q, map_g, g, s) : run<128>(map_q, map_g, g, s);
    if (rc || g.splits == 1) return rc;
  }
  const int64_t joins = ((int64_t)d.depth + 4 * kJoinThreads - 1) / (4 * kJoinThreads) * (int64_t)d.channels;
  return launch(grad_join_kernel, dim3((unsigned)(joins < (1 << 30) ? joins : 1 << 30)), kJoinThreads, 0, 1, s, g,
                tile_n ? tile_n : 1);
}

}  // namespace dcf
