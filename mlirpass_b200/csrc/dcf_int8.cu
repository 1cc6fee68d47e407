// dcf_int8.cu — the product of 8-bit matrices with scales for each token and
// channel:
//   out[t][c] = (sum over k of a[t][k] * b[c][k]) * a_scale[t] * b_scale[c] + bias[c]
// Sums of whole numbers are exact in 32 bits (2^14 * 131071 < 2^31), in any
// order, so a sum is split and joined wherever that helps.
//
// Three ways, by what bounds them:
//   up to four tokens       the weight's bytes: int8_few_kernel, on the CUDA cores (one bf16 token, 4096 x 4096 in
//                           L2: 4.6 us, 2.6 us of bytes at HBM's rate; 16384 x 8192: 30 us, 20.5 us of bytes)
//   some tens of tokens     the weight's bytes: int8_gemm_kernel with tiles of 64 tokens, the depth cut in parts
//                           where channels are few (48 x 16384 x 4096: 17 us, 10.5 us of bytes)
//   more                    the tensor cores: tiles of 128 and 256 tokens (bursts of thirty, and long runs at the
//                           power limit: 8192 x 8192 x 8192 365 and 454 us, the SM at 1.1 GHz, 328 us at twice the
//                           measured bf16 burst rate; 4096 x 4096 x 4096 48 and 54 us at 1.57 GHz, 41 us at that
//                           rate: 256 tiles on 74 pairs of CTAs are 3.5 rounds of work in 4)
#include "dcf_quant.cuh"

namespace dcf {

namespace {

constexpr int kSide = 128;                // channels of a CTA
constexpr int kTileM = 2 * kSide;         // of a pair
constexpr int kAtom = 128;                // k of a 128-byte swizzle row
template <bool READ> constexpr int kOutWarps = READ ? 8 : 16;  // warps that write results
template <bool READ> constexpr int kGemmThreads = 128 + 32 * kOutWarps<READ>;  // warp 0 loads, warp 1 multiplies
constexpr int kReaders = 256;             // threads that read a weight's rows where no tensor map describes them
constexpr int kPairs = 74;                // of SMs on a B200; any number runs the persistent grid

// What becomes of sums.
struct Result {
  const float* a_scale;  // null: the sums themselves
  const float* b_scale;
  const float* bias;
  void* out;
  int out_dtype;
  int pairs;             // two neighbours of a row of a 16-bit result make an aligned word
  int tokens, channels;
  int64_t stride;
};

// The result of one token and channel; a bias of -0 adds nothing to any value.
__device__ __forceinline__ void put(const Result& g, int64_t t, int64_t c, int sum, float a_scale, float b_scale,
                                    float bias) {
  const int64_t at = t * g.stride + c;
  if (g.out_dtype == DCF_I32) {
    ((int*)g.out)[at] = sum;
    return;
  }
  const float v = __fadd_rn(__fmul_rn(__fmul_rn((float)sum, a_scale), b_scale), bias);
  if (g.out_dtype == DCF_F32) ((float*)g.out)[at] = v;
  else if (g.out_dtype == DCF_F16) ((__half*)g.out)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)g.out)[at] = __float2bfloat16_rn(v);
}

// ------------------------------------------------- tensor-core product

// k of a stage: two swizzle rows, so that half as many waits come between the
// products and memory is read 256 bytes of a row at a time; one where threads read the weight.
template <bool READ> constexpr int kAtoms = READ ? 1 : 2;
template <bool READ> constexpr int kBK = kAtoms<READ> * kAtom;
template <int TN, bool READ> constexpr int kStage = (kSide + TN / 2) * kBK<READ>;
template <int TN, bool READ> constexpr int kStages = (TN == 256 ? 6 : TN == 128 ? 8 : 10) / kAtoms<READ>;
template <int TN, bool READ> constexpr int kGemmSmem = kStages<TN, READ> * kStage<TN, READ> + 4 * TN * 4 + 512 + 1024;

struct GemmArgs {
  Result to;
  int blocks;              // stages along the whole depth
  int tiles_m;             // tiles along the channels
  int splits, split_k;     // parts of the depth, stages of each
  int64_t total;           // tiles times splits
  int* part;               // sums of the parts, where there is more than one
  const int8_t* b;         // the weight, where threads read it
  int64_t b_stride;
  int whole;               // rows whose last vector lies in the weight's memory
  int depth;
  int early;               // only the kernel that quantised the tokens ran since the weight may have changed
  dcf_status* st;
};

__device__ __forceinline__ void pair_mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Rows of 128 bytes with the 128-byte swizzle; groups of eight lie 1024 bytes apart.
__device__ __forceinline__ uint64_t row_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// Sums of a part: [column of the tile][channel of the tile].
template <int TN> __device__ __forceinline__ int* part_of(const GemmArgs& g, int64_t item) {
  return g.part + item * (kTileM * TN);
}

// kBlock columns (tokens from t0 on) of 32 channels, a channel in each lane, on their way out.
// A tile is as good as written once, so what counts is how few instructions and
// how short a code do it (32 columns at a time by 8 warps and a predicate for
// each: 6.2 us a tile of 256 x 256).
constexpr int kBlock = 16;
template <bool WHOLE>
__device__ __forceinline__ void write_block(const Result& g, const uint32_t (&r)[kBlock], const float* scales, int64_t t0,
                                            int64_t c, uint64_t b, float bias) {
  const int there = WHOLE ? kBlock : (int)(g.tokens - t0);
  const bool mine = c < g.channels;
  const int64_t step = g.stride;
  auto values = [&](int j) {
    const float2 a = *(const float2*)&scales[j];
    const float2 v = apart(mul2(mul2(two((float)(int)r[j], (float)(int)r[j + 1]), two(a.x, a.y)), b));
    return make_float2(__fadd_rn(v.x, bias), __fadd_rn(v.y, bias));
  };
  auto each = [&](auto* out, auto cast) {
    out += t0 * step + c;
    if (!mine) return;
#pragma unroll
    for (int j = 0; j < kBlock; j += 2, out += 2 * step) {
      const auto v = cast(j);
      if (WHOLE || j < there) out[0] = v.x;
      if (WHOLE || j + 1 < there) out[step] = v.y;
    }
  };
  if (g.out_dtype == DCF_I32) {
    each((int*)g.out, [&](int j) { return make_int2((int)r[j], (int)r[j + 1]); });
  } else if (g.out_dtype == DCF_F32) {
    each((float*)g.out, values);
  } else if (g.pairs) {
    // Lanes trade: an even one writes its token for two channels, an odd one the next token.
    const int odd = threadIdx.x & 1;
    uint16_t* out = (uint16_t*)g.out + (t0 + odd) * step + (c & ~1ll);
    const bool both = (c | 1) < g.channels, one = (c & ~1ll) < g.channels;
    const bool half = g.out_dtype == DCF_F16;
#pragma unroll
    for (int j = 0; j < kBlock; j += 2, out += 2 * step) {
      const float2 v = values(j);
      const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v.x : v.y, 1);
      const float lo = odd ? got : v.x, hi = odd ? v.y : got;
      uint32_t w;
      if (half) {
        const __half2 h = __floats2half2_rn(lo, hi);
        w = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        w = *(const uint32_t*)&h;
      }
      if (WHOLE) {
        if (both) *(uint32_t*)out = w;
      } else if (j + odd < there) {
        if (both) *(uint32_t*)out = w;
        else if (one) *out = (uint16_t)w;
      }
    }
  } else if (g.out_dtype == DCF_F16) {
    each((__half*)g.out, [&](int j) { return __float22half2_rn(values(j)); });
  } else {
    each((__nv_bfloat16*)g.out, [&](int j) { return __float22bfloat162_rn(values(j)); });
  }
}

// A row's vectors may start before it, in the allocation that holds it, and hold what follows it, but for the last rows
// (all but `whole`), behind which the memory may end: the ends of these are left out at first and read by bytes before
// they are used.  Of the rows up to `whole` and `rows`, the number whose vector with `have` bytes up to the row's
// end is read at once (asked for a row's last turn only; with all of this at each load 48 x 16384 x 4095 took 43 us
// instead of 34):
__device__ __forceinline__ int read_at_once(int have, int whole, int rows) {
  return have >= 16 ? rows : have > 0 ? whole : 0;
}

__device__ __forceinline__ void last_bytes(uint4& v, const int8_t* p, int have) {
  if (have > 0 && have < 16) v = first_bytes(p, have);
}

// Sixteen bytes of a row from k on, zeros behind its end, where the row may start
// at any byte.  L neighbours in a warp read 16 L bytes of the row
// as the 16-byte vectors that hold them, and take what they lack from each other.
template <int L, bool LAST>
__device__ __forceinline__ void read_start(const int8_t* row, int k, int depth, bool there, bool whole, int lane, uint4& own,
                                           uint4& next) {
  const int8_t* p = row + k;
  const int off = (int)((uintptr_t)p & 15), have = depth - k + off;
  own = next = make_uint4(0, 0, 0, 0);
  if (LAST ? read_at_once(have, whole, there) : there) own = *(const uint4*)(p - off);
  if (off && (lane & (L - 1)) == L - 1 && (LAST ? read_at_once(have - 16, whole, there) : there))
    next = *(const uint4*)(p - off + 16);
}

template <int L>
__device__ __forceinline__ void read_last(const int8_t* row, int k, int depth, int lane, uint4& own, uint4& next) {
  const int8_t* p = row + k;
  const int off = (int)((uintptr_t)p & 15), have = depth - k + off;
  last_bytes(own, p - off, have);
  if (off && (lane & (L - 1)) == L - 1) last_bytes(next, p - off + 16, have - 16);
}

template <int L>
__device__ __forceinline__ uint4 read_end(const int8_t* row, int k, int depth, int lane, const uint4& own, uint4 next) {
  const uint4 beside = make_uint4(__shfl_down_sync(0xFFFFFFFFu, own.x, 1), __shfl_down_sync(0xFFFFFFFFu, own.y, 1),
                                  __shfl_down_sync(0xFFFFFFFFu, own.z, 1), __shfl_down_sync(0xFFFFFFFFu, own.w, 1));
  if ((lane & (L - 1)) != L - 1) next = beside;
  uint4 v = bytes_from(own, next, (int)((uintptr_t)(row + k) & 15));
  uint32_t* w = (uint32_t*)&v;
  const int have = depth - k;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int here = have - 4 * j;  // bytes of this word in the row
    if (here < 4) w[j] = here > 0 ? w[j] & (0xFFFFFFFFu >> (32 - 8 * here)) : 0u;
  }
  return v;
}

// D = B A^T in tiles of 256 channels x TN tokens by persistent pairs of CTAs:
// each loads 128 channels and half of the tokens, one instruction multiplies
// 32 k of both, and each keeps the sums of its channels in TMEM, in two
// buffers, so that a tile is written while the next is summed.  Channels lie
// in the lanes, so that a warp writes neighbours of a row.  Warp 0 keeps the
// ring of stages full; one thread of the first CTA issues the products of
// both: its barrier counts the bytes of both CTAs' loads, as each wait on
// another costs that thread 160 cycles, and four products take 512 (probe: 136
// cycles a product with one wait between four of them, 176 with two).
// READ: no tensor map describes the weight, and eight more warps read it.
template <int TN, bool READ>
__global__ void __launch_bounds__(kGemmThreads<READ> + (READ ? kReaders : 0), 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                     const GemmArgs args) {
  const GemmArgs g = args;  // a reference to the parameter itself would be read through memory
  constexpr int OW = kOutWarps<READ>, kMine = TN / (OW / 4);  // columns of one out warp
  constexpr int S = kStages<TN, READ>, BK = kBK<READ>, kSize = kStage<TN, READ>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = smem_raw + (-smem_addr(smem_raw) & 1023);
  float* scales = (float*)(base + S * kSize);
  uint64_t* full = (uint64_t*)(scales + OW * kMine);
  uint64_t* empty = full + S;             // (the first CTA's `full` counts what both have loaded)
  uint64_t* sum_full = empty + S;
  uint64_t* sum_empty = sum_full + 2;     // the first CTA's
  uint64_t* read = sum_empty + 2;         // READ: this CTA's part of the weight is in its memory
  uint64_t* peer = read + S;              // and the second's is, the first CTA's
  uint32_t* tmem_at = (uint32_t*)(peer + S);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
  const uint32_t stage0 = smem_addr(base);
  uint32_t full0;  // the first CTA's
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(full0) : "r"(smem_addr(full)));
  auto begin_of = [&](int64_t t) { return (int)(t % g.splits) * g.split_k; };
  auto count_of = [&](int64_t t) { return min(g.split_k, g.blocks - begin_of(t)); };

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < S; s++) {
      mbar_init(&full[s], READ ? 2 : 1);
      mbar_init(&empty[s], 1);
      if (READ) mbar_init(&read[s], kReaders);
      if (READ) mbar_init(&peer[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sum_full[b], 1);
      mbar_init(&sum_empty[b], 2 * OW);
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
    if (!READ) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_b) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&map_a) : "memory");
  }
  // What reads the weight alone need not wait for the tokens.
  if (!g.early || (warp != 0 && warp < 4 + OW)) pdl_begin();

  bool fail = false;
  if (warp == 0) {
    if (lane == 0) {
      Ring<S> at;
      int used = 0;  // stages filled, S at most
      int ahead = 0; // stages whose weight is on its way
      if (g.early) {
        if (!READ && first < g.total) {
          const int row = (int)(first / g.splits % g.tiles_m) * kTileM + (int)rank * kSide;
          for (const int end = min(S, count_of(first)); ahead < end; ahead++) {
            if (!rank) mbar_expect_tx(&full[ahead], 2 * kSize);
#pragma unroll
            for (int h = 0; h < kAtoms<READ>; h++)
              pair_load_2d(stage0 + ahead * kSize + h * (kSide * kAtom), &map_b, (begin_of(first) + ahead) * BK + h * kAtom, row,
                           full0 + ahead * 8);
          }
        }
        pdl_begin();
      }
      for (int64_t t = first; t < g.total && !fail; t += step) {
        const int64_t tile = t / g.splits;
        const int row = (int)(tile % g.tiles_m) * kTileM + (int)rank * kSide;
        const int col = (int)(tile / g.tiles_m) * TN + (int)rank * (TN / 2);
        const int b0 = begin_of(t), blocks = count_of(t);
        for (int k = b0 * BK, end = (b0 + blocks) * BK; k < end; k += BK, at.next()) {
          if (!mbar_wait_parked(&empty[at.s], at.turn ^ 1)) {
            fail = true;
            break;
          }
          const uint32_t to = stage0 + at.s * kSize;
          const uint32_t bar = full0 + at.s * 8;
          if (ahead > 0) {
            ahead--;
          } else {
            if (!rank) mbar_expect_tx(&full[at.s], 2 * (READ ? TN / 2 * BK : kSize));
#pragma unroll
            for (int h = 0; h < kAtoms<READ>; h++)
              if (!READ) pair_load_2d(to + h * (kSide * kAtom), &map_b, k + h * kAtom, row, bar);
          }
#pragma unroll
          for (int h = 0; h < kAtoms<READ>; h++)
            pair_load_2d(to + kSide * BK + h * (TN / 2 * kAtom), &map_a, k + h * kAtom, col, bar);
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
      constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
      const uint64_t desc = row_desc(stage0);
      Ring<S> at;
      Ring<2> sum;
      bool there = false;
      for (int64_t t = first; t < g.total && !fail; t += step, sum.next()) {
        const int blocks = count_of(t);
        if (!pair_wait_parked(&sum_empty[sum.s], sum.turn ^ 1)) {
          fail = true;
          break;
        }
        for (int b = 0; b < blocks; b++) {
          if (!there && !mbar_wait_parked(&full[at.s], at.turn)) {
            fail = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t pb = desc + (uint64_t)(at.s * (kSize >> 4)), pa = pb + (kSide * BK >> 4);
          uint64_t* const done = &empty[at.s];
          at.next();
#pragma unroll
          for (int j = 0; j < BK / 32; j++) {
            const int h = j / 4, at32 = j % 4 * 2;  // the swizzle row, and 32 bytes in it
            pair_mma_i8(tmem + sum.s * TN, pb + h * (kSide * kAtom >> 4) + at32, pa + h * (TN / 2 * kAtom >> 4) + at32, idesc, b | j);
            if (j == BK / 32 - 3) there = mbar_test(&full[at.s], at.turn);  // before the tensor core runs out of products
          }
          pair_commit(done);
        }
        if (!fail) pair_commit(&sum_full[sum.s]);
      }
    }
  } else if (READ && warp == 2) {
    // Passes on that a stage's weight is there, so that neither the readers, who have loads on their way, nor the
    // thread that issues products spend time on the other CTA.
    if (lane == 0) {
      Ring<S> at;
      for (int64_t t = first; t < g.total && !fail; t += step)
        for (int left = count_of(t); left > 0; left--, at.next()) {
          if (!mbar_wait_parked(&read[at.s], at.turn) || (!rank && !pair_acquire(&peer[at.s], at.turn))) {
            fail = true;
            break;
          }
          if (rank) arrive_first<true>(&peer[at.s]);
          else mbar_arrive(&full[at.s]);
        }
    }
  } else if (warp >= 4 + OW) {
    const int id = threadIdx.x - kGemmThreads<READ>, chunk = id & 7;
    constexpr int kRows = kSide * 8 / kReaders;
    uint4 own[kRows], next[kRows];
    const int8_t* rows[kRows];
    bool there[kRows], whole[kRows];
    auto rows_of = [&](int64_t t) {
#pragma unroll
      for (int j = 0; j < kRows; j++) {
        const int64_t r = (t / g.splits) % g.tiles_m * kTileM + rank * kSide + id / 8 + j * (kReaders / 8);
        rows[j] = g.b + r * g.b_stride;
        there[j] = r < g.to.channels;
        whole[j] = r < g.whole;
      }
    };
    auto start = [&](int k) {
      if (k + BK + 16 <= g.depth) {
#pragma unroll
        for (int j = 0; j < kRows; j++)
          read_start<8, false>(rows[j], k + chunk * 16, g.depth, there[j], whole[j], lane, own[j], next[j]);
      } else {
#pragma unroll
        for (int j = 0; j < kRows; j++)
          read_start<8, true>(rows[j], k + chunk * 16, g.depth, there[j], whole[j], lane, own[j], next[j]);
      }
    };
    Ring<S> at;
    if (first < g.total) {
      rows_of(first);
      start(begin_of(first) * BK);
    }
    for (int64_t t = first; t < g.total && !fail; t += step) {
      const int k0 = begin_of(t) * BK, end = k0 + count_of(t) * BK;
      for (int k = k0; k < end; k += BK, at.next()) {
        uint4 v[kRows];
        if (k + BK + 16 > g.depth) {
#pragma unroll
          for (int j = 0; j < kRows; j++)
            if (there[j] && !whole[j]) read_last<8>(rows[j], k + chunk * 16, g.depth, lane, own[j], next[j]);
        }
#pragma unroll
        for (int j = 0; j < kRows; j++) v[j] = read_end<8>(rows[j], k + chunk * 16, g.depth, lane, own[j], next[j]);
        // The next stage is on its way while this one waits for room.
        if (k + BK < end) {
          start(k + BK);
        } else if (t + step < g.total) {
          rows_of(t + step);
          start(begin_of(t + step) * BK);
        }
        if (__any_sync(0xFFFFFFFFu, !mbar_wait_parked(&empty[at.s], at.turn ^ 1))) {
          fail = true;
          break;
        }
        uint8_t* to = base + at.s * kSize;
#pragma unroll
        for (int j = 0; j < kRows; j++) {
          const int r = id / 8 + j * (kReaders / 8);
          *(uint4*)(to + r * BK + ((chunk ^ (r & 7)) << 4)) = v[j];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&read[at.s]);
      }
    }
  } else if (warp >= 4) {
    const int part = warp & 3;               // the 32 TMEM lanes this warp may read
    const int col = (warp - 4) / 4 * kMine;  // and its part of the columns
    const uint32_t lanes = tmem + ((uint32_t)(part * 32) << 16) + col;
    float* mine = scales + (warp - 4) * kMine;
    Ring<2> sum;
    for (int64_t t = first; t < g.total && !fail; t += step, sum.next()) {
      const int64_t tile = t / g.splits;
      const int row = (int)rank * kSide + part * 32 + lane;  // of the tile
      const int64_t c = (tile % g.tiles_m) * kTileM + row, t0 = tile / g.tiles_m * TN + col;
      const bool whole = g.splits == 1;
      float b = 0, bias = -0.0f;  // adds nothing to any value
      if (whole && g.to.b_scale) {
        if (c < g.to.channels) {
          b = g.to.b_scale[c];
          if (g.to.bias) bias = g.to.bias[c];
        }
        __syncwarp();
        for (int j = lane; j < kMine; j += 32) mine[j] = t0 + j < g.to.tokens ? g.to.a_scale[t0 + j] : 0.0f;
        __syncwarp();
      }
      if (__any_sync(0xFFFFFFFFu, !mbar_wait_parked(&sum_full[sum.s], sum.turn))) {
        fail = true;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int j = 0; j < kMine; j += kBlock) {
        uint32_t r[kBlock];
        tmem_load16(lanes + sum.s * TN + j, r);
        tmem_wait(r);
        if (j + kBlock == kMine) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          if (lane == 0) arrive_first<false>(&sum_empty[sum.s]);
        }
        if (t0 + j >= g.to.tokens) continue;
        if (whole) {
          const uint64_t b2 = two(b, b);
          // (a block over the last channel takes the careful path when they are odd)
          if (t0 + j + kBlock <= g.to.tokens && (c - lane + 32 <= g.to.channels || !g.to.pairs))
            write_block<true>(g.to, r, mine + j, t0 + j, c, b2, bias);
          else
            write_block<false>(g.to, r, mine + j, t0 + j, c, b2, bias);
        } else {
          int* p = part_of<TN>(g, t) + (int64_t)(col + j) * kTileM + row;
#pragma unroll
          for (int k = 0; k < kBlock; k++) p[k * kTileM] = (int)r[k];
        }
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

// Joins the parts of each sum; a thread takes four neighbouring channels of a
// token, a block 512.  Also what writes the result of a depth of 0, whose sums have no parts.
constexpr int kJoinThreads = 128;
__global__ void __launch_bounds__(kJoinThreads) int8_join_kernel(const __grid_constant__ GemmArgs g, int tile_n) {
  pdl_begin();
  const int across = (g.to.channels + 4 * kJoinThreads - 1) / (4 * kJoinThreads);
  const int64_t all = (int64_t)across * g.to.tokens;
  const bool scaled = g.to.b_scale != nullptr;
  for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const int t = (int)(i / across), c = ((int)(i - (int64_t)t * across) * kJoinThreads + (int)threadIdx.x) * 4;
    if (c >= g.to.channels) continue;
    int4 sum = make_int4(0, 0, 0, 0);
    if (g.splits) {
      const int64_t size = (int64_t)kTileM * tile_n, tile = (int64_t)(t / tile_n) * g.tiles_m + c / kTileM;
      const int* p = g.part + tile * g.splits * size + (int64_t)(t % tile_n) * kTileM + c % kTileM;
#pragma unroll 4
      for (int s = 0; s < g.splits; s++, p += size) {
        const int4 v = *(const int4*)p;
        sum = make_int4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
      }
    }
    const int v[4] = {sum.x, sum.y, sum.z, sum.w};
    const float a = scaled ? g.to.a_scale[t] : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (c + e < g.to.channels)
        put(g.to, t, c + e, v[e], a, scaled ? g.to.b_scale[c + e] : 0.0f, g.to.bias ? g.to.bias[c + e] : -0.0f);
  }
}

// -------------------------------------------------------- few tokens

// Up to four tokens are bound by the weight's bytes.  A group of warps takes
// eight channels, its warps 32 vectors of 16 bytes of their rows in turn (eight
// loads in each lane, the next eight under way while these are multiplied).
// More than one warp to a group only where there are too few channels: joining
// their sums makes warps wait for each other.  The tokens are in shared memory,
// where a block quantises them itself while that is little work.  One wave of
// blocks takes all channels in turns.
//
// A weight off 16-byte boundaries is read as the vectors that hold its rows,
// and each lane makes up its sixteen bytes from its vector and its neighbour's; the last
// lane lends its vector only.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewTokens = 4, kFewChannels = 8;
constexpr int kFewResident = 2;          // blocks to an SM
template <bool READ> constexpr int kFewBytes = READ ? 31 * 16 : 32 * 16;  // of a row that a warp takes
constexpr int kFewSmem = 64 << 10;
constexpr int kFewOwn = 8192;            // values of tokens that each block quantises for itself

struct FewArgs {
  Result to;
  const void* a;
  int a_dtype, a_vectors;  // vectors: rows of the tokens start on 16-byte boundaries
  int64_t a_stride;
  const int8_t* b;
  int64_t b_stride;
  int whole;               // rows whose last vector lies in the weight's memory
  int depth, padded;       // padded: to whole turns of a warp, and a vector of zeros
  int across;              // warps along the depth
  int early;               // only the kernel that quantised the tokens ran since the weight may have changed
};

// Sixteen bytes from byte `off` of a lane's vector and the next lane's on.
__device__ __forceinline__ uint4 shifted_down(const uint4& own, int off) {
  const uint4 beside = make_uint4(__shfl_down_sync(0xFFFFFFFFu, own.x, 1), __shfl_down_sync(0xFFFFFFFFu, own.y, 1),
                                  __shfl_down_sync(0xFFFFFFFFu, own.z, 1), __shfl_down_sync(0xFFFFFFFFu, own.w, 1));
  return bytes_from(own, beside, off);
}

// Tokens as whole numbers in shared memory, zeros behind them; warps share a token.
template <class V, int E, int T>
__device__ __forceinline__ void few_quantise(const FewArgs& g, int8_t* x, float* scales, uint32_t* keys) {
  constexpr int kShare = kFewThreads / T;  // threads to a token
  const int groups = (g.depth + E - 1) / E, t = threadIdx.x / kShare, first = threadIdx.x % kShare;
  const V* in = (const V*)g.a + t * g.a_stride;
  const bool there = t < g.to.tokens;
  uint32_t key = 0;
  if (there) {
    for (int c = first; c < groups; c += kShare) {
      Group<V, E> v;
      load_group(v, in + c * E, g.depth - c * E);
      key = group_key(v, key);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = key_max<V>(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
  if (threadIdx.x % 32 == 0) keys[threadIdx.x / 32] = key;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kShare / 32; j++) key = key_max<V>(key, keys[t * (kShare / 32) + j]);
  const Scale s(key_value<V>(key));
  if (!there) return;
  if (first == 0) scales[t] = s.scale;
  for (int c = first; c < groups; c += kShare) {
    Group<V, E> v;
    load_group(v, in + c * E, g.depth - c * E);
    uint32_t w[kLevelWords<E>];
    quantise_group(v, s, w);
    store_levels<E>(x + t * g.padded + c * E, w, g.depth - c * E);
  }
}

template <int T, bool READ>
__global__ void __launch_bounds__(kFewThreads, kFewResident) int8_few_kernel(const __grid_constant__ FewArgs args) {
  const FewArgs g = args;
  constexpr int C = kFewChannels;
  extern __shared__ __align__(16) int8_t x[];
  __shared__ float scales[T];
  __shared__ uint32_t keys[kFewWarps];
  __shared__ int parts[2][kFewWarps][C * T];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = kFewWarps / g.across, start = warp % g.across * kFewBytes<READ>, turn = g.across * kFewBytes<READ>;
  const int64_t step = (int64_t)gridDim.x * groups * C;
  int64_t c0 = ((int64_t)blockIdx.x * groups + warp / g.across) * C;
  uint4 own[C];
  auto load = [&](int64_t c, int k) {
    const int have = g.depth - k - lane * 16, whole = (int)(g.whole - c), rows = (int)(g.to.channels - c);
    const int8_t* p = g.b + c * g.b_stride + k + lane * 16;
    auto each = [&](auto at_once) {
#pragma unroll
      for (int j = 0; j < C; j++, p += g.b_stride) {
        const int off = READ ? (int)((uintptr_t)p & 15) : 0;  // bytes before the row, or the end of the vector before
        own[j] = make_uint4(0, 0, 0, 0);
        if (j < at_once(off)) own[j] = *(const uint4*)(p - off);  // what else they hold meets zeros
      }
    };
    if (k + 512 <= g.depth) each([&](int) { return rows; });
    else each([&](int off) { return read_at_once(have + off, whole, rows); });
  };
  if (!g.early) pdl_begin();
  load(c0, start);
  if (g.early) pdl_begin();

  for (int i = threadIdx.x * 16; i < T * g.padded; i += kFewThreads * 16) *(uint4*)(x + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (g.a_dtype == DCF_F32) {
    g.a_vectors ? few_quantise<float, 4, T>(g, x, scales, keys) : few_quantise<float, 1, T>(g, x, scales, keys);
  } else if (g.a_dtype == DCF_F16) {
    g.a_vectors ? few_quantise<__half, 8, T>(g, x, scales, keys) : few_quantise<__half, 1, T>(g, x, scales, keys);
  } else if (g.a_dtype == DCF_BF16) {
    g.a_vectors ? few_quantise<__nv_bfloat16, 8, T>(g, x, scales, keys) : few_quantise<__nv_bfloat16, 1, T>(g, x, scales, keys);
  } else {
    for (int t = 0; t < g.to.tokens; t++) {
      const int8_t* in = (const int8_t*)g.a + t * g.a_stride;
      if (g.a_vectors) {
        for (int k = threadIdx.x * 16; k + 16 <= g.depth; k += kFewThreads * 16)
          *(uint4*)(x + t * g.padded + k) = *(const uint4*)(in + k);
        const int k = g.depth / 16 * 16 + threadIdx.x;
        if (k < g.depth) x[t * g.padded + k] = in[k];
      } else {
        for (int k = threadIdx.x; k < g.depth; k += kFewThreads) x[t * g.padded + k] = in[k];
      }
    }
    if (threadIdx.x < g.to.tokens && g.to.a_scale) scales[threadIdx.x] = g.to.a_scale[threadIdx.x];
  }
  __syncthreads();

  for (int buffer = 0; c0 < g.to.channels; c0 += step, buffer ^= 1) {
    int sum[C][T];
#pragma unroll
    for (int j = 0; j < C; j++)
#pragma unroll
      for (int t = 0; t < T; t++) sum[j][t] = 0;
    // What the result of this lane, token lane / C of channel lane % C, is multiplied by.
    const int id = lane % (C * T);
    const int64_t c = c0 + id % C;
    const bool mine = lane < C * T && c < g.to.channels && id / C < g.to.tokens;
    float b = 0, bias = -0.0f;
    if (mine && g.to.b_scale) {
      b = g.to.b_scale[c];
      if (g.to.bias) bias = g.to.bias[c];
    }
    for (int k0 = start; k0 < g.depth; k0 += turn) {
      if (c0 + C > g.whole && k0 + 512 > g.depth) {
#pragma unroll
        for (int j = 0; j < C; j++) {
          const int8_t* p = g.b + (c0 + j) * g.b_stride + k0 + lane * 16;
          const int off = READ ? (int)((uintptr_t)p & 15) : 0;
          if (c0 + j >= g.whole && c0 + j < g.to.channels) last_bytes(own[j], p - off, g.depth - k0 - lane * 16 + off);
        }
      }
      uint4 w[C];
#pragma unroll
      for (int j = 0; j < C; j++) {
        w[j] = own[j];
        if (READ) w[j] = shifted_down(w[j], (int)((uintptr_t)(g.b + (c0 + j) * g.b_stride) & 15));
      }
      const bool more = k0 + turn < g.depth;
      load(more ? c0 : c0 + step, more ? k0 + turn : start);
      const int k = READ && lane == 31 ? g.padded - 16 : k0 + lane * 16;
#pragma unroll
      for (int t = 0; t < T; t++) {
        const uint4 v = *(const uint4*)(x + t * g.padded + k);
#pragma unroll
        for (int j = 0; j < C; j++) {
          sum[j][t] = __dp4a((int)w[j].x, (int)v.x, sum[j][t]);
          sum[j][t] = __dp4a((int)w[j].y, (int)v.y, sum[j][t]);
          sum[j][t] = __dp4a((int)w[j].z, (int)v.z, sum[j][t]);
          sum[j][t] = __dp4a((int)w[j].w, (int)v.w, sum[j][t]);
        }
      }
    }
    int all = 0;
#pragma unroll
    for (int j = 0; j < C; j++)
#pragma unroll
      for (int t = 0; t < T; t++) {
        const int one = __reduce_add_sync(0xFFFFFFFFu, sum[j][t]);
        if (lane == t * C + j) all = one;
      }
    if (g.across > 1) {
      const int group = warp / g.across;
      if (lane < C * T) parts[buffer][warp][id] = all;
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(g.across * 32) : "memory");
      if (warp % g.across) continue;
      all = 0;
      for (int w = 0; w < g.across; w++) all += parts[buffer][warp + w][id];
    }
    if (mine) put(g.to, id / C, c, all, scales[id / C], b, bias);
  }
}

// ---------------------------------------------------------------- host

bool encode_rows(CUtensorMap* map, const int8_t* p, int64_t rows, int64_t cols, int64_t stride, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {kAtom, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

int64_t stride_of(int64_t given, uint64_t cols) { return given ? given : (int64_t)cols; }

// Whether a tensor map describes rows of bytes as they lie.
bool mappable(const void* p, int64_t stride, uint64_t cols) {
  return (uintptr_t)p % 16 == 0 && stride % 16 == 0 && stride >= (int64_t)cols && stride < (1ll << 40);
}

// The rows of a weight that are followed by another 15 bytes of it.
int whole_rows(uint64_t rows, int64_t stride) {
  const int64_t last = (15 + stride - 1) / stride;
  return (int64_t)rows > last ? (int)((int64_t)rows - last) : 0;
}

// How a product is laid out: tokens of a tile, and the parts into which its
// depth is cut, `stages` stages each.
struct Cut {
  int tile_n;
  int64_t tiles_m, tiles;
  int splits, stages;
};

// In units of a stage of a 256 x 256 tile (0.55 us): every round of tiles costs its stages (those of narrower
// tiles less, but not by as much: their loads bound them) and four to start and to write; parts cost five more to
// join.  (32 x 4096 x 4096: 9.8 us whole, 8.7 us in parts; 256 x 4096 x 4096: 12.9 us in more parts, 11.2 us in fewer.)
Cut cut_of(const dcf_int8_desc& d) {
  const int blocks = (int)((d.depth + kBK<false> - 1) / kBK<false>);
  Cut best = {};
  double least = 1e300;
  for (int tn : {64, 128, 256}) {
    const int64_t tm = (int64_t)(d.channels + kTileM - 1) / kTileM, tiles = tm * (int64_t)((d.tokens + tn - 1) / tn);
    const double stage = tn == 256 ? 1 : tn == 128 ? 0.65 : 0.5;
    for (int s = 1; s == 1 || (s <= blocks && tiles * s <= kPairs); s++) {
      const int each = (blocks + s - 1) / s, parts = each ? (blocks + each - 1) / each : 1;
      const double rounds = (double)((tiles * parts + kPairs - 1) / kPairs);
      const double cost = rounds * each * stage + (parts > 1 ? 5 : 0) + 4 * stage;
      if (cost < least) {
        least = cost;
        best = {tn, tm, tiles, parts, each};
      }
    }
  }
  return best;
}

// The workspace: tokens of a float type as whole numbers and their scales (or a
// copy of whole numbers that no tensor map describes), a copy of a weight whose stride no
// tensor map takes, and the parts of sums.
struct Layout {
  bool few, own;           // few tokens; each block quantises them
  Cut cut;
  int64_t stride;
  bool copy_b;
  size_t a, scale, b, part, bytes;
};

// (Room for the turns of either width: 496 bytes reach less than 512 past the depth, too.)
int few_padded(const dcf_int8_desc& d) { return (int)((d.depth + 511) / 512 * 512) + 512; }
int few_bucket(const dcf_int8_desc& d) { return d.tokens <= 1 ? 1 : d.tokens <= 2 ? 2 : 4; }
bool few(const dcf_int8_desc& d) {
  return d.tokens <= kFewTokens && d.depth && few_bucket(d) * few_padded(d) <= kFewSmem;
}

// A weight whose rows are no multiple of 16 bytes apart is copied first where tiles are wider than 64 tokens. In
// narrower ones, which read it once or twice, and where only its start lies off a boundary, which is not known before
// the launch, it is read by threads (1001 x 2048 x 1536: 16 us, 7.4 us by map and some 6 us for a copy).
Layout layout_of(const dcf_int8_desc& d) {
  Layout l = {};
  auto take = [&](size_t bytes) {
    const size_t at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  l.stride = (int64_t)((d.depth + 15) / 16 * 16);
  l.few = few(d);
  if (l.few) {
    l.own = d.a_dtype == DCF_I8 || d.tokens * d.depth <= kFewOwn;
    l.a = take(l.own ? 0 : (size_t)d.tokens * l.stride);
    l.scale = take(l.own ? 0 : (size_t)d.tokens * 4);
    return l;
  }
  l.cut = cut_of(d);
  l.a = take((size_t)d.tokens * l.stride);
  l.scale = take(d.a_dtype != DCF_I8 ? (size_t)d.tokens * 4 : 0);
  l.copy_b = l.cut.tile_n > 64 && d.channels > 1 && stride_of(d.b_row_stride, d.depth) % 16;
  l.b = take(l.copy_b ? (size_t)d.channels * l.stride : 0);
  l.part = take(l.cut.splits > 1 ? (size_t)l.cut.tiles * l.cut.splits * kTileM * l.cut.tile_n * 4 : 0);
  return l;
}

template <int T, bool READ> int few_run(const FewArgs& g, cudaStream_t s) {
  if (!prepare_smem((const void*)int8_few_kernel<T, READ>, kFewSmem)) return DCF_ECUDA;
  const int smem = T * g.padded, each = kFewWarps / g.across * kFewChannels;
  const int64_t blocks = ((int64_t)g.to.channels + each - 1) / each, wave = 2 * kPairs * kFewResident;
  return launch(int8_few_kernel<T, READ>, dim3((unsigned)(blocks < wave ? blocks : wave)), kFewThreads, smem, 1, s, g);
}

template <bool READ> int few_product(int bucket, const FewArgs& g, cudaStream_t s) {
  switch (bucket) {
    case 1: return few_run<1, READ>(g, s);
    case 2: return few_run<2, READ>(g, s);
    default: return few_run<4, READ>(g, s);
  }
}

template <int TN, bool READ>
int gemm(const CUtensorMap& mb, const CUtensorMap& ma, const GemmArgs& g, cudaStream_t s) {
  if (!prepare_smem((const void*)int8_gemm_kernel<TN, READ>, kGemmSmem<TN, READ>)) return DCF_ECUDA;
  const unsigned pairs = (unsigned)(g.total < kPairs ? g.total : kPairs);
  return launch(int8_gemm_kernel<TN, READ>, dim3(2 * pairs), kGemmThreads<READ> + (READ ? kReaders : 0), kGemmSmem<TN, READ>, 2, s, mb, ma, g);
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
  const Layout l = layout_of(d);
  const Cut& cut = l.cut;
  uint8_t* work = (uint8_t*)ws;
  int64_t as = stride_of(d.a_row_stride, d.depth), bs = stride_of(d.b_row_stride, d.depth);
  auto pack = [&](const int8_t** p, int64_t* stride, uint64_t rows, size_t at) {
    const int rc = launch_pack_rows(*p, *stride, (int64_t)rows, (int64_t)d.depth, work + at, l.stride, s);
    *p = (int8_t*)work + at;
    *stride = l.stride;
    return rc;
  };
  int rc = DCF_OK;
  const bool ours = d.a_dtype != DCF_I8 && !l.own;  // tokens to quantise first
  if (ours) {
    const dcf_quant_desc tokens = {d.a_dtype, DCF_QUANT_ROWS, d.tokens, d.depth, as, l.stride};
    a_scale = (float*)(work + l.scale);
    as = l.stride;
    if ((rc = launch_quantize(tokens, a, (int8_t*)work + l.a, (float*)a_scale, s))) return rc;
    a = work + l.a;
  }
  Result to;
  to.a_scale = a_scale;
  to.b_scale = b_scale;
  to.bias = bias;
  to.out = out;
  to.out_dtype = (int)d.out_dtype;
  to.tokens = (int)d.tokens;
  to.channels = (int)d.channels;
  to.stride = stride_of(d.out_row_stride, d.channels);
  to.pairs = (uintptr_t)out % 4 == 0 && (d.tokens == 1 || to.stride % 2 == 0);
  auto on16 = [&](const void* p, int64_t stride, uint64_t rows, size_t es) {
    return (uintptr_t)p % 16 == 0 && (rows == 1 || stride * (int64_t)es % 16 == 0);
  };
  if (l.few) {
    FewArgs g = {};
    g.to = to;
    g.a = a;
    g.a_dtype = (int)(ours ? (uint32_t)DCF_I8 : d.a_dtype);
    g.a_stride = as;
    g.a_vectors = on16(a, as, d.tokens, dtype_size(g.a_dtype));
    g.b = b;
    g.b_stride = bs;
    g.whole = whole_rows(d.channels, bs);
    g.depth = (int)d.depth;
    g.padded = few_padded(d);
    g.early = ours;
    const int64_t groups = ((int64_t)d.channels + kFewChannels - 1) / kFewChannels;
    for (g.across = 1; g.across < kFewWarps && g.across * 512 < (int)d.depth &&
                       groups * g.across < 2 * kPairs * kFewResident * kFewWarps * 3 / 4;)
      g.across *= 2;
    const int bucket = few_bucket(d);
    const bool read = !on16(b, bs, d.channels, 1);
    return !read ? few_product<false>(bucket, g, s) : few_product<true>(bucket, g, s);
  }
  const int8_t* q = (const int8_t*)a;
  GemmArgs g = {};
  g.to = to;
  g.tiles_m = (int)cut.tiles_m;
  g.splits = d.depth ? cut.splits : 0;
  g.total = cut.tiles * cut.splits;
  g.part = (int*)(work + l.part);
  g.st = st;
  if (d.depth) {
    if (!mappable(q, as, d.depth) && (rc = pack(&q, &as, d.tokens, l.a))) return rc;
    if (l.copy_b && (rc = pack(&b, &bs, d.channels, l.b))) return rc;
    const bool read = !mappable(b, bs, d.depth);
    const int bk = read ? kBK<true> : kBK<false>;
    g.blocks = (int)((d.depth + bk - 1) / bk);
    g.split_k = cut.stages * (kBK<false> / bk);
    g.b = b;
    g.b_stride = bs;
    g.whole = whole_rows(d.channels, bs);
    g.depth = (int)d.depth;
    g.early = ours && !l.copy_b;
    if (!encoder()) return DCF_EUNSUPPORTED;
    CUtensorMap ma, mb = {};
    if ((!read && !encode_rows(&mb, b, (int64_t)d.channels, (int64_t)d.depth, bs, kSide)) ||
        !encode_rows(&ma, q, (int64_t)d.tokens, (int64_t)d.depth, as, cut.tile_n / 2))
      return DCF_ECUDA;
    switch (cut.tile_n) {
      case 64: rc = read ? gemm<64, true>(mb, ma, g, s) : gemm<64, false>(mb, ma, g, s); break;
      case 128: rc = read ? gemm<128, true>(mb, ma, g, s) : gemm<128, false>(mb, ma, g, s); break;
      default: rc = read ? gemm<256, true>(mb, ma, g, s) : gemm<256, false>(mb, ma, g, s);
    }
    if (rc || cut.splits == 1) return rc;
  }
  const int64_t joins = ((int64_t)d.channels + 4 * kJoinThreads - 1) / (4 * kJoinThreads) * (int64_t)d.tokens;
  return launch(int8_join_kernel, dim3((unsigned)(joins < (1 << 30) ? joins : 1 << 30)), kJoinThreads, 0, 1, s, g,
                cut.tile_n);
}

}  // namespace dcf
