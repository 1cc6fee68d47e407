// dcf_bias.cu — the relative position bias expanded from a learned table of
// buckets, and the gradient of that table.
//
//   bias:      out[h][i][j] = table[bucket(j - pos(i))][h]
//   gradient:  d table[v][h] = sum of g[b][h][i][j] over b and the (i, j)
//              whose bucket is v
//
// An exported model holds the first as iota, sub, abs, log, floor, min,
// select, gather and transpose; here the bucket of a distance is a search
// in the sorted list of distances at which buckets begin.  That list is
// made on the host by comparing integer powers (bias_starts), so no device
// log decides a border.
//
// Both are bound by HBM: one write, or one read, per element of the bias,
// against one table value or one addition.  What has to be kept small is the
// work per element around that, above all finding its bucket: a row is
// cut once into the two far ranges, which have one bucket each, and the near
// columns between, whose buckets come from a table of distances in shared
// memory; a thread owns one 16-byte vector of a row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "dcf_kernels.cuh"

namespace dcf {

namespace {

constexpr int kMaxB = DCF_BIAS_MAX_BUCKETS;
// A B200's, for the sizes of grids and splits.  Not asked of the device: sums then split alike
// wherever they run, and a workspace's size needs no device.  Any number of SMs runs them.
constexpr int kSms = 148;
constexpr int kTable = 256;  // distances whose bucket is looked up rather than searched

// How a distance maps to its bucket; a kernel parameter.
struct Buckets {
  int half;           // buckets per direction
  int both;           // keys after the query have buckets half .. 2 half - 1
  int causal;
  int last;           // distances >= last have bucket half - 1
  int start[kMaxB];   // first distance of each bucket, sorted
  alignas(4) uint8_t near[kTable];  // bucket number of each distance below min(last, kTable)
};

struct BiasArgs {
  uint64_t queries;
  int keys;
  int64_t first;
  int64_t rs, hs, bs;   // strides in elements
  int heads, nb;
  uint64_t batch;
  const int32_t* pos;
};

// A row's columns: those up to `left` have the last bucket of the query's
// side, those from `right` on one bucket as well (the last of the other side, or,
// with one direction only, bucket 0), those from `end` on are masked or not there.
// Between left and right the bucket depends on the distance, column - query,
// which fits 32 bits there.
struct Row {
  int left, right, end, query;
};

__device__ __forceinline__ int clip(int64_t x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }

__device__ __forceinline__ Row row_of(const Buckets& t, const BiasArgs& a, uint64_t i) {
  const int64_t q = a.pos ? (int64_t)a.pos[i] : a.first + (int64_t)i;
  Row r;
  r.left = clip(q - t.last, -1, a.keys);
  r.right = clip(q + (t.both && t.last > 1 ? t.last : 1), 0, a.keys);
  r.end = t.causal ? clip(q + 1, 0, a.keys) : a.keys;
  r.query = (int)q;  // near columns: their distance is right modulo 2^32
  return r;
}

// The bucket number of every near distance, in shared memory.
struct Near {
  alignas(4) uint8_t of[kTable];
  int start[kMaxB];
};

__device__ __forceinline__ int search(const int* start, int half, int n) {
  int lo = 0, hi = half;  // start[lo] <= n < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

// By all threads of the block; the caller synchronises.
__device__ __forceinline__ void fill_near(Near& near, const Buckets& t, int threads) {
  for (int i = threadIdx.x; i < t.half; i += threads) near.start[i] = t.start[i];
  for (int i = threadIdx.x; i < kTable / 4; i += threads) ((uint32_t*)near.of)[i] = ((const uint32_t*)t.near)[i];
}

// Bucket of a column between a row's left and right.
__device__ __forceinline__ int near_bucket(const Near& near, const Buckets& t, const Row& r, int col) {
  const int d = (int)((unsigned)col - (unsigned)r.query), n = d < 0 ? -d : d;
  return (t.both && d > 0 ? t.half : 0) + (n < kTable ? near.of[n] : search(near.start, t.half, n));
}

template <class T> __device__ __forceinline__ T minus_infinity();
template <> __device__ __forceinline__ float minus_infinity<float>() { return -INFINITY; }
template <> __device__ __forceinline__ double minus_infinity<double>() { return -(double)INFINITY; }
template <> __device__ __forceinline__ __half minus_infinity<__half>() { return __ushort_as_half(0xFC00); }
template <> __device__ __forceinline__ __nv_bfloat16 minus_infinity<__nv_bfloat16>() {
  return __ushort_as_bfloat16(0xFF80);
}

// The table's value in the bias's type: the same bits, or one rounding to
// nearest from a f32 table.
template <class T, class S> __device__ __forceinline__ T cast(S v) { return v; }
template <> __device__ __forceinline__ __half cast<__half, float>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 cast<__nv_bfloat16, float>(float v) {
  return __float2bfloat16_rn(v);
}

template <class T> struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

// ---------------------------------------------------------------- bias

constexpr int kFwdThreads = 256, kFwdWarps = kFwdThreads / 32;

// A block writes rows of one head, one after the other, a warp to a row or to a
// part of one: what is being written at any time then lies close
// together (blocks that wrote one row of many heads, sharing the lookup of buckets, reached
// 3.3 - 5.5 TB/s, the less the more heads).  Vectors sit on 16-byte addresses, rows
// need not; the ones at a row's ends are written element by element.  Vectors that
// lie in a far range, or behind the mask, are one of three constants;
// a near column reads its value from a table by distance.
template <class T, class S>
__global__ void __launch_bounds__(kFwdThreads) bias_kernel(const __grid_constant__ Buckets t,
                                                           const __grid_constant__ BiasArgs a,
                                                           const S* __restrict__ table, T* __restrict__ out,
                                                           uint32_t chunk, uint32_t chunks, uint64_t items, int turns,
                                                           int team) {
  constexpr int N = Vec<T>::N;
  __shared__ Near near;
  __shared__ T tab[kMaxB], value[2 * kTable];  // by bucket; by distance + last
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  fill_near(near, t, kFwdThreads);
  for (int v = threadIdx.x; v < a.nb; v += kFwdThreads) tab[v] = cast<T, S>(table[(size_t)v * a.heads + h]);
  __syncthreads();
  const bool tabled = t.last <= kTable;
  if (tabled) {
    for (int i = threadIdx.x; i < 2 * t.last; i += kFwdThreads) {
      const int d = i - t.last, n = d < 0 ? -d : d;
      if (d != -t.last) value[i] = tab[(d > 0 ? (t.both ? t.half : 0) : 0) + (d > 0 && !t.both ? 0 : near.of[n])];
    }
    __syncthreads();
  }
  Vec<T> left, right, masked;
#pragma unroll
  for (int k = 0; k < N; k++) {
    left.e[k] = tab[t.half - 1];
    right.e[k] = tab[t.both ? 2 * t.half - 1 : 0];
    masked.e[k] = minus_infinity<T>();
  }

  for (int turn = 0; turn < turns; turn++) {
    const uint64_t item = ((uint64_t)blockIdx.x * turns + turn) * (kFwdWarps / team) + warp / team;
    if (item >= items) return;
    uint64_t row;
    uint32_t part;
    if (items < (1ull << 32)) {
      row = (uint32_t)item / chunks;
      part = (uint32_t)item - (uint32_t)row * chunks;
    } else {
      row = item / chunks;
      part = (uint32_t)(item - row * chunks);
    }
    const Row r = row_of(t, a, row);
    T* line = out + (int64_t)h * a.hs + (int64_t)row * a.rs;
    int c = (int)((part * chunk + warp % team) * 32 + lane) * N - (int)(((uintptr_t)line / sizeof(T)) % N);
    line += c;
    for (uint32_t i = warp % team; i < chunk && c < a.keys; i += team, c += team * 32 * N, line += team * 32 * N) {
      Vec<T> x;
      if (c >= r.end) {
        x = masked;
      } else if (c + N - 1 <= r.left) {
        x = left;
      } else if (c >= r.right && c + N <= r.end) {
        x = right;
      } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
          const int e = c + k;
          x.e[k] = e >= r.end    ? masked.e[0]
                   : e <= r.left ? left.e[0]
                   : e >= r.right ? right.e[0]
                   : tabled       ? value[(int)((unsigned)e - (unsigned)r.query) + t.last]
                                  : tab[near_bucket(near, t, r, e)];
        }
      }
      if (c >= 0 && c + N <= a.keys) {
        *(uint4*)line = *(const uint4*)&x;
      } else {
#pragma unroll
        for (int k = 0; k < N; k++)
          if (c + k >= 0 && c + k < a.keys) line[k] = x.e[k];
      }
    }
  }
}

// ------------------------------------------------------------ gradient

template <class T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
// s + x in the sum's type.  16-bit values are added by one instruction, exact but
// for the sum's rounding, where a conversion and an addition are two.
__device__ __forceinline__ float plus(float s, float x) { return s + x; }
__device__ __forceinline__ double plus(double s, double x) { return s + x; }
__device__ __forceinline__ float plus(float s, __half x) {
  asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(s) : "h"(__half_as_ushort(x)));
  return s;
}
__device__ __forceinline__ float plus(float s, __nv_bfloat16 x) {
  asm("add.rn.f32.bf16 %0, %1, %0;" : "+f"(s) : "h"(__bfloat16_as_ushort(x)));
  return s;
}

constexpr size_t kAccBytes = 48 << 10;
constexpr int kOffsets = 2048;  // distances (each way) for which a block tables where their sums are

BiasArgs args_of(const dcf_bias_desc& d, const int32_t* pos) {
  BiasArgs a;
  a.queries = d.queries;
  a.keys = (int)d.keys;
  a.first = d.first_query;
  a.rs = d.row_stride ? d.row_stride : (int64_t)d.keys;
  a.hs = d.head_stride ? d.head_stride : (int64_t)d.queries * a.rs;
  a.bs = d.batch_stride ? d.batch_stride : (int64_t)d.heads * a.hs;
  a.heads = (int)d.heads;
  a.nb = (int)d.num_buckets;
  a.batch = d.batch;
  a.pos = pos;
  return a;
}

// How the gradient is split: `splits` CTAs per head, each with `warps`
// warps, every warp taking items (`batch` entries of one row, or `chunk` steps of
// 32 vectors of it) in turn.  Fixed by the sizes and strides alone: sums keep
// their order, as long as rows begin at the same places within 16 bytes.
struct GradPlan {
  int warps, splits;
  uint32_t chunk, chunks, batches;
  uint64_t batch, items;
};

// Vectors that a row of `keys` elements can touch: one more where rows need
// not start on a 16-byte boundary.
uint64_t vectors_of_row(uint64_t keys, uint64_t n, bool aligned) { return (keys + (aligned ? n - 1 : 2 * n - 2)) / n; }

bool strides_aligned(const BiasArgs& a, uint64_t n) {
  return a.rs % (int64_t)n == 0 && a.hs % (int64_t)n == 0 && a.bs % (int64_t)n == 0;
}

GradPlan grad_plan(const dcf_bias_desc& d) {
  GradPlan p;
  const size_t es = dtype_size((int)d.dtype), acc = d.dtype == DCF_F64 ? 8 : 4;
  const uint64_t n = 16 / es;
  p.warps = (int)(kAccBytes / (d.num_buckets * 32 * acc));
  p.warps = p.warps > 8 ? 8 : p.warps < 1 ? 1 : p.warps;
  const int64_t rs = d.row_stride ? d.row_stride : (int64_t)d.keys;
  const int64_t hs = d.head_stride ? d.head_stride : (int64_t)d.queries * rs;
  const int64_t bs = d.batch_stride ? d.batch_stride : (int64_t)d.heads * hs;
  // (Where only the first row is not aligned, a row's last part takes the
  // vector more that it may have.)
  const bool aligned = rs % (int64_t)n == 0 && hs % (int64_t)n == 0 && bs % (int64_t)n == 0;
  const uint64_t steps = (vectors_of_row(d.keys, n, aligned) + 31) / 32, rows = d.queries;
  const uint64_t ctas = d.heads ? (uint64_t)(kSms * 4 + d.heads - 1) / d.heads : 1;  // per head: four to an SM
  const uint64_t slots = ctas * p.warps;
  if (rows == 0 || d.batch == 0 || steps == 0) {
    p.chunk = p.chunks = p.batches = 1;
    p.batch = 1;
    p.items = 0;
    p.splits = 1;
    return p;
  }
  // Batch entries of a row share the buckets, as long as their rows are aligned
  // alike; where that leaves few items, rows are cut into parts, then the batch,
  // as far as each warp has no more than three (8 x 12 x 512 x 512 bf16: 24.6 us
  // with up to six smaller items, 18.4 us with three).
  uint64_t cuts = slots * 3 / rows;
  cuts = cuts < 1 ? 1 : cuts > steps ? steps : cuts;
  p.chunk = (uint32_t)((steps + cuts - 1) / cuts);
  p.chunks = (uint32_t)((steps + p.chunk - 1) / p.chunk);
  uint64_t batches = slots * 3 / (rows * p.chunks);
  if (batches < 1) batches = 1;
  if (batches > d.batch || bs % (int64_t)n) batches = d.batch;
  p.batch = (d.batch + batches - 1) / batches;
  p.batches = (uint32_t)((d.batch + p.batch - 1) / p.batch);
  p.items = rows * p.batches * p.chunks;
  // As few CTAs as take no more turns than the most would.
  const uint64_t turns = (p.items + slots - 1) / slots;
  const uint64_t want = (p.items + turns * p.warps - 1) / (turns * p.warps);
  p.splits = (int)(want < 1 ? 1 : want);
  return p;
}

template <class A, int N> __device__ __forceinline__ A total(A (&s)[N]) {
#pragma unroll
  for (int u = N / 2; u > 0; u >>= 1)
#pragma unroll
    for (int k = 0; k < u; k++) s[k] += s[k + u];
  return s[0];
}

// A warp walks along a row in steps of 32 vectors.  Steps that lie wholly in a
// far range are only summed, one instruction per element; the others
// are summed over the batch entries, then every element adds into its bucket's
// sum, which each lane has for itself in shared memory, found by a table of
// distances.  2 x 16 x 4001 x 4001 causal f16: 126 us, 4.1 TB/s; what it waits for
// is its loads (half of the stalls).  Eight loads in flight per lane, or five CTAs
// to an SM, need more registers than there are: 157 and 172 us.
template <class T>
__global__ void __launch_bounds__(256, 4) bias_grad_kernel(const __grid_constant__ Buckets t,
                                                           const __grid_constant__ BiasArgs a, const T* __restrict__ g,
                                                           const __grid_constant__ GradPlan p,
                                                           typename AccOf<T>::type* __restrict__ part,
                                                           typename AccOf<T>::type* __restrict__ dtable, int add) {
  using A = typename AccOf<T>::type;
  constexpr int N = Vec<T>::N, kStep = 32 * N;
  extern __shared__ __align__(16) uint8_t smem[];
  A* acc = (A*)smem;   // [warp][bucket][lane]: every lane adds into its own column, in its own order
  __shared__ Near near;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int threads = p.warps * 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for the whole grid
  uint16_t* offset = (uint16_t*)(acc + (size_t)p.warps * a.nb * 32);  // by distance + far: 32 x bucket
  const bool tabled = t.last <= kOffsets;
  const int far = max(t.last, 1);
  fill_near(near, t, threads);
  for (int i = threadIdx.x; i < p.warps * a.nb * 32; i += threads) acc[i] = 0;
  __syncthreads();
  if (tabled) {
    for (int i = threadIdx.x; i <= 2 * far; i += threads) {
      const int d = i - far, n = d < 0 ? -d : t.both ? d : 0;
      const int bucket = n < kTable ? near.of[n] : search(near.start, t.half, n);
      offset[i] = (uint16_t)(32 * ((t.both && d > 0 ? t.half : 0) + bucket));
    }
    __syncthreads();
  }
  A* mine = acc + (size_t)warp * a.nb * 32 + lane;

  const int h = blockIdx.y;
  A far_left = 0, far_right = 0;
  const uint64_t warps = (uint64_t)gridDim.x * p.warps, self = (uint64_t)blockIdx.x * p.warps + warp;
  for (uint64_t turn = 0; turn * warps < p.items; turn++) {
    // Forth and back: with a causal mask later rows are longer.
    const uint64_t item = turn * warps + (turn & 1 ? warps - 1 - self : self);
    if (item >= p.items) continue;
    uint64_t row, b;
    uint32_t cut;
    if (p.items < (1ull << 32)) {
      const uint32_t x = (uint32_t)item / p.chunks;
      cut = (uint32_t)item - x * p.chunks;
      row = x / p.batches;
      b = x - (uint32_t)row * p.batches;
    } else {
      const uint64_t x = item / p.chunks;
      cut = (uint32_t)(item - x * p.chunks);
      row = x / p.batches;
      b = x - row * p.batches;
    }
    const Row r = row_of(t, a, row);
    // Near enough for every distance to fit 32 bits, far enough to change no bucket
    // that the table has.
    const int64_t at = a.pos ? (int64_t)a.pos[row] : a.first + (int64_t)row;
    const int query = clip(at, -kOffsets - 1, (int64_t)a.keys + kOffsets + 1);
    b *= p.batch;
    const uint64_t b_end = min(a.batch, b + p.batch);
    const T* line = g + (int64_t)b * a.bs + (int64_t)h * a.hs + (int64_t)row * a.rs;
    const int entries = (int)(b_end - b);
    const int shift = (int)(((uintptr_t)line / sizeof(T)) % N);  // elements behind a 16-byte boundary, for all entries
    const T* lane_at = line - shift + lane * N;
    // Steps [l0, l1) lie in the left range, [r0, r1) in the right one.
    const int l0 = shift ? 1 : 0, l1 = (min(r.left + 1, r.end) + shift) / kStep;
    const int r0 = max(l0, (r.right + shift + kStep - 1) / kStep), r1 = (r.end + shift) / kStep;
    int stop = r.end > 0 ? (r.end + shift + kStep - 1) / kStep : 0;
    if (cut + 1 < p.chunks) stop = min(stop, (int)((cut + 1) * p.chunk));
    int i = (int)(cut * p.chunk);
    while (i < stop) {
      const bool left = i >= l0 && i < l1;
      if (left || (i >= r0 && i < r1)) {
        const int to = min(stop, left ? l1 : r1);
        A s[N];
#pragma unroll
        for (int k = 0; k < N; k++) s[k] = 0;
        // Four loads in flight, the last ones too, along what is longer: the steps
        // or the batch entries.
        const bool across = entries > to - i;
        const int fast = across ? entries : to - i, slow = across ? to - i : entries;
        const int64_t fast_by = across ? a.bs : kStep, slow_by = across ? kStep : a.bs;
        const T* at = lane_at + (int64_t)i * kStep;
        for (int e = 0; e < slow; e++, at += slow_by) {
          const T* from = at;
          for (int j = 0; j < fast; j += 4, from += 4 * fast_by) {
            Vec<T> x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              *(uint4*)&x[k] = make_uint4(0, 0, 0, 0);
              if (j + k < fast) *(uint4*)&x[k] = __ldg((const uint4*)(from + k * fast_by));
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
              for (int k = 0; k < N; k++) s[k] = plus(s[k], x[u].e[k]);
          }
        }
        if (left) far_left += total(s);
        else far_right += total(s);
        i = to;
        continue;
      }
      const int c = i * kStep + lane * N - shift;
      i++;
      if (max(c, 0) >= r.end) continue;
      A sum[N];
#pragma unroll
      for (int k = 0; k < N; k++) sum[k] = 0;
      const T* at = line + c;
      if (c >= 0 && c + N <= a.keys) {
        for (int e = 0; e < entries; e += 4, at += 4 * a.bs) {
          Vec<T> x[4];
#pragma unroll
          for (int u = 0; u < 4; u++) {
            *(uint4*)&x[u] = make_uint4(0, 0, 0, 0);
            if (e + u < entries) *(uint4*)&x[u] = __ldg((const uint4*)(at + u * a.bs));
          }
#pragma unroll
          for (int k = 0; k < N; k++)
#pragma unroll
            for (int u = 0; u < 4; u++) sum[k] = plus(sum[k], x[u].e[k]);
        }
      } else {
        for (int e = 0; e < entries; e++, at += a.bs)
#pragma unroll
          for (int k = 0; k < N; k++)
            if (c + k >= 0 && c + k < r.end) sum[k] = plus(sum[k], at[k]);
      }
      if (c < 0 || c + N > r.end) {  // what lies outside adds nothing
#pragma unroll
        for (int k = 0; k < N; k++)
          if (c + k < 0 || c + k >= r.end) sum[k] = 0;
      }
      // A first or last step that a far range covers as far as the row reaches.
      const int from = i * kStep - kStep - shift;
      if (from + kStep <= r.left + 1 || from >= r.right) {
        if (from >= r.right) far_right += total(sum);
        else far_left += total(sum);
        continue;
      }
      // (Lanes in a far range add into its bucket the same way: a branch of
      // their own cost the warp more.)
      if (tabled) {
        const int d0 = c - query + far;
#pragma unroll
        for (int k = 0; k < N; k++) mine[offset[min(max(d0 + k, 0), 2 * far)]] += sum[k];
      } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
          const int e = c + k;
          const int bucket = e <= r.left    ? t.half - 1
                             : e >= r.right ? (t.both ? 2 * t.half - 1 : 0)
                                            : near_bucket(near, t, r, e);
          mine[32 * bucket] += sum[k];
        }
      }
    }
  }
  mine[(t.half - 1) * 32] += far_left;
  mine[(t.both ? 2 * t.half - 1 : 0) * 32] += far_right;
  __syncthreads();
  for (int v = warp; v < a.nb; v += p.warps) {
    A s = 0;
    for (int w = 0; w < p.warps; w++) s += acc[((size_t)w * a.nb + v) * 32 + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) {
      if (gridDim.x == 1) {
        A* d = dtable + (size_t)v * a.heads + h;
        *d = add ? *d + s : s;
      } else {
        part[((size_t)h * gridDim.x + blockIdx.x) * a.nb + v] = s;
      }
    }
  }
}

// One warp per table entry adds the splits' parts, always in the same order.
template <class A>
__global__ void __launch_bounds__(256) bias_grad_join_kernel(const A* __restrict__ part, int splits, int nb, int heads,
                                                             A* __restrict__ dtable, int add) {
  // Launched as a programmatic dependent: its start overlaps the parts' end.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= nb * heads) return;
  const int h = e / nb, v = e - h * nb;
  A s = 0;
  for (int k = lane; k < splits; k += 32) s += part[((size_t)h * splits + k) * nb + v];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (lane == 0) {
    A* d = dtable + (size_t)v * heads + h;
    *d = add ? *d + s : s;
  }
}

// -------------------------------------------------------------- host

// A non-negative whole number of up to 31 * DCF_BIAS_MAX_BUCKETS bits.
struct Big {
  uint32_t w[kMaxB + 4];
  int n = 1;
  Big() { w[0] = 1; }
  void times(uint32_t f) {
    uint64_t carry = 0;
    for (int i = 0; i < n; i++) {
      carry += (uint64_t)w[i] * f;
      w[i] = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) w[n++] = (uint32_t)carry;
  }
  bool at_least(const Big& o) const {
    if (n != o.n) return n > o.n;
    for (int i = n - 1; i >= 0; i--)
      if (w[i] != o.w[i]) return w[i] > o.w[i];
    return true;
  }
};

// The first distance of each of `half` buckets.  Bucket e + k (k >= 1)
// begins at the smallest n with n^m >= last^k e^(m - k), m = half - e: at
// x = e (last / e)^(k / m), rounded up.  x in 64 bits is off by some 1e-14 of
// itself (an exponential of a product below 22), so unless a whole number
// lies within 1e-13 of it the integers need not be asked.
void bias_starts(int half, uint32_t last, int* start) {
  const int e = half / 2, m = half - e;
  for (int v = 0; v <= e && v < half; v++) start[v] = v;
  for (int k = 1; k < m; k++) {
    const double x = e * exp((double)k / m * log((double)last / e));
    const double near = floor(x * (1 + 1e-13));
    uint32_t n = (uint32_t)floor(x) + 1;
    if (near != floor(x * (1 - 1e-13))) {
      Big l, r;
      n = (uint32_t)near;
      for (int i = 0; i < m; i++) l.times(n);
      for (int i = 0; i < k; i++) r.times(last);
      for (int i = k; i < m; i++) r.times((uint32_t)e);
      if (!l.at_least(r)) n++;
    }
    start[e + k] = (int)n;
  }
}

Buckets buckets_of(const dcf_bias_desc& d) {
  Buckets t;
  t.both = (d.flags & DCF_BIAS_BIDIRECTIONAL) != 0;
  t.causal = (d.flags & DCF_BIAS_CAUSAL) != 0;
  t.half = (int)(t.both ? d.num_buckets / 2 : d.num_buckets);
  bias_starts(t.half, d.max_distance, t.start);
  t.last = t.start[t.half - 1];
  for (int n = 0, v = 0; n < kTable; n++) {
    while (v + 1 < t.half && t.start[v + 1] <= n) v++;
    t.near[n] = (uint8_t)v;
  }
  return t;
}

template <class T, class S>
int launch_bias_t(const dcf_bias_desc& d, const void* table, const int32_t* pos, void* out, cudaStream_t stream) {
  constexpr uint64_t N = Vec<T>::N;
  const Buckets t = buckets_of(d);
  BiasArgs a = args_of(d, pos);
  a.bs = 0;
  const bool aligned = (uintptr_t)out % 16 == 0 && strides_aligned(a, N);
  // A warp's steps along a row; whole rows, or parts where there are few.
  const uint64_t steps = (vectors_of_row(d.keys, N, aligned) + 31) / 32, rows = d.queries * d.heads;
  uint64_t cuts = kSms * 32 / rows;
  cuts = cuts < 1 ? 1 : cuts > steps ? steps : cuts;
  const uint32_t chunk = (uint32_t)((steps + cuts - 1) / cuts), chunks = (uint32_t)((steps + chunk - 1) / chunk);
  const uint64_t items = d.queries * chunks;
  // Up to 32 KB for the tables that a block sets up, where there is enough to do.
  // Warps that share a row, by turns of a step: long rows then keep a block's writes
  // together (250 scattered rows of 8192, 32 heads: 24.8 us with two, 29.3 us with one), short
  // ones pay for every warp's look at the row (4001: 180 and 196 us).
  int team = 1;
  while (team < kFwdWarps && chunk >= 32u * team) team *= 2;
  uint64_t turns = (32 << 10) / (kFwdWarps / team * chunk * 512);
  const uint64_t most = items * d.heads / (kFwdWarps / team * kSms * 8);
  if (turns > most) turns = most;
  if (turns < 1) turns = 1;
  const uint64_t blocks = (items + kFwdWarps / team * turns - 1) / (kFwdWarps / team * turns);
  bias_kernel<T, S><<<dim3((unsigned)blocks, d.heads), kFwdThreads, 0, stream>>>(t, a, (const S*)table, (T*)out, chunk,
                                                                                chunks, items, (int)turns, team);
  note_launch();
  return cudaPeekAtLastError() == cudaSuccess ? DCF_OK : DCF_ECUDA;
}

template <class T>
int launch_grad_t(const dcf_bias_desc& d, const void* g, const int32_t* pos, void* dtable, void* ws,
                  cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  const Buckets t = buckets_of(d);
  const BiasArgs a = args_of(d, pos);
  const GradPlan p = grad_plan(d);
  const int add = (d.flags & DCF_BIAS_ACCUMULATE) != 0;
  const size_t offsets = t.last <= kOffsets ? 2 * (size_t)(t.last < 1 ? 1 : t.last) + 1 : 0;
  const size_t smem = (size_t)p.warps * d.num_buckets * 32 * sizeof(A) + offsets * 2;
  if (smem > kAccBytes - 4096 &&
      cudaFuncSetAttribute(bias_grad_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 80 << 10) != cudaSuccess)
    return DCF_ECUDA;
  bias_grad_kernel<T><<<dim3((unsigned)p.splits, d.heads), p.warps * 32, smem, stream>>>(
      t, a, (const T*)g, p, (A*)ws, (A*)dtable, add);
  note_launch();
  if (p.splits > 1) {
    const unsigned entries = d.num_buckets * d.heads;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((entries + 7) / 8);
    c.blockDim = dim3(256);
    c.stream = stream;
    cudaLaunchAttribute dependent[1];
    dependent[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    c.attrs = dependent;
    c.numAttrs = 1;
    note_launch();
    if (cudaLaunchKernelEx(&c, bias_grad_join_kernel<A>, (const A*)ws, p.splits, a.nb, a.heads, (A*)dtable, add) !=
        cudaSuccess)
      return DCF_ECUDA;
  }
  return cudaPeekAtLastError() == cudaSuccess ? DCF_OK : DCF_ECUDA;
}

}  // namespace

int bias_desc_check(const dcf_bias_desc* d, bool grad) {
  auto bad = [](const char* m) { return record_error(DCF_EINVAL, m); };
  if (!d) return bad("null descriptor");
  if (d->dtype != DCF_F16 && d->dtype != DCF_BF16 && d->dtype != DCF_F32 && d->dtype != DCF_F64)
    return bad("position bias: dtype must be f16, bf16, f32 or f64");
  if (!grad && d->table_dtype != d->dtype &&
      !(d->table_dtype == DCF_F32 && (d->dtype == DCF_F16 || d->dtype == DCF_BF16)))
    return bad("position bias: table_dtype must be dtype, or f32 beside f16 / bf16");
  if (d->flags & ~(DCF_BIAS_BIDIRECTIONAL | DCF_BIAS_CAUSAL | (grad ? DCF_BIAS_ACCUMULATE : 0u)))
    return bad("position bias: unknown flag");
  const uint32_t both = d->flags & DCF_BIAS_BIDIRECTIONAL;
  if (d->num_buckets < (both ? 2u : 1u) || d->num_buckets > DCF_BIAS_MAX_BUCKETS)
    return bad("position bias: num_buckets out of range");
  const uint32_t half = both ? d->num_buckets / 2 : d->num_buckets;
  if (d->max_distance <= half / 2 || d->max_distance >= 1u << 31)
    return bad("position bias: max_distance must be above the exact buckets and below 2^31");
  if (d->heads > 65535) return bad("position bias: at most 65535 heads");
  const uint64_t lim = 1ull << 31;
  if (d->queries >= lim || d->keys > lim - 65536 || (grad && d->batch >= lim))
    return bad("position bias: queries and batch must be below 2^31, keys at most 2^31 - 65536");
  if (d->first_query > (1ll << 40) || d->first_query < -(1ll << 40)) return bad("position bias: first_query out of range");
  if (d->row_stride < 0 || d->head_stride < 0 || d->batch_stride < 0) return bad("position bias: negative stride");
  // Extents in 128 bits, so that no product of the checks wraps.
  const __int128 rs = d->row_stride ? d->row_stride : (int64_t)d->keys;
  const __int128 hs = d->head_stride ? d->head_stride : (__int128)d->queries * rs;
  const __int128 bs = d->batch_stride ? d->batch_stride : (__int128)d->heads * hs;
  const uint64_t batch = grad ? d->batch : 1;
  if (!d->queries || !d->keys || !d->heads || !batch) return DCF_OK;
  const __int128 span = (__int128)(d->queries - 1) * rs + (__int128)(d->heads - 1) * hs + (__int128)(batch - 1) * bs +
                        (__int128)d->keys;
  if (span > ((__int128)1 << 46)) return bad("position bias: tensor too large");
  if (!grad) {
    // Rows that overlap would be written twice.  Either dim may be the outer one.
    const __int128 nq = d->queries, nh = d->heads, nk = d->keys;
    const bool rows_in_heads = (nq == 1 || rs >= nk) && (nh == 1 || hs >= (nq - 1) * rs + nk);
    const bool heads_in_rows = (nh == 1 || hs >= nk) && (nq == 1 || rs >= (nh - 1) * hs + nk);
    if (!rows_in_heads && !heads_in_rows) return bad("position bias: strides make rows overlap");
  }
  return DCF_OK;
}

size_t bias_grad_workspace(const dcf_bias_desc& d) {
  const GradPlan p = grad_plan(d);
  const size_t acc = d.dtype == DCF_F64 ? 8 : 4;
  const size_t bytes = p.splits > 1 ? (size_t)p.splits * d.heads * d.num_buckets * acc : 0;
  return (bytes + 255) / 256 * 256;
}

int launch_position_bias(const dcf_bias_desc& d, const void* table, const int32_t* pos, void* out,
                         cudaStream_t stream) {
  const bool from32 = d.table_dtype == DCF_F32;
  switch (d.dtype) {
    case DCF_F16:
      return from32 ? launch_bias_t<__half, float>(d, table, pos, out, stream)
                    : launch_bias_t<__half, __half>(d, table, pos, out, stream);
    case DCF_BF16:
      return from32 ? launch_bias_t<__nv_bfloat16, float>(d, table, pos, out, stream)
                    : launch_bias_t<__nv_bfloat16, __nv_bfloat16>(d, table, pos, out, stream);
    case DCF_F32: return launch_bias_t<float, float>(d, table, pos, out, stream);
    case DCF_F64: return launch_bias_t<double, double>(d, table, pos, out, stream);
    default: return DCF_EUNSUPPORTED;
  }
}

int launch_position_bias_grad(const dcf_bias_desc& d, const void* g, const int32_t* pos, void* dtable, void* ws,
                              cudaStream_t stream) {
  switch (d.dtype) {
    case DCF_F16: return launch_grad_t<__half>(d, g, pos, dtable, ws, stream);
    case DCF_BF16: return launch_grad_t<__nv_bfloat16>(d, g, pos, dtable, ws, stream);
    case DCF_F32: return launch_grad_t<float>(d, g, pos, dtable, ws, stream);
    case DCF_F64: return launch_grad_t<double>(d, g, pos, dtable, ws, stream);
    default: return DCF_EUNSUPPORTED;
  }
}

}  // namespace dcf
