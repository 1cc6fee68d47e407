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
// columns between, whose buckets come from a table of distances in shared memory;
// a thread owns one 16-byte vector, and in the bias its lookup serves all heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "dcf_launch.h"

namespace dcf {

namespace {

constexpr int kMaxB = DCF_BIAS_MAX_BUCKETS;
constexpr int kSms = 148;

// How a distance maps to its bucket; a kernel parameter.
struct Buckets {
  int half;           // buckets per direction
  int both;           // keys after the query have buckets half .. 2 half - 1
  int causal;
  int last;           // distances >= last have bucket half - 1
  int start[kMaxB];   // first distance of each bucket, sorted
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
  r.query = (int)q;
  return r;
}

constexpr int kTable = 2048;  // distances whose bucket is looked up rather than searched

// The bucket number of every near distance, in shared memory.
struct Near {
  uint8_t of[kTable];
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
  for (int n = threadIdx.x; n < kTable && n < t.last; n += threads) near.of[n] = (uint8_t)search(t.start, t.half, n);
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

constexpr int kFwdThreads = 256;

// A thread owns one 16-byte vector of a row and writes it for `hc` heads.
// Rows need not be aligned: vectors sit on 16-byte addresses, the ones at a
// row's ends are written element by element.  Masked columns read the
// table's row nb, which holds -inf.
template <class T, class S>
__global__ void __launch_bounds__(kFwdThreads) bias_kernel(const __grid_constant__ Buckets t,
                                                           const __grid_constant__ BiasArgs a,
                                                           const S* __restrict__ table, T* __restrict__ out, int hc,
                                                           int aligned, uint32_t vecs, uint64_t items) {
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Near near;
  T* tab = (T*)smem;                       // [hc][nb + 1]
  const int pitch = a.nb + 1;
  const int h0 = blockIdx.y * hc;
  const int hn = min(hc, a.heads - h0);
  fill_near(near, t, kFwdThreads);
  for (int i = threadIdx.x; i < a.nb * hn; i += kFwdThreads) {
    const int v = i / hn, h = i - v * hn;
    tab[h * pitch + v] = cast<T, S>(table[(size_t)v * a.heads + h0 + h]);
  }
  for (int h = threadIdx.x; h < hn; h += kFwdThreads) tab[h * pitch + a.nb] = minus_infinity<T>();
  __syncthreads();
  const int far_left = t.half - 1, far_right = t.both ? 2 * t.half - 1 : 0;

  for (uint64_t item = (uint64_t)blockIdx.x * kFwdThreads + threadIdx.x; item < items;
       item += (uint64_t)gridDim.x * kFwdThreads) {
    uint64_t row;
    if (items < (1ull << 32)) row = (uint32_t)item / vecs;
    else row = item / vecs;
    const int v = (int)(item - row * vecs);
    const Row r = row_of(t, a, row);
    T* line = out + (int64_t)h0 * a.hs + (int64_t)row * a.rs;
    int which[N];            // the bucket of each of the vector's columns
    bool one;                // whether it is one for all
#define LOOK_UP(c0)                                                                                                      \
  which[0] = (c0) >= r.end ? a.nb : (c0) + N - 1 <= r.left ? far_left : far_right;                                       \
  one = (c0) >= r.end || (c0) + N - 1 <= r.left || ((c0) >= r.right && (c0) + N <= r.end);                               \
  if (!one) {                                                                                                            \
    _Pragma("unroll") for (int k = 0; k < N; k++) {                                                                      \
      const int c = (c0) + k;                                                                                            \
      which[k] = c >= r.end ? a.nb : c <= r.left ? far_left : c >= r.right ? far_right : near_bucket(near, t, r, c);     \
    }                                                                                                                    \
  }
    if (aligned) {           // every head's rows start on a 16-byte boundary: one lookup serves all
      const int c0 = v * N;
      LOOK_UP(c0)
      line += c0;
      if (c0 + N > a.keys) {
        for (int h = 0; h < hn; h++, line += a.hs)
#pragma unroll
          for (int k = 0; k < N; k++)
            if (c0 + k < a.keys) line[k] = tab[h * pitch + (one ? which[0] : which[k])];
      } else if (one) {
        const T* ht = tab + which[0];
#pragma unroll 4
        for (int h = 0; h < hn; h++, line += a.hs, ht += pitch) {
          const T e = *ht;
          Vec<T> x;
#pragma unroll
          for (int k = 0; k < N; k++) x.e[k] = e;
          *(uint4*)line = *(const uint4*)&x;
        }
      } else {
        const T* ht = tab;
#pragma unroll 2
        for (int h = 0; h < hn; h++, line += a.hs, ht += pitch) {
          Vec<T> x;
#pragma unroll
          for (int k = 0; k < N; k++) x.e[k] = ht[which[k]];
          *(uint4*)line = *(const uint4*)&x;
        }
      }
      continue;
    }
    int shift = -1, c0 = 0;  // elements by which this head's rows lie behind a 16-byte boundary
    one = false;
    for (int h = 0; h < hn; h++, line += a.hs) {
      const int s = (int)(((uintptr_t)line / sizeof(T)) % N);
      if (s != shift) {
        shift = s;
        c0 = v * N - s;
        LOOK_UP(c0)
      }
      if (c0 >= a.keys) continue;
      const T* ht = tab + h * pitch;
      Vec<T> x;
#pragma unroll
      for (int k = 0; k < N; k++) x.e[k] = ht[one ? which[0] : which[k]];
      if (c0 >= 0 && c0 + N <= a.keys) {
        *(uint4*)(line + c0) = *(const uint4*)&x;
      } else {
#pragma unroll
        for (int k = 0; k < N; k++)
          if (c0 + k >= 0 && c0 + k < a.keys) line[c0 + k] = x.e[k];
      }
    }
#undef LOOK_UP
  }
}

// ------------------------------------------------------------ gradient

template <class T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

constexpr int kRows = 4;            // rows of a warp's tile (their four loads are in flight together)
constexpr size_t kAccBytes = 48 << 10;

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
// warps, every warp taking items (four rows of one batch entry x `chunk` times
// 32 vectors) in turn.  Fixed by the sizes and strides alone, so sums keep
// their order.
struct GradPlan {
  int warps, splits;
  uint32_t tiles_v, chunk, chunks;
  uint64_t items;
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
  p.tiles_v = d.keys ? (uint32_t)((vectors_of_row(d.keys, n, false) + 31) / 32) : 0;
  const uint64_t groups = (d.queries + kRows - 1) / kRows * d.batch;
  const uint64_t ctas = d.heads ? (uint64_t)(kSms * 3 + d.heads - 1) / d.heads : 1;  // per head: three to an SM
  const uint64_t slots = ctas * p.warps;
  // Whole rows where there are enough of them for every warp, else parts.
  uint64_t cuts = groups ? slots / groups : 1;
  cuts = cuts < 1 ? 1 : cuts > p.tiles_v ? p.tiles_v : cuts;
  p.chunk = cuts ? (uint32_t)((p.tiles_v + cuts - 1) / cuts) : 1;
  p.chunks = p.chunk ? (p.tiles_v + p.chunk - 1) / p.chunk : 0;
  p.items = groups * p.chunks;
  // As few CTAs as take no more turns than the most would.
  const uint64_t turns = (p.items + slots - 1) / slots;
  const uint64_t want = turns ? (p.items + turns * p.warps - 1) / (turns * p.warps) : 1;
  p.splits = (int)(want < 1 ? 1 : want);
  return p;
}

template <class T>
__global__ void __launch_bounds__(256, 3) bias_grad_kernel(const __grid_constant__ Buckets t,
                                                           const __grid_constant__ BiasArgs a, const T* __restrict__ g,
                                                           const __grid_constant__ GradPlan p,
                                                           typename AccOf<T>::type* __restrict__ part,
                                                           typename AccOf<T>::type* __restrict__ dtable, int add) {
  using A = typename AccOf<T>::type;
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  A* acc = (A*)smem;   // [warp][bucket][lane]: every lane adds into its own column, in its own order
  __shared__ Near near;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int threads = p.warps * 32;
  fill_near(near, t, threads);
  for (int i = threadIdx.x; i < p.warps * a.nb * 32; i += threads) acc[i] = 0;
  __syncthreads();
  A* mine = acc + (size_t)warp * a.nb * 32 + lane;

  const int h = blockIdx.y;
  A far_left = 0, far_right = 0;
  const uint64_t warps = (uint64_t)gridDim.x * p.warps, self = (uint64_t)blockIdx.x * p.warps + warp;
  for (uint64_t turn = 0; turn * warps < p.items; turn++) {
    // Forth and back: with a causal mask later rows are longer.
    const uint64_t item = turn * warps + (turn & 1 ? warps - 1 - self : self);
    if (item >= p.items) continue;
    uint64_t group, b;
    uint32_t part_v;
    if (p.items < (1ull << 32)) {
      group = (uint32_t)item / p.chunks;
      part_v = (uint32_t)item - (uint32_t)group * p.chunks;
      const uint32_t batch = (uint32_t)a.batch, g4 = (uint32_t)group / batch;
      b = (uint32_t)group - g4 * batch;
      group = g4;
    } else {
      group = item / p.chunks;
      part_v = (uint32_t)(item - group * p.chunks);
      b = group % a.batch;
      group /= a.batch;
    }
    const uint64_t r0 = group * kRows;
    Row own = {-1, 0, 0, 0};        // of row r0 + lane; no row there: nothing is read
    if (lane < kRows && r0 + lane < a.queries) own = row_of(t, a, r0 + lane);
    const T* line = g + (int64_t)b * a.bs + (int64_t)h * a.hs + (int64_t)r0 * a.rs;
    int left[kRows], right[kRows], end[kRows], shift[kRows];
    int reach = 0;
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      left[r] = __shfl_sync(0xFFFFFFFFu, own.left, r);
      right[r] = __shfl_sync(0xFFFFFFFFu, own.right, r);
      end[r] = __shfl_sync(0xFFFFFFFFu, own.end, r);
      // elements by which the row lies behind a 16-byte boundary
      shift[r] = (int)(((uintptr_t)(line + r * a.rs) / sizeof(T)) % N);
      reach = max(reach, end[r]);
    }
    const uint32_t last = min(p.tiles_v, (part_v + 1) * p.chunk);
    for (uint32_t tv = part_v * p.chunk; tv < last && (int)tv * 32 * N - (N - 1) < reach; tv++) {
      const int v0 = (int)(tv * 32 + lane) * N;
      // Vectors that lie wholly in a far range; the others are noted.
      Vec<T> x[kRows];
      unsigned slow[kRows];
#pragma unroll
      for (int r = 0; r < kRows; r++) {
        const int c = v0 - shift[r];
        if (c >= 0 && c < end[r] && c + N <= a.keys) *(uint4*)&x[r] = __ldg((const uint4*)(line + r * a.rs + c));
      }
#pragma unroll
      for (int r = 0; r < kRows; r++) {
        const int c = v0 - shift[r];
        const bool whole = c >= 0 && c + N <= end[r];
        const bool is_left = whole && c + N - 1 <= left[r], is_right = whole && c >= right[r];
        if (is_left || is_right) {
          A s[N];
#pragma unroll
          for (int k = 0; k < N; k++) s[k] = widen(x[r].e[k]);
#pragma unroll
          for (int u = N / 2; u > 0; u >>= 1)
#pragma unroll
            for (int k = 0; k < u; k++) s[k] += s[k + u];
          if (is_left) far_left += s[0];
          else far_right += s[0];
        }
        slow[r] = __ballot_sync(0xFFFFFFFFu, max(c, 0) < end[r] && !is_left && !is_right);
      }
      // Their elements, one to a lane: near ones each into its bucket.  (One copy
      // of this code: unrolled over rows and vectors, fetching it took longer than
      // running it.)
#pragma unroll 1
      for (int r = 0; r < kRows; r++) {
        unsigned todo = r == 0 ? slow[0] : r == 1 ? slow[1] : r == 2 ? slow[2] : slow[3];
        if (!todo) continue;
        const Row w = {__shfl_sync(0xFFFFFFFFu, own.left, r), __shfl_sync(0xFFFFFFFFu, own.right, r),
                       __shfl_sync(0xFFFFFFFFu, own.end, r), __shfl_sync(0xFFFFFFFFu, own.query, r)};
        const T* at = line + r * a.rs;
        const int base = (int)tv * 32 * N - (int)(((uintptr_t)at / sizeof(T)) % N) + lane;
#pragma unroll 1
        while (todo) {
          const int first = __ffs(todo) - 1, vec = first + lane / N, c = base + first * N;
          const bool here = vec < 32 && (todo >> (vec & 31) & 1) && c >= 0 && c < w.end;
          const unsigned upto = first + 32 / N;
          todo = upto < 32 ? todo >> upto << upto : 0;
          if (!here) continue;
          const A e = widen(__ldg(at + c));
          if (c <= w.left) far_left += e;
          else if (c >= w.right) far_right += e;
          else mine[near_bucket(near, t, w, c) * 32] += e;
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
  return t;
}

template <class T, class S>
int launch_bias_t(const dcf_bias_desc& d, const void* table, const int32_t* pos, void* out, cudaStream_t stream) {
  constexpr uint64_t N = Vec<T>::N;
  const Buckets t = buckets_of(d);
  BiasArgs a = args_of(d, pos);
  a.bs = 0;
  const bool aligned = (uintptr_t)out % 16 == 0 && strides_aligned(a, N);
  const uint64_t vecs = vectors_of_row(d.keys, N, aligned);
  const uint64_t items = vecs * d.queries;
  const uint64_t blocks = (items + kFwdThreads - 1) / kFwdThreads;
  // Heads per block: as many as share the bucket lookup without leaving SMs
  // idle, within 16 KB of table.
  const uint64_t room = (16 << 10) / ((d.num_buckets + 1) * sizeof(T));
  uint64_t hc = blocks >= kSms * 8 ? d.heads : (d.heads * blocks + kSms * 8 - 1) / (kSms * 8);
  if (hc > room) hc = room;
  if (hc < 1) hc = 1;
  uint64_t groups = (d.heads + hc - 1) / hc;
  hc = (d.heads + groups - 1) / groups;
  groups = (d.heads + hc - 1) / hc;
  const size_t smem = hc * (d.num_buckets + 1) * sizeof(T);
  // A block's table and near buckets serve several items.
  const uint64_t most = (kSms * 12 + groups - 1) / groups;
  const dim3 grid((unsigned)(blocks < most ? blocks : most), (unsigned)groups);
  bias_kernel<T, S><<<grid, kFwdThreads, smem, stream>>>(t, a, (const S*)table, (T*)out, (int)hc, aligned, (uint32_t)vecs, items);
  note_launch();
  return cudaPeekAtLastError() == cudaSuccess ? DCF_OK : DCF_ECUDA;
}

template <class T>
int launch_grad_t(const dcf_bias_desc& d, const void* g, const int32_t* pos, void* dtable, void* ws,
                  cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  const Buckets t = buckets_of(d);
  const BiasArgs a = args_of(d, pos);
  GradPlan p = grad_plan(d);
  if ((uintptr_t)g % 16 == 0 && strides_aligned(a, Vec<T>::N))
    p.tiles_v = (uint32_t)((vectors_of_row(d.keys, Vec<T>::N, true) + 31) / 32);
  const int add = (d.flags & DCF_BIAS_ACCUMULATE) != 0;
  const size_t smem = (size_t)p.warps * d.num_buckets * 32 * sizeof(A);
  if (smem > kAccBytes - 4096 &&
      cudaFuncSetAttribute(bias_grad_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 << 10) != cudaSuccess)
    return DCF_ECUDA;
  bias_grad_kernel<T><<<dim3((unsigned)p.splits, d.heads), p.warps * 32, smem, stream>>>(
      t, a, (const T*)g, p, (A*)ws, (A*)dtable, add);
  note_launch();
  if (p.splits > 1) {
    const unsigned entries = d.num_buckets * d.heads;
    bias_grad_join_kernel<A><<<(entries + 7) / 8, 256, 0, stream>>>((const A*)ws, p.splits, a.nb, a.heads, (A*)dtable,
                                                                    add);
    note_launch();
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
  if (d->queries >= lim || d->keys >= lim - 64 || (grad && d->batch >= lim))
    return bad("position bias: queries and batch must be below 2^31, keys below 2^31 - 64");
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
