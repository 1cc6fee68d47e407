// dcf_quant.cuh — how values become 8-bit whole numbers and back, shared by
// the kernels that do either.
//
// With m the largest magnitude beside a value: scale = m / 127, q = the whole
// number nearest x * (127 / m), ties to even.  Adding 1.5 * 2^23 to a value
// below 2^22 rounds it to a whole number, which then stands in the sum's low
// bits; as one fused multiply-add the exact product is rounded once, so a
// quotient on a border goes the same way in every kernel and in 64 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dcf_tensor.cuh"

namespace dcf {

constexpr int kRun = DCF_QUANT_RUN;
constexpr float kLeastMagnitude = 0x1p-119f;  // 127 / m is finite from here on, and m / 127 a normal number
constexpr float kRounder = 12582912.0f;       // 1.5 * 2^23

// Bits of E values of T: one 16-byte vector, or, of rows that are none, a word of two 16-bit values, or a single
// value in the low bits.
template <class T, int E> struct Group {
  static constexpr int kWords = E > 1 ? E * (int)sizeof(T) / 4 : 1;
  uint32_t w[kWords];
};

template <class T> __device__ __forceinline__ uint32_t bits_of(const T* p) {
  if constexpr (sizeof(T) == 4) return *(const uint32_t*)p;
  else return *(const uint16_t*)p;
}

// The first `have` values at p, zeros behind them.
template <class T, int E> __device__ __forceinline__ void load_group(Group<T, E>& g, const T* p, int have) {
  if constexpr (E == 1) {
    g.w[0] = have > 0 ? bits_of(p) : 0;
  } else {
    if (have >= E) {
      if constexpr (E == 2) {
        g.w[0] = *(const uint32_t*)p;
      } else {
        const uint4 v = *(const uint4*)p;
        g.w[0] = v.x, g.w[1] = v.y, g.w[2] = v.z, g.w[3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < Group<T, E>::kWords; j++) g.w[j] = 0;
#pragma unroll
      for (int j = 0; j < E; j++)
        if (j < have) g.w[j * sizeof(T) / 4] |= bits_of(p + j) << (j * sizeof(T) % 4 * 8);
    }
  }
}

// Magnitudes compare as their bits do: NaN above infinity above the rest.  The
// key of a 16-bit type holds two of them.
template <class T> __device__ __forceinline__ uint32_t key_max(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return a > b ? a : b;
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <class T> constexpr uint32_t kMagnitude = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;

template <class T, int E> __device__ __forceinline__ uint32_t group_key(const Group<T, E>& g, uint32_t key) {
#pragma unroll
  for (int j = 0; j < Group<T, E>::kWords; j++) key = key_max<T>(key, g.w[j] & kMagnitude<T>);
  return key;
}

template <class T> __device__ __forceinline__ float value_of(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
  else return __uint_as_float(bits << 16);
}

// The magnitude that a key of one value stands for.
template <class T> __device__ __forceinline__ float key_value(uint32_t key) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(key);
  const uint32_t hi = key >> 16, lo = key & 0xFFFF;
  return value_of<T>(hi > lo ? hi : lo);
}

// What a largest magnitude gives.
struct Scale {
  float scale, factor;  // of q, of x
  uint32_t keep;        // 0 beside a NaN or an infinity: x counts as 0 there
  __device__ __forceinline__ explicit Scale(float m) {
    const bool fine = m < INFINITY, some = m >= kLeastMagnitude;
    scale = !fine ? __uint_as_float(0x7FC00000u) : some ? __fdiv_rn(m, 127.0f) : 0.0f;
    factor = fine && some ? __fdiv_rn(127.0f, m) : 0.0f;
    keep = fine ? 0xFFFFFFFFu : 0u;
  }
};

// x * factor as a whole number in the low byte.
__device__ __forceinline__ uint32_t level(float x, float factor) {
  return __float_as_uint(__fmaf_rn(x, factor, kRounder));
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Bytes of E whole numbers.
template <int E> constexpr int kLevelWords = E > 4 ? 2 : 1;

// E whole numbers from the values that a group and the factors beside them give.
template <int E, class F> __device__ __forceinline__ void pack_levels(uint32_t (&w)[kLevelWords<E>], F at) {
  if constexpr (E == 1) {
    w[0] = at(0);
  } else if constexpr (E == 2) {
    w[0] = __byte_perm(at(0), at(1), 0x0040);
  } else {
#pragma unroll
    for (int j = 0; j < E; j += 4) w[j / 4] = pack4(at(j), at(j + 1), at(j + 2), at(j + 3));
  }
}

// Value j of a group.
template <class T, int E> __device__ __forceinline__ float group_value(const Group<T, E>& g, int j) {
  if constexpr (sizeof(T) == 4 || E == 1) return value_of<T>(g.w[j]);
  else if constexpr (std::is_same<T, __half>::value) return value_of<T>(g.w[j >> 1] >> ((j & 1) * 16) & 0xFFFF);
  else return __uint_as_float(j & 1 ? g.w[j >> 1] & 0xFFFF0000u : g.w[j >> 1] << 16);
}

// The whole numbers of a group, all beside the same largest magnitude.
template <class T, int E>
__device__ __forceinline__ void quantise_group(Group<T, E>& v, const Scale& s, uint32_t (&w)[kLevelWords<E>]) {
#pragma unroll
  for (int j = 0; j < Group<T, E>::kWords; j++) v.w[j] &= s.keep;
  pack_levels<E>(w, [&](int j) { return level(group_value(v, j), s.factor); });
}

// The first `have` bytes of q's words to p, which vectors of E bytes divide.
template <int E> __device__ __forceinline__ void store_levels(int8_t* p, const uint32_t* w, int have) {
  if constexpr (E == 1) {
    if (have > 0) *p = (int8_t)w[0];
  } else {
    if (have >= E) {
      if constexpr (E == 8) *(uint2*)p = make_uint2(w[0], w[1]);
      else if constexpr (E == 4) *(uint32_t*)p = w[0];
      else *(uint16_t*)p = (uint16_t)w[0];
    } else {
#pragma unroll
      for (int j = 0; j < E; j++)
        if (j < have) p[j] = (int8_t)(w[j >> 2] >> ((j & 3) * 8));
    }
  }
}

// Sixteen bytes from byte `off` of two neighbouring vectors on.
__device__ __forceinline__ uint4 bytes_from(const uint4& own, const uint4& next, int off) {
  uint32_t w[8] = {own.x, own.y, own.z, own.w, next.x, next.y, next.z, next.w};
  if (off & 8) {
#pragma unroll
    for (int j = 0; j < 6; j++) w[j] = w[j + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int j = 0; j < 5; j++) w[j] = w[j + 1];
  }
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = __funnelshift_r(w[j], w[j + 1], (off & 3) * 8);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The vector at p (a 16-byte boundary), of which the first `have` bytes (1 to 15) are there, zeros behind them.
__device__ __forceinline__ uint4 first_bytes(const void* at, int have) {
  const uint8_t* p = (const uint8_t*)at;
  const int n8 = have & 8, n4 = have & 4, n2 = have & 2;
  const uint64_t eight = n8 ? *(const uint64_t*)p : 0;
  uint64_t rest = n4 ? *(const uint32_t*)(p + n8) : 0;
  rest |= (uint64_t)(n2 ? *(const uint16_t*)(p + n8 + n4) : 0) << (8 * n4);
  rest |= (uint64_t)(have & 1 ? p[have - 1] : 0) << (8 * (n4 + n2));
  const uint64_t lo = n8 ? eight : rest, hi = n8 ? rest : 0;
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// Sixteen bytes of a row of `bytes` from byte c (a multiple of 16) on, zeros behind its end; the row may start anywhere.
__device__ __forceinline__ uint4 row_bytes(const uint8_t* row, int64_t c, int64_t bytes) {
  const uint8_t* p = row + c;
  const int64_t have = bytes - c;
  if (have >= 16 && (uintptr_t)p % 16 == 0) return *(const uint4*)p;
  const int off = (int)((uintptr_t)p & 3);
  uint32_t w[4] = {0, 0, 0, 0};
  if (have >= 20 && c >= 4) {  // the words around these bytes lie in the row
    const uint32_t* a = (const uint32_t*)(p - off);
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 5; j++) v[j] = a[j];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = __funnelshift_r(v[j], v[j + 1], off * 8);
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (e < have) w[e >> 2] |= (uint32_t)p[e] << ((e & 3) * 8);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Copies rows that no tensor map describes (they start off 16-byte boundaries)
// to rows of whole vectors; sizes and strides in bytes.
int launch_pack_rows(const void* from, int64_t stride, int64_t rows, int64_t bytes, void* to, int64_t to_stride,
                     cudaStream_t s);

// The signed byte j of a word as a float: a byte (its sign turned) under the
// exponent of 2^23 is 2^23 + 128 + q.
__device__ __forceinline__ float byte_value(uint32_t turned, int j) {
  return __fsub_rn(__uint_as_float(__byte_perm(turned, 0x4B000000u, 0x7440 | j)), 8388736.0f);
}

}  // namespace dcf
