// pz_rowvec.cuh — a row of logits as 16-byte vectors, whatever its address.
//
// Rows start anywhere (ld may be odd), so vectors are counted from the last
// 16-byte boundary at or before the row: `shift` elements before column 0.
// Vector k covers the columns [k*N - shift, k*N - shift + N); the first and
// the last may reach outside the row, and those columns are read and
// written one element at a time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace pz {

// Two fp32 values in one 64-bit register: sm_100 adds and multiplies both in
// one instruction.  A product that feeds a sum may be joined with it into one
// rounding: where two roundings are the definition, take scalars.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 p, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The larger of two values, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct bf16_t {  // a bf16 element as it lies in memory
  uint16_t bits;
};

template <typename T>
struct RowElem;

template <>
struct RowElem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const float *p) { return *p; }
  static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4 &u, float *x) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float *x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ void pairs(const uint4 &u, f32x2 *p) {
    p[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
    p[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack_pairs(const f32x2 *p) {
    float x[4];
    unpair(p[0], x[0], x[1]);
    unpair(p[1], x[2], x[3]);
    return pack(x);
  }
  static __device__ __forceinline__ float max(const uint4 &u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  // the largest magnitude, NaN where any value is
  static __device__ __forceinline__ float max_abs_nan(const uint4 &u) {
    return max_nan(max_nan(fabsf(__uint_as_float(u.x)), fabsf(__uint_as_float(u.y))),
                   max_nan(fabsf(__uint_as_float(u.z)), fabsf(__uint_as_float(u.w))));
  }
  // the elements whose bit is set, -inf for the others
  static __device__ __forceinline__ uint4 keep(const uint4 &u, uint32_t bits) {
    return make_uint4((bits & 1u) ? u.x : kNegInf2, (bits & 2u) ? u.y : kNegInf2, (bits & 4u) ? u.z : kNegInf2,
                      (bits & 8u) ? u.w : kNegInf2);
  }
  static constexpr uint32_t kNegInf2 = 0xFF800000u;  // what a 32-bit word of -inf holds
};

template <>
struct RowElem<bf16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const bf16_t *p) {
    return __uint_as_float(static_cast<uint32_t>(p->bits) << 16);
  }
  // one rounding to nearest even, the output's type being bf16
  static __device__ __forceinline__ void put(bf16_t *p, float v) {
    p->bits = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
  static __device__ __forceinline__ void unpack(const uint4 &u, float *x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ uint4 pack(const float *x) {
    return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
  }
  static __device__ __forceinline__ void pairs(const uint4 &u, f32x2 *p) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint4 pack_pairs(const f32x2 *p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float lo, hi;
      unpair(p[j], lo, hi);
      w[j] = pack2(lo, hi);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the largest value that is not NaN (NaN where all are), two at a time
  static __device__ __forceinline__ float max(const uint4 &u) {
    const __nv_bfloat162 *v = reinterpret_cast<const __nv_bfloat162 *>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float max_abs_nan(const uint4 &u) {
    const __nv_bfloat162 *v = reinterpret_cast<const __nv_bfloat162 *>(&u);
    const __nv_bfloat162 m =
        __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
    return max_nan(__low2float(m), __high2float(m));
  }
  // Selectors of a byte permutation for four elements: 0x54 and 0x76 take the
  // two bytes of an element from the second operand, 0x10 and 0x32 (0x44
  // less) from the first.  The product spreads four bits over four bytes.
  static __device__ __forceinline__ uint32_t selectors(uint32_t bits) {
    return 0x76547654u - (((bits & 0xFu) * 0x00204081u) & 0x01010101u) * 0x44u;
  }
  static __device__ __forceinline__ uint4 keep(const uint4 &u, uint32_t bits) {
    const uint32_t lo = selectors(bits), hi = selectors(bits >> 4);
    return make_uint4(__byte_perm(u.x, kNegInf2, lo), __byte_perm(u.y, kNegInf2, lo >> 16),
                      __byte_perm(u.z, kNegInf2, hi), __byte_perm(u.w, kNegInf2, hi >> 16));
  }
  static constexpr uint32_t kNegInf2 = 0xFF80FF80u;
};

// Elements between the last 16-byte boundary at or before p and p.
template <typename T>
__device__ __forceinline__ int row_shift(const T *p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

// Streaming 16-byte load (read once: not kept in L1) and store.
__device__ __forceinline__ uint4 load16(const void *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void store16(void *p, const uint4 &v) {
  __stcs(reinterpret_cast<uint4 *>(p), v);
}
// A store of what is written again soon: it stays in L2.
__device__ __forceinline__ void store16_keep(void *p, const uint4 &v) { *reinterpret_cast<uint4 *>(p) = v; }

// Vectors [first, last) of a row lie in it whole.
struct WholeVecs {
  int first, last;
};
template <typename T>
__device__ __forceinline__ WholeVecs whole_vecs(int shift, int V) {
  return WholeVecs{shift > 0 ? 1 : 0, (V + shift) / RowElem<T>::N};
}

// Columns [c, c + N) that reach outside the row, those outside as `fill`.  Out
// of line: at most two vectors of a row take this way.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T *row, int V, int c, float fill = -INFINITY) {
  constexpr int N = RowElem<T>::N;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; j++)
    x[j] = (c + j >= 0 && c + j < V) ? RowElem<T>::get(row + c + j) : fill;
  return RowElem<T>::pack(x);
}
// A packed vector to the columns [c, c + N) of a row, those inside [0, V).
template <typename T>
__device__ __noinline__ void store_edge(T *row, int V, int c, uint4 v) {
  constexpr int N = RowElem<T>::N;
  float x[N];
  RowElem<T>::unpack(v, x);
#pragma unroll
  for (int j = 0; j < N; j++)
    if (c + j >= 0 && c + j < V) RowElem<T>::put(row + c + j, x[j]);
}

}  // namespace pz
