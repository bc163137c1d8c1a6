// Rows in registers and their INT8 codes, for the kernels that quantize a row: the residual stream's norm, the quantizer, and the
// quantizer beside low-rank adapters.
#pragma once

#include "serve_common.h"

namespace {

struct F32 {};
template <typename T>
struct Elem {
  using type = uint16_t;
};
template <>
struct Elem<F32> {
  using type = float;
};

// A thread's 8 NV entries of a row: eight adjacent ones at a time (VEC: the row starts on a 16-byte boundary and its length is a multiple
// of 8), else one at a time.  Entries past the row read as zero.
template <typename T, int NV, int TH, bool VEC>
struct Row {
  using E = typename Elem<T>::type;
  static LQ_DEV float one(E u) {
    if constexpr (std::is_same<T, F32>::value) return u;
    else return T::to(u);
  }
  static LQ_DEV void load(const void* base, int64_t at, int dim, int tid, float (&v)[8 * NV]) {
    const E* p = (const E*)base + at;
    if constexpr (VEC) {
      typedef E V8 __attribute__((ext_vector_type(8)));
      V8 raw[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i] = *(const V8*)(p + min((i * TH + tid) * 8, dim - 8));
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * i + e] = (i * TH + tid) * 8 < dim ? one(raw[i][e]) : 0.0f;
    } else {
      E raw[8 * NV];
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) raw[i] = p[min(i * TH + tid, dim - 1)];
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) v[i] = i * TH + tid < dim ? one(raw[i]) : 0.0f;
    }
  }
  static LQ_DEV void store(void* base, int64_t at, int dim, int tid, const float (&v)[8 * NV]) {
    E* p = (E*)base + at;
    auto bits = [](float f) -> E {
      if constexpr (std::is_same<T, F32>::value) return f;
      else return T::from(f);
    };
    if constexpr (VEC) {
      typedef E V8 __attribute__((ext_vector_type(8)));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        V8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = bits(v[8 * i + e]);
        if ((i * TH + tid) * 8 < dim) *(V8*)(p + (i * TH + tid) * 8) = o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i)
        if (i * TH + tid < dim) p[i * TH + tid] = bits(v[i]);
    }
  }
};

// over the threads of a row: a wave's own, or through LDS over the workgroup's four.  `turn` keeps two reductions apart.
template <int TH, typename F>
LQ_DEV float over_row(float v, F op, float* lds, int turn) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
  if constexpr (TH > 64) {
    float* s = lds + turn * (TH / 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < TH / 64; ++w) v = op(v, s[w]);
  }
  return v;
}
LQ_DEV float plus(float a, float b) { return a + b; }
// the larger magnitude by its bits, in which an infinity is above every number and a NaN above that
LQ_DEV float larger(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

// codes clamp(rint(y / s), lo, 127).  y / s correctly rounded: q0 = RN(y (1/s)), rem = y - q0 s exact in one fma, q0 + rem (1/s) rounds
// to the quotient where nothing leaves the normal range; s within 2^-60 .. 2^60 leaves room for that where |y / s| is near the code range,
// and further out only the clamp matters (an infinite or overflowing y keeps q0).
LQ_DEV int code_of(float y, float s, float inv, bool fast, float lo) {
  float q;
  if (fast) {
    const float q0 = y * inv;
    const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, s, y), inv, q0);
    q = q1 == q1 ? q1 : q0;
  } else {
    q = y / s;
  }
  return (int)fminf(fmaxf(__builtin_rintf(q), lo), 127.0f);
}

template <int NV, int TH, bool VEC>
LQ_DEV void store_codes(int8_t* base, int64_t at, int dim, int tid, const float (&y)[8 * NV], float s, float lo) {
  const float as = __builtin_fabsf(s);
  const bool fast = as > 0x1p-60f && as < 0x1p60f;
  const float inv = 1.0f / s;
  int8_t* p = base + at;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = code_of(y[8 * i + e], s, inv, fast, lo);
    if constexpr (VEC) {
      const lq_v2i o = {(int)lq_pack4(c[0], c[1], c[2], c[3]), (int)lq_pack4(c[4], c[5], c[6], c[7])};
      if ((i * TH + tid) * 8 < dim) *(lq_v2i*)(p + (i * TH + tid) * 8) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((i * 8 + e) * TH + tid < dim) p[(i * 8 + e) * TH + tid] = (int8_t)c[e];
    }
  }
}

// codes on the row's own scale; the thread that is the row's first stores it.  A row of zeros: 0 and codes 0; one with an infinity or
// a NaN: NaN and codes 0.
template <int NV, int TH, bool VEC>
LQ_DEV void row_codes(float* scale, int8_t* codes, int64_t at, int dim, int tid, const float (&y)[8 * NV], float* lds, int turn) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) m = larger(m, __builtin_fabsf(y[i]));
  m = over_row<TH>(m, larger, lds, turn);
  const bool finite = __float_as_uint(m) < 0x7f800000u;
  const float s = finite ? m / 127.0f : __uint_as_float(0x7fc00000u);
  if (tid == 0) *scale = s;
  float z[8 * NV];
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) z[i] = finite && s > 0.0f ? y[i] : 0.0f;
  store_codes<NV, TH, VEC>(codes, at, dim, tid, z, finite && s > 0.0f ? s : 1.0f, -127.0f);
}

}  // namespace
