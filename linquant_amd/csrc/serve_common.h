// Shared pieces of the serving kernels: 16-bit activations of either type, where a packed sequence lies.
#pragma once

#include <type_traits>

#include "lq_common.h"
#include "../../include/linquant_hip.h"

namespace {

typedef __bf16 sv_v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 sv_v2bf __attribute__((ext_vector_type(2)));
typedef uint16_t sv_v8u __attribute__((ext_vector_type(8)));
typedef uint16_t sv_v4u __attribute__((ext_vector_type(4)));

struct F16 {
  static constexpr int code = LQ_DT_F16;
  static LQ_DEV float to(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
  static LQ_DEV uint16_t from(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
struct BF16 {
  static constexpr int code = LQ_DT_BF16;
  static LQ_DEV float to(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
  static LQ_DEV uint16_t from(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }  // to nearest even
};

// one value of a type that is the same for the whole launch
LQ_DEV float sv_load(const void* p, int64_t i, int dtype) {
  if (dtype == LQ_DT_F32) return ((const float*)p)[i];
  const uint16_t u = ((const uint16_t*)p)[i];
  return dtype == LQ_DT_F16 ? F16::to(u) : BF16::to(u);
}

// a * sigmoid(a) on the hardware exp2 / reciprocal units, as the convolution without a state has it
LQ_DEV float sv_silu(float a) { return a * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * -1.44269504088896340736f)); }

// log(1 + exp(v)), accurate where exp(v) is far below one: max(v, 0) + log1p(e) with e = exp(-|v|) <= 1, and
// log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3 (the series' next term is below 2^-29 of the sum).  Once a token and head.
LQ_DEV float sv_softplus(float v) {
  const float e = lq_expf(-__builtin_fabsf(v));
  const float s = e / (2.0f + e), q = s * s;
  float p = 1.0f / 17.0f;
  p = __builtin_fmaf(p, q, 1.0f / 15.0f);
  p = __builtin_fmaf(p, q, 1.0f / 13.0f);
  p = __builtin_fmaf(p, q, 1.0f / 11.0f);
  p = __builtin_fmaf(p, q, 1.0f / 9.0f);
  p = __builtin_fmaf(p, q, 1.0f / 7.0f);
  p = __builtin_fmaf(p, q, 1.0f / 5.0f);
  p = __builtin_fmaf(p, q, 1.0f / 3.0f);
  p = __builtin_fmaf(p, q, 1.0f);
  const float r = fmaxf(v, 0.0f) + 2.0f * s * p;
  return v != v ? v : r;
}

// the step size of a token: softplus of dt + bias where asked for, within [lo, hi]; NaN stays NaN
LQ_DEV float sv_step_size(float raw, float bias, int softplus, float lo, float hi) {
  float d = raw + bias;
  if (softplus) d = sv_softplus(d);
  return d != d ? d : fminf(fmaxf(d, lo), hi);
}

// a log decay: above zero counts as zero; NaN stays NaN
LQ_DEV float sv_decay(float g) { return g != g ? g : fminf(g, 0.0f); }

// What a sequence's slot asks for.  kSlotPad: no state; kSlotBad: out of range, the outputs are NaN.
enum { kSlotPad = -1, kSlotBad = -2 };
LQ_DEV int sv_slot(const int32_t* slots, int seq, int num_slots) {
  const int s = slots ? slots[seq] : seq;
  return s < 0 ? kSlotPad : (s >= num_slots ? kSlotBad : s);
}

// Packed prompts in units of U tokens, each sequence rounded up to whole units: which sequence unit `u` belongs to and which of its
// units it is.  The 64 lanes of a wave look at 64 sequences at a time (one load and a prefix sum over the wave) instead of walking
// the list.  begin, end: the sequence's tokens.  seq < 0: there are fewer units.  Starts that do not ascend or leave [0, tokens]
// describe empty sequences, so that no token out of range is touched.
struct Unit {
  int seq, index, begin, end;
};
template <int U>
LQ_DEV Unit sv_locate(const int32_t* __restrict__ starts, int nseq, int tokens, int u) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < nseq; s0 += 64) {
    const int s = s0 + lane;
    int b = 0, e = 0;
    if (s < nseq) b = starts[s], e = starts[s + 1];
    if (b < 0 || e > tokens || e < b) b = e = 0;
    const int units = (int)(((uint32_t)(e - b) + (U - 1)) / U);
    int sum = units;  // inclusive prefix sum
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(sum, off, 64);
      sum += lane >= off ? o : 0;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (u < before + total) {  // (u is the same for the whole wave)
      const uint64_t m = __ballot(u < before + sum);
      const int l = __builtin_ctzll(m);
      Unit r;
      r.seq = s0 + l;
      r.index = u - (before + __builtin_amdgcn_readlane(sum - units, l));
      r.begin = __builtin_amdgcn_readlane(b, l), r.end = __builtin_amdgcn_readlane(e, l);
      return r;
    }
    before += total;
  }
  return Unit{-1, 0, 0, 0};
}

// 16 bytes a lane from base + offset straight into LDS, at `at` and on, lane after lane (base and at are the same for the wave).  As an
// instruction: where the compiler knows of such a write it waits for all memory operations in front of every LDS access that might be meant,
// the caller's stores among them; so the caller waits for vmcnt itself before it reads.
// (m0 cannot be named as overwritten; nothing else in a kernel that calls this may need it: no __builtin_amdgcn_global_load_lds.)
LQ_DEV void sv_fetch16(const void* base, uint32_t offset, const void* at) {
  typedef const __attribute__((address_space(3))) char lds_char;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_char*)at;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

// 4 bytes a lane likewise
LQ_DEV void sv_fetch4(const void* base, uint32_t offset, const void* at) {
  typedef const __attribute__((address_space(3))) char lds_char;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_char*)at;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

// Matrix results that a loop of run-time length leaves are read behind this.  The vector unit may read a result some cycles after its product
// was issued, which the compiler has to see to; where the last product stands in front of a branch out of the loop it did not (ROCm 7.2: no
// waits in front of the first reads, and old values there).
template <typename V>
LQ_DEV void sv_settle(V& v) { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(v)); }

// whether a grid's first dimension fits a launch (2^32 - 1 threads)
static inline bool sv_fits(int64_t workgroups, int threads) { return workgroups * threads <= 0xffffffffll; }
static inline bool sv_al(const void* q, int n) { return ((uintptr_t)q % n) == 0; }
static inline bool sv_act(int dtype) { return dtype == LQ_DT_F16 || dtype == LQ_DT_BF16; }
static inline bool sv_float(int dtype) { return sv_act(dtype) || dtype == LQ_DT_F32; }
static inline int sv_size(int dtype) { return dtype == LQ_DT_F32 ? 4 : 2; }

}  // namespace
