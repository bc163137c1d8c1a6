// The short causal depthwise convolution (+ SiLU) with the inputs in front of a call kept in a state.
//   lq_conv1d_prompt   prompts of any lengths (packed, or a batch of one length)
//   lq_conv1d_step     one token of each sequence
//   y[t, c] = act(bias[c] + sum_j weight[c, j] * x[t - (W-1) + j, c]), fp32, taps in order j = 0 .. W-1
// HBM-bound streaming, 16 bytes a lane.  10,021 tokens of ten ragged prompts, 5376 channels, fp16: 48 us, 4.5 TB/s of what has to move (a
// large copy reaches 5.1); 64 single tokens: 3.4 us, a launch and one round trip to memory.
#include "serve_common.h"

namespace {

struct ConvParams {
  const uint16_t* x;
  int64_t sx_b, sx_l;
  const uint16_t* weight;
  const uint16_t* bias;
  uint16_t* out;
  uint16_t* state;
  int64_t ss_s, ss_w;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, dim;
};

template <typename T, int W>
LQ_DEV void load_taps(const ConvParams& p, int c, float (&w)[W][8], float (&bv)[8]) {
  sv_v8u wraw[W];
#pragma unroll
  for (int j = 0; j < W; ++j) wraw[j] = *(const sv_v8u*)(p.weight + (int64_t)c * W + 8 * j);
  const sv_v8u braw = *(const sv_v8u*)(p.bias ? p.bias + c : p.weight + (int64_t)c * W);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    bv[e] = p.bias ? T::to(braw[e]) : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = T::to(wraw[(e * W + j) >> 3][(e * W + j) & 7]);  // weight[(c + e) * W + j]
  }
}

// Tokens a thread computes; the W-1 rows in front of them are read again (from the caches).  us with 4 / 8 / 16 / 32: 10,021 ragged tokens 53 / 48
// / 51 / 57, 4 prompts of 8192 150 / 139 / 141, one of 512 6.1 / 5.8 / 7.8.
constexpr int kTL = 8;

// A wave has kTL tokens of one sequence and 512 channels.  The wave with a sequence's first tokens is the only one that looks at its state:
// it reads what lies in front of the prompt, then writes the last W-1 inputs, so no other wave can see the new state for the old.
template <typename T, int W, bool SILU>
__global__ __launch_bounds__(256) void conv1d_prompt_kernel(ConvParams p) {
  const int cg = (blockIdx.y * 4 + (threadIdx.x >> 6)) * 64 + (threadIdx.x & 63);
  Unit u;
  const uint16_t* xb = p.x;
  uint16_t* ob = p.out;
  if (p.starts) {
    u = sv_locate<kTL>(p.starts, p.nseq, p.tokens, blockIdx.x);
    if (u.seq < 0) return;
  } else {
    const int per = (p.seqlen + kTL - 1) / kTL;
    u.seq = blockIdx.x / per, u.index = blockIdx.x - u.seq * per, u.begin = 0, u.end = p.seqlen;
    xb += u.seq * p.sx_b, ob += (int64_t)u.seq * p.seqlen * p.dim;
  }
  const int c = cg * 8;
  if (c >= p.dim) return;
  const int L = u.end - u.begin, t0 = u.index * kTL;
  const uint16_t* xs = xb + (int64_t)u.begin * p.sx_l + c;  // the sequence's first token
  const int slot = p.state || p.slots ? sv_slot(p.slots, u.seq, p.num_slots) : kSlotPad;
  const bool keeps = p.state && slot >= 0;
  uint16_t* st = keeps ? p.state + slot * p.ss_s + c : nullptr;
  sv_v8u rows[kTL + W - 1];  // rows[i]: token t0 - (W-1) + i
#pragma unroll
  for (int i = 0; i < kTL + W - 1; ++i) rows[i] = *(const sv_v8u*)(xs + (int64_t)min(max(t0 - (W - 1) + i, 0), L - 1) * p.sx_l);
  float w[W][8], bv[8];
  load_taps<T, W>(p, c, w, bv);
  if (t0 == 0) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      rows[i] = sv_v8u{0, 0, 0, 0, 0, 0, 0, 0};
      if (keeps) rows[i] = *(const sv_v8u*)(st + i * p.ss_w);
    }
    if (keeps) {
      sv_v8u last[W - 1];
#pragma unroll
      for (int i = 0; i < W - 1; ++i) {
        const int t = L - (W - 1) + i;  // below 0: what was in front of the prompt
        if (t >= 0) last[i] = *(const sv_v8u*)(xs + (int64_t)t * p.sx_l);
        else last[i] = *(const sv_v8u*)(st + (t + W - 1) * p.ss_w);
      }
#pragma unroll
      for (int i = 0; i < W - 1; ++i) *(sv_v8u*)(st + i * p.ss_w) = last[i];
    }
  }
  float win[W][8];
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) win[j + 1][e] = T::to(rows[j][e]);
  uint16_t* op = ob + ((int64_t)u.begin + t0) * p.dim + c;
  const float bad = slot == kSlotBad ? __builtin_nanf("") : 0.0f;
#pragma unroll
  for (int i = 0; i < kTL; ++i) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) win[j][e] = win[j + 1][e];
    sv_v8u o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      win[W - 1][e] = T::to(rows[W - 1 + i][e]);
      float a = bv[e];
#pragma unroll
      for (int j = 0; j < W; ++j) a = a + w[j][e] * win[j][e];
      if constexpr (SILU) a = sv_silu(a);
      o[e] = T::from(a + bad);
    }
    if (t0 + i < L) __builtin_nontemporal_store(o, (sv_v8u*)op);
    op += p.dim;
  }
}

template <typename T, int W, bool SILU>
__global__ __launch_bounds__(64) void conv1d_step_kernel(ConvParams p) {
  const int b = blockIdx.x, c = (blockIdx.y * 64 + threadIdx.x) * 8;
  if (c >= p.dim) return;
  const int slot = sv_slot(p.slots, b, p.num_slots);
  uint16_t* op = p.out + (int64_t)b * p.dim + c;
  if (slot < 0) {
    const uint16_t v = slot == kSlotBad ? T::from(__builtin_nanf("")) : 0;
    *(sv_v8u*)op = sv_v8u{v, v, v, v, v, v, v, v};
    return;
  }
  uint16_t* st = p.state + slot * p.ss_s + c;
  sv_v8u rows[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) rows[j] = *(const sv_v8u*)(st + j * p.ss_w);
  rows[W - 1] = *(const sv_v8u*)(p.x + b * p.sx_b + c);
  float w[W][8], bv[8];
  load_taps<T, W>(p, c, w, bv);
  sv_v8u o;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float a = bv[e];
#pragma unroll
    for (int j = 0; j < W; ++j) a = a + w[j][e] * T::to(rows[j][e]);
    if constexpr (SILU) a = sv_silu(a);
    o[e] = T::from(a);
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) *(sv_v8u*)(st + j * p.ss_w) = rows[j + 1];
  *(sv_v8u*)op = o;
}

// the kernel of a call's type, width and activation
template <typename F>
int for_form(int dtype, int width, int silu, F f) {
  auto with = [&](auto t) {
    auto wide = [&](auto w) { return silu ? f(t, w, std::true_type{}) : f(t, w, std::false_type{}); };
    if (width == 2) return wide(std::integral_constant<int, 2>{});
    if (width == 3) return wide(std::integral_constant<int, 3>{});
    return wide(std::integral_constant<int, 4>{});
  };
  return dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}

}  // namespace

extern "C" int lq_conv1d_prompt(const lq_conv1d_prompt_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->weight || !a->out) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || a->dim <= 0 || a->dim % 8 != 0 || a->width < 2 || a->width > 4 || a->nseq <= 0) return LQ_ERR_SHAPE;
  if (a->seq_starts ? a->tokens <= 0 : a->seqlen <= 0) return LQ_ERR_SHAPE;
  if (a->x_stride_l % 8 != 0 || (!a->seq_starts && a->x_stride_b % 8 != 0) || !sv_al(a->x, 16) || !sv_al(a->out, 16)) return LQ_ERR_SHAPE;
  if (!sv_al(a->weight, 16) || !sv_al(a->bias, 16) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4)) return LQ_ERR_SHAPE;
  if (a->state && (!sv_al(a->state, 16) || a->state_stride_s % 8 != 0 || a->state_stride_w % 8 != 0 || a->num_slots <= 0)) return LQ_ERR_SHAPE;
  // every sequence is rounded up to whole units, so a packed call has at most so many; the surplus ends at once
  const int64_t units = a->seq_starts ? (int64_t)a->tokens / kTL + a->nseq : (int64_t)a->nseq * (((int64_t)a->seqlen + kTL - 1) / kTL), groups = ((int64_t)a->dim + 2047) / 2048;
  if (!sv_fits(units, 256) || groups > 65535) return LQ_ERR_SHAPE;
  ConvParams p = {(const uint16_t*)a->x, a->x_stride_b, a->x_stride_l, (const uint16_t*)a->weight, (const uint16_t*)a->bias, (uint16_t*)a->out,
                  (uint16_t*)a->state, a->state_stride_s, a->state_stride_w, a->slots, a->seq_starts, a->num_slots, a->nseq, a->seqlen, a->tokens, a->dim};
  const dim3 grid((unsigned)units, (unsigned)groups);
  return for_form(a->dtype, a->width, a->silu, [&](auto t, auto w, auto s) {
    hipLaunchKernelGGL((conv1d_prompt_kernel<decltype(t), decltype(w)::value, decltype(s)::value>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  });
}

extern "C" int lq_conv1d_step(const lq_conv1d_step_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->weight || !a->out || !a->state) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || a->dim <= 0 || a->dim % 8 != 0 || a->width < 2 || a->width > 4 || a->batch <= 0 || a->num_slots <= 0) return LQ_ERR_SHAPE;
  if (a->x_stride % 8 != 0 || !sv_al(a->x, 16) || !sv_al(a->out, 16) || !sv_al(a->weight, 16) || !sv_al(a->bias, 16) || !sv_al(a->slots, 4)) return LQ_ERR_SHAPE;
  if (!sv_al(a->state, 16) || a->state_stride_s % 8 != 0 || a->state_stride_w % 8 != 0) return LQ_ERR_SHAPE;
  const int64_t parts = ((int64_t)a->dim + 511) / 512;
  if (parts > 65535 || !sv_fits(a->batch, 64)) return LQ_ERR_SHAPE;
  ConvParams p = {(const uint16_t*)a->x, a->x_stride, 0, (const uint16_t*)a->weight, (const uint16_t*)a->bias, (uint16_t*)a->out, (uint16_t*)a->state,
                  a->state_stride_s, a->state_stride_w, a->slots, nullptr, a->num_slots, a->batch, 1, 0, a->dim};
  return for_form(a->dtype, a->width, a->silu, [&](auto t, auto w, auto s) {
    hipLaunchKernelGGL((conv1d_step_kernel<decltype(t), decltype(w)::value, decltype(s)::value>), dim3((unsigned)a->batch, (unsigned)parts), dim3(64), 0, stream, p);
    return lq_check_launch();
  });
}
