// lq_ssm_prompt: the selective state space scan over prompts of any lengths, from and into an fp32 state.
//   S = exp(d A) S + d x B^T,  y = S C + D x,  d = softplus(dt + bias)
// Token by token, eight lanes to a row of the state, as in the single-token kernel.
#include "serve_common.h"

namespace {

struct PromptParams {
  const uint16_t* x;
  int64_t sx_b, sx_l, sx_h;
  const void* dt;
  int64_t sdt_b, sdt_l, sdt_h;
  int dt_dtype;
  const float* A;
  const uint16_t* B;
  int64_t sB_b, sB_l, sB_g;
  const uint16_t* C;
  int64_t sC_b, sC_l, sC_g;
  const float* D;
  int D_has_hdim;
  const float* dt_bias;
  int softplus;
  float dt_min, dt_max;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, H, P, G, N;
};

template <typename T, int KN>
__global__ __launch_bounds__(256) void ssm_prompt_kernel(PromptParams p) {
  const int h = blockIdx.x, seq = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & 7;
  const int row = blockIdx.z * 32 + 8 * wave + (lane >> 3);
  int t0 = 0, L = p.seqlen;
  int64_t ob = (int64_t)seq * p.seqlen;
  const int64_t b = p.starts ? 0 : seq;
  if (p.starts) {
    t0 = p.starts[seq];
    const int t1 = p.starts[seq + 1];
    L = t0 < 0 || t1 > p.tokens || t1 < t0 ? 0 : t1 - t0;
    ob = t0;
  }
  if (row >= p.P || L == 0) return;
  const int slot = p.state || p.slots ? sv_slot(p.slots, seq, p.num_slots) : kSlotPad;
  const bool keeps = p.state && slot >= 0;
  const int g = h / (p.H / p.G);
  float* S = keeps ? p.state + slot * p.ss_s + ((int64_t)h * p.P + row) * p.N : nullptr;
  lq_v4f s[KN];
#pragma unroll
  for (int k = 0; k < KN; ++k) {
    s[k] = lq_v4f{0.f, 0.f, 0.f, 0.f};
    if (keeps) s[k] = *(const lq_v4f*)(S + min(32 * k + 4 * sub, p.N - 4));
  }
  const float A = p.A[h], bias = p.dt_bias ? p.dt_bias[h] : 0.0f, D = p.D ? p.D[p.D_has_hdim ? h * p.P + row : h] : 0.0f;
  for (int i = 0; i < L; ++i) {
    const int64_t t = t0 + i;
    const float d = sv_step_size(sv_load(p.dt, b * p.sdt_b + t * p.sdt_l + h * p.sdt_h, p.dt_dtype), bias, p.softplus, p.dt_min, p.dt_max);
    const float decay = lq_expf(d * A);
    const float xv = T::to(p.x[b * p.sx_b + t * p.sx_l + h * p.sx_h + row]), dx = d * xv;
    const uint16_t* Bp = p.B + b * p.sB_b + t * p.sB_l + g * p.sB_g;
    const uint16_t* Cp = p.C + b * p.sC_b + t * p.sC_l + g * p.sC_g;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < KN; ++k) {
      const int n = 32 * k + 4 * sub, at = min(n, p.N - 4);
      const sv_v4u rb = *(const sv_v4u*)(Bp + at), rc = *(const sv_v4u*)(Cp + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[k][e] = __builtin_fmaf(dx, T::to(rb[e]), decay * s[k][e]);
        y += n < p.N ? s[k][e] * T::to(rc[e]) : 0.0f;
      }
    }
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) y += __shfl_xor(y, off, 64);
    y = __builtin_fmaf(D, xv, y);
    if (slot == kSlotBad) y = __builtin_nanf("");
    if (sub == 0) p.out[((ob + i) * p.H + h) * p.P + row] = T::from(y);
  }
  if (keeps) {
#pragma unroll
    for (int k = 0; k < KN; ++k)
      if (32 * k + 4 * sub < p.N) *(lq_v4f*)(S + 32 * k + 4 * sub) = s[k];
  }
}

int check_dims(const lq_ssm_prompt_args* a) {
  if (a->nseq <= 0 || a->nseq > 65535 || a->nheads <= 0 || a->ngroups <= 0 || a->nheads % a->ngroups != 0) return LQ_ERR_SHAPE;
  if (a->headdim <= 0 || a->headdim % 8 != 0 || a->dstate <= 0 || a->dstate % 8 != 0 || a->dstate > 256) return LQ_ERR_SHAPE;
  if (a->seq_starts ? a->tokens <= 0 : a->seqlen <= 0) return LQ_ERR_SHAPE;
  return LQ_OK;
}

}  // namespace

extern "C" int lq_ssm_prompt_workspace_bytes(const lq_ssm_prompt_args* a, int64_t* bytes) {
  if (!a || !bytes) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc == LQ_OK) *bytes = 0;
  return rc;
}

extern "C" int lq_ssm_prompt(const lq_ssm_prompt_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->dt || !a->A || !a->B || !a->C || !a->out) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc != LQ_OK) return rc;
  if (!sv_act(a->dtype) || !sv_float(a->dt_dtype) || (a->state && a->num_slots <= 0)) return LQ_ERR_SHAPE;
  for (const int64_t s : {a->B_stride_b, a->B_stride_l, a->B_stride_g, a->C_stride_b, a->C_stride_l, a->C_stride_g})
    if (s % 8 != 0) return LQ_ERR_SHAPE;
  if (a->x_stride_b % 8 != 0 || a->x_stride_l % 8 != 0 || a->x_stride_h % 8 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->x, 16) || !sv_al(a->B, 16) || !sv_al(a->C, 16) || !sv_al(a->out, 16) || !sv_al(a->state, 16) || a->state_stride_s % 4 != 0 ||
      !sv_al(a->dt, sv_size(a->dt_dtype)) || !sv_al(a->A, 4) || !sv_al(a->D, 4) || !sv_al(a->dt_bias, 4) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4))
    return LQ_ERR_SHAPE;
  PromptParams p = {(const uint16_t*)a->x, a->x_stride_b, a->x_stride_l, a->x_stride_h, a->dt, a->dt_stride_b, a->dt_stride_l, a->dt_stride_h, a->dt_dtype, a->A,
                    (const uint16_t*)a->B, a->B_stride_b, a->B_stride_l, a->B_stride_g, (const uint16_t*)a->C, a->C_stride_b, a->C_stride_l, a->C_stride_g,
                    a->D, a->D_has_hdim, a->dt_bias, a->dt_softplus, a->dt_min, a->dt_max, (uint16_t*)a->out, a->state, a->state_stride_s, a->slots,
                    a->seq_starts, a->num_slots, a->nseq, a->seqlen, a->tokens, a->nheads, a->headdim, a->ngroups, a->dstate};
  const dim3 grid((unsigned)a->nheads, (unsigned)a->nseq, (unsigned)((a->headdim + 31) / 32));
  auto go = [&](auto t, auto k) {
    hipLaunchKernelGGL((ssm_prompt_kernel<decltype(t), decltype(k)::value>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  auto with = [&](auto t) {
    if (a->dstate <= 32) return go(t, std::integral_constant<int, 1>{});
    if (a->dstate <= 64) return go(t, std::integral_constant<int, 2>{});
    if (a->dstate <= 128) return go(t, std::integral_constant<int, 4>{});
    return go(t, std::integral_constant<int, 8>{});
  };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
