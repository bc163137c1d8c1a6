// lq_linear_attention_prompt: linear attention over prompts of any lengths, from and into an fp32 state.
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t
// Token by token: four waves share the rows of 64 columns of a head's state.
#include "serve_common.h"

namespace {

struct PromptParams {
  const uint16_t* q;
  int64_t sq_b, sq_l, sq_h;
  const uint16_t* k;
  int64_t sk_b, sk_l, sk_h;
  const uint16_t* v;
  int64_t sv_b, sv_l, sv_h;
  const void* g;
  int64_t sg_b, sg_l, sg_h;
  int g_dtype;
  float scale;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, H, K, V;
};

template <typename T, int KP>
__global__ __launch_bounds__(256) void linear_attention_prompt_kernel(PromptParams p) {
  __shared__ float sums[2][4][64];
  const int seq = blockIdx.x, h = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = blockIdx.z * 64 + (threadIdx.x & 63), cc = min(c, p.V - 1);
  int begin = 0, end = p.seqlen;
  if (p.starts) {
    begin = p.starts[seq], end = p.starts[seq + 1];
    if (begin < 0 || end > p.tokens || end < begin) begin = end = 0;
  }
  if (begin == end) return;
  const int64_t b = p.starts ? 0 : seq, row0 = p.starts ? begin : (int64_t)seq * p.seqlen;
  const int slot = p.state || p.slots ? sv_slot(p.slots, seq, p.num_slots) : kSlotPad;
  const bool keeps = p.state && slot >= 0;
  float S[KP];
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    const int n = wave * KP + i;
    S[i] = slot == kSlotBad ? __builtin_nanf("") : keeps && n < p.K ? p.state[slot * p.ss_s + ((int64_t)h * p.K + n) * p.V + cc] : 0.0f;
  }
  for (int t = 0; t < end - begin; ++t) {
    const int64_t at = (p.starts ? begin : 0) + (int64_t)t;
    const uint16_t *q = p.q + b * p.sq_b + at * p.sq_l + h * p.sq_h, *k = p.k + b * p.sk_b + at * p.sk_l + h * p.sk_h;
    const float v = T::to(p.v[b * p.sv_b + at * p.sv_l + h * p.sv_h + cc]);
    const float decay = p.g ? lq_expf(sv_decay(sv_load(p.g, b * p.sg_b + at * p.sg_l + h * p.sg_h, p.g_dtype))) : 1.0f;
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int n = wave * KP + i;
      if (n < p.K) {
        S[i] = __builtin_fmaf(T::to(k[n]), v, decay * S[i]);
        o = __builtin_fmaf(T::to(q[n]), S[i], o);
      }
    }
    float(*s)[64] = sums[t & 1];
    s[wave][threadIdx.x & 63] = o;
    __syncthreads();
    if (wave == 0 && c < p.V) p.out[((row0 + t) * p.H + h) * p.V + c] = T::from((s[0][threadIdx.x] + s[1][threadIdx.x] + s[2][threadIdx.x] + s[3][threadIdx.x]) * p.scale);
  }
  if (keeps && c < p.V) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int n = wave * KP + i;
      if (n < p.K) p.state[slot * p.ss_s + ((int64_t)h * p.K + n) * p.V + c] = S[i];
    }
  }
}

int check_dims(const lq_linear_attention_prompt_args* a) {
  if (a->nseq <= 0 || a->nheads <= 0 || a->kdim <= 0 || a->kdim % 8 != 0 || a->kdim > 256 || a->vdim <= 0 || a->vdim % 8 != 0) return LQ_ERR_SHAPE;
  if ((a->seq_starts ? a->tokens <= 0 : a->seqlen <= 0) || (int64_t)a->nheads * a->vdim > 1 << 23 || a->nheads > 65535) return LQ_ERR_SHAPE;
  return LQ_OK;
}

}  // namespace

extern "C" int lq_linear_attention_prompt_workspace_bytes(const lq_linear_attention_prompt_args* a, int64_t* bytes) {
  if (!a || !bytes) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc != LQ_OK) return rc;
  *bytes = 0;
  return LQ_OK;
}

extern "C" int lq_linear_attention_prompt(const lq_linear_attention_prompt_args* a, hipStream_t stream) {
  if (!a || !a->q || !a->k || !a->v || !a->out) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc != LQ_OK) return rc;
  if (!sv_act(a->dtype) || (a->g && !sv_float(a->g_dtype)) || (a->state && a->num_slots <= 0)) return LQ_ERR_SHAPE;
  for (const int64_t s : {a->q_stride_l, a->k_stride_l, a->v_stride_l})
    if (s < 0 || s >= 1 << 24) return LQ_ERR_SHAPE;  // a chunk's rows are reached by 32-bit offsets
  for (const int64_t s : {a->q_stride_b, a->q_stride_l, a->q_stride_h, a->k_stride_b, a->k_stride_l, a->k_stride_h, a->v_stride_b, a->v_stride_l, a->v_stride_h})
    if (s % 8 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->q, 16) || !sv_al(a->k, 16) || !sv_al(a->v, 16) || !sv_al(a->out, 16) || !sv_al(a->state, 16) || a->state_stride_s % 4 != 0 ||
      (a->g && !sv_al(a->g, sv_size(a->g_dtype))) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4))
    return LQ_ERR_SHAPE;
  PromptParams p = {(const uint16_t*)a->q, a->q_stride_b, a->q_stride_l, a->q_stride_h, (const uint16_t*)a->k, a->k_stride_b, a->k_stride_l, a->k_stride_h,
                    (const uint16_t*)a->v, a->v_stride_b, a->v_stride_l, a->v_stride_h, a->g, a->g_stride_b, a->g_stride_l, a->g_stride_h, a->g_dtype, a->scale,
                    (uint16_t*)a->out, a->state, a->state_stride_s, a->slots, a->seq_starts, a->num_slots, a->nseq, a->seqlen, a->tokens, a->nheads, a->kdim, a->vdim};
  const dim3 grid((unsigned)a->nseq, (unsigned)a->nheads, (unsigned)((a->vdim + 63) / 64));
  if (!sv_fits(a->nseq, 256) || grid.z > 65535) return LQ_ERR_SHAPE;
  auto go = [&](auto t, auto k) {
    hipLaunchKernelGGL((linear_attention_prompt_kernel<decltype(t), decltype(k)::value>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  auto with = [&](auto t) {
    using std::integral_constant;
    if (a->kdim <= 64) return go(t, integral_constant<int, 16>{});
    if (a->kdim <= 128) return go(t, integral_constant<int, 32>{});
    return go(t, integral_constant<int, 64>{});
  };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
