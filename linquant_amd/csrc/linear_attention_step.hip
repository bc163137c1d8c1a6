// lq_linear_attention_step: one token of each sequence through linear attention, the fp32 state updated in place.
//   S = exp(g) S + k v^T,  o = scale S^T q
// HBM-bound: 8 bytes for each entry of the state, five operations.
//
// A group of lanes has one row of the state's columns in pieces of 16 bytes, so that a wave's request covers whole 128-byte lines; each
// thread keeps its columns' sums over its rows, and the rows' sums meet in LDS at the end.  Where sequences times heads are few, a head's
// columns are cut into blocks of 32, a workgroup each.
//
// 256 sequences of 32 heads of 128 by 128: 211 us, 5.1 TB/s, the rate of a copy.  4 of 16 heads, 8 MB: 4.9 us, 2 of them the launch, then two
// round trips to memory, one for the slot and one for the rest.
#include "serve_common.h"

namespace {

struct StepParams {
  const uint16_t* q;
  int64_t sq_b, sq_h;
  const uint16_t* k;
  int64_t sk_b, sk_h;
  const uint16_t* v;
  int64_t sv_b, sv_h;
  const void* g;
  int64_t sg_b, sg_h;
  int g_dtype;
  float scale;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  int num_slots, H, K, V;
};

constexpr int kThreads = 256, kMaxK = 256;

// LR lanes to a row of the block's 4 LR columns, U rows of a thread requested at a time
template <typename T, int LR, int U>
__global__ __launch_bounds__(kThreads) void linear_attention_step_kernel(StepParams p) {
  constexpr int R = kThreads / LR;  // rows of a pass
  __shared__ __align__(16) float qk[2][kMaxK];
  __shared__ __align__(16) lq_v4f sums[kThreads / 64][LR];
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y, c0 = blockIdx.z * 4 * LR;
  const int slot = sv_slot(p.slots, b, p.num_slots);
  uint16_t* op = p.out + ((int64_t)b * p.H + h) * p.V;
  if (slot < 0) {
    const uint16_t x = slot == kSlotBad ? T::from(__builtin_nanf("")) : 0;
    for (int i = c0 + tid; i < min(c0 + 4 * LR, p.V); i += kThreads) op[i] = x;
    return;
  }
  const int c = c0 + 4 * (tid % LR), r0 = tid / LR, cc = min(c, p.V - 4);
  float* S = p.state + slot * p.ss_s + (int64_t)h * p.K * p.V;
  lq_v4f s[U];
  auto request = [&](int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = *(const lq_v4f*)(S + (int64_t)min(at + R * u + r0, p.K - 1) * p.V + cc);
  };
  request(0);
  const sv_v4u v4 = *(const sv_v4u*)(p.v + b * p.sv_b + h * p.sv_h + cc);
  float decay = 1.0f;
  if (p.g) decay = lq_expf(sv_decay(sv_load(p.g, b * p.sg_b + h * p.sg_h, p.g_dtype)));
  if (tid < p.K) {
    qk[0][tid] = T::to(p.q[b * p.sq_b + h * p.sq_h + tid]) * p.scale;
    qk[1][tid] = T::to(p.k[b * p.sk_b + h * p.sk_h + tid]);
  }
  __syncthreads();
  float v[4];
  lq_v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = T::to(v4[e]);
  for (int at = 0; at < p.K; at += R * U) {
    if (at) request(at);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = at + R * u + r0;
      if (row < p.K && c < p.V) {  // (a lane behind the row or the head has another's entries, which are not its own to add)
        const float qr = qk[0][row], kr = qk[1][row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][e] = __builtin_fmaf(kr, v[e], decay * s[u][e]);
          o[e] = __builtin_fmaf(qr, s[u][e], o[e]);
        }
        *(lq_v4f*)(S + (int64_t)row * p.V + c) = s[u];
      }
    }
  }
#pragma unroll
  for (int off = LR; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off, 64);
  if ((tid & 63) < LR) sums[tid >> 6][tid & 63] = o;
  __syncthreads();
  if (tid < LR && c < p.V) {
    sv_v4u y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = T::from(sums[0][tid][e] + sums[1][tid][e] + sums[2][tid][e] + sums[3][tid][e]);
    *(sv_v4u*)(op + c) = y;
  }
}

}  // namespace

extern "C" int lq_linear_attention_step(const lq_linear_attention_step_args* a, hipStream_t stream) {
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->state) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || (a->g && !sv_float(a->g_dtype)) || a->batch <= 0 || a->batch > 65535 || a->nheads <= 0 || a->num_slots <= 0) return LQ_ERR_SHAPE;
  if (a->kdim <= 0 || a->kdim > kMaxK || a->vdim <= 0 || a->vdim % 4 != 0 || !sv_fits(a->nheads, kThreads)) return LQ_ERR_SHAPE;
  if ((int64_t)a->nheads * a->vdim > 0x7fffffff || a->v_stride_b % 4 != 0 || a->v_stride_h % 4 != 0 || a->state_stride_s % 4 != 0) return LQ_ERR_SHAPE;
  if (a->num_slots > 1 && a->state_stride_s < (int64_t)a->nheads * a->kdim * a->vdim) return LQ_ERR_SHAPE;  // slots that overlap
  if (!sv_al(a->q, 2) || !sv_al(a->k, 2) || !sv_al(a->v, 8) || !sv_al(a->out, 8) || !sv_al(a->state, 16) || !sv_al(a->slots, 4) ||
      (a->g && !sv_al(a->g, sv_size(a->g_dtype))))
    return LQ_ERR_SHAPE;
  StepParams p = {(const uint16_t*)a->q, a->q_stride_b, a->q_stride_h, (const uint16_t*)a->k, a->k_stride_b, a->k_stride_h, (const uint16_t*)a->v,
                  a->v_stride_b, a->v_stride_h, a->g, a->g_stride_b, a->g_stride_h, a->g_dtype, a->scale, (uint16_t*)a->out, a->state,
                  a->state_stride_s, a->slots, a->num_slots, a->nheads, a->kdim, a->vdim};
  auto go = [&](auto t, auto lr) {
    constexpr int LR = decltype(lr)::value;
    const int64_t blocks = ((int64_t)a->vdim + 4 * LR - 1) / (4 * LR);
    if (blocks > 65535) return (int)LQ_ERR_SHAPE;
    const dim3 grid((unsigned)a->nheads, (unsigned)a->batch, (unsigned)blocks);
    hipLaunchKernelGGL((linear_attention_step_kernel<decltype(t), LR, LR == 8 ? 4 : 16>), grid, dim3(kThreads), 0, stream, p);
    return lq_check_launch();
  };
  auto with = [&](auto t) {
    using std::integral_constant;
    if (a->vdim <= 32 || (int64_t)a->nheads * a->batch < 512) return go(t, integral_constant<int, 8>{});
    if (a->vdim <= 64) return go(t, integral_constant<int, 16>{});
    if (a->vdim <= 128) return go(t, integral_constant<int, 32>{});
    return go(t, integral_constant<int, 64>{});
  };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
