// lq_ssm_step: one token of each sequence through the selective state space scan, the fp32 state updated in place.
//   S = exp(d A) S + d x B^T,  y = S C + D x,  d = softplus(dt + bias)
// HBM-bound: 8 bytes for each entry of the state, five operations.  80 heads of 64 by 128: 256 sequences 266 us, 5.1 TB/s, the rate
// of a large copy; 4 sequences 6.5 us, 21 MB behind a launch and two round trips to memory.
//
// Eight lanes have one row of the state (a head channel) in pieces of 16 bytes, so that a wave's request covers eight whole 128-byte
// lines and the sum over the row is three exchanges.
#include "serve_common.h"

namespace {

struct StepParams {
  const uint16_t* x;
  int64_t sx_b, sx_h;
  const void* dt;
  int64_t sdt_b, sdt_h;
  int dt_dtype;
  const float* A;
  const uint16_t* B;
  int64_t sB_b, sB_g;
  const uint16_t* C;
  int64_t sC_b, sC_g;
  const float* D;
  int D_has_hdim;
  const float* dt_bias;
  int softplus;
  float dt_min, dt_max;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  int num_slots, H, P, G, N;
};

// KN: pieces of 32 state columns.  A wave works on eight rows at a time.
template <typename T, int KN>
__global__ __launch_bounds__(256) void ssm_step_kernel(StepParams p) {
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & 7, r8 = lane >> 3;
  const int slot = sv_slot(p.slots, b, p.num_slots);
  uint16_t* op = p.out + ((int64_t)b * p.H + h) * p.P;
  if (slot < 0) {
    const uint16_t v = slot == kSlotBad ? T::from(__builtin_nanf("")) : 0;
    for (int i = threadIdx.x; i < p.P; i += 256) op[i] = v;
    return;
  }
  const int g = h / (p.H / p.G);
  const float d = sv_step_size(sv_load(p.dt, b * p.sdt_b + h * p.sdt_h, p.dt_dtype), p.dt_bias ? p.dt_bias[h] : 0.0f, p.softplus, p.dt_min, p.dt_max);
  const float decay = lq_expf(d * p.A[h]);
  const uint16_t* Bp = p.B + b * p.sB_b + g * p.sB_g;
  const uint16_t* Cp = p.C + b * p.sC_b + g * p.sC_g;
  float Bv[KN][4], Cv[KN][4];
#pragma unroll
  for (int k = 0; k < KN; ++k) {
    const int n = 32 * k + 4 * sub, at = min(n, p.N - 4);
    const sv_v4u rb = *(const sv_v4u*)(Bp + at), rc = *(const sv_v4u*)(Cp + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) Bv[k][e] = n < p.N ? T::to(rb[e]) : 0.0f, Cv[k][e] = n < p.N ? T::to(rc[e]) : 0.0f;
  }
  float* S = p.state + slot * p.ss_s + (int64_t)h * p.P * p.N;
  const uint16_t* xp = p.x + b * p.sx_b + h * p.sx_h;
  // 16 rows of a wave requested together: one round trip to memory where a head has 64 (eight at a time: 271 and 6.8 us)
  for (int r0 = 8 * wave; r0 < p.P; r0 += 64) {
    lq_v4f s[2][KN];
    float xv[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = min(r0 + 32 * u, p.P - 8) + r8;  // (P is a multiple of 8)
      xv[u] = T::to(xp[row]);
#pragma unroll
      for (int k = 0; k < KN; ++k) s[u][k] = *(const lq_v4f*)(S + (int64_t)row * p.N + min(32 * k + 4 * sub, p.N - 4));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (r0 + 32 * u >= p.P) break;
      const int row = r0 + 32 * u + r8;
      float* Sr = S + (int64_t)row * p.N;
      const float dx = d * xv[u];
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < KN; ++k) {
        if (32 * k + 4 * sub < p.N) {  // (a lane behind the row has another's entries, which are no numbers of its own to add)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][k][e] = __builtin_fmaf(dx, Bv[k][e], decay * s[u][k][e]);
            y = __builtin_fmaf(s[u][k][e], Cv[k][e], y);
          }
          *(lq_v4f*)(Sr + 32 * k + 4 * sub) = s[u][k];
        }
      }
#pragma unroll
      for (int off = 4; off >= 1; off >>= 1) y += __shfl_xor(y, off, 64);
      if (p.D) y = __builtin_fmaf(p.D[p.D_has_hdim ? h * p.P + row : h], xv[u], y);
      if (sub == 0) op[row] = T::from(y);
    }
  }
}

}  // namespace

extern "C" int lq_ssm_step(const lq_ssm_step_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->dt || !a->A || !a->B || !a->C || !a->out || !a->state) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || !sv_float(a->dt_dtype) || a->batch <= 0 || a->batch > 65535 || a->nheads <= 0 || a->ngroups <= 0 || a->nheads % a->ngroups != 0)
    return LQ_ERR_SHAPE;
  if (a->headdim <= 0 || a->headdim % 8 != 0 || a->dstate <= 0 || a->dstate % 8 != 0 || a->dstate > 256 || a->num_slots <= 0) return LQ_ERR_SHAPE;
  if ((int64_t)a->nheads * a->headdim > 0x7fffffff || !sv_fits(a->nheads, 256)) return LQ_ERR_SHAPE;
  if (a->B_stride_b % 4 != 0 || a->B_stride_g % 4 != 0 || a->C_stride_b % 4 != 0 || a->C_stride_g % 4 != 0 || a->state_stride_s % 4 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->B, 8) || !sv_al(a->C, 8) || !sv_al(a->state, 16) || !sv_al(a->x, 2) || !sv_al(a->out, 2) || !sv_al(a->dt, sv_size(a->dt_dtype)) ||
      !sv_al(a->A, 4) || !sv_al(a->D, 4) || !sv_al(a->dt_bias, 4) || !sv_al(a->slots, 4))
    return LQ_ERR_SHAPE;
  StepParams p = {(const uint16_t*)a->x, a->x_stride_b, a->x_stride_h, a->dt, a->dt_stride_b, a->dt_stride_h, a->dt_dtype, a->A,
                  (const uint16_t*)a->B, a->B_stride_b, a->B_stride_g, (const uint16_t*)a->C, a->C_stride_b, a->C_stride_g, a->D, a->D_has_hdim,
                  a->dt_bias, a->dt_softplus, a->dt_min, a->dt_max, (uint16_t*)a->out, a->state, a->state_stride_s, a->slots, a->num_slots,
                  a->nheads, a->headdim, a->ngroups, a->dstate};
  const dim3 grid((unsigned)a->nheads, (unsigned)a->batch);
  auto go = [&](auto t, auto k) {
    hipLaunchKernelGGL((ssm_step_kernel<decltype(t), decltype(k)::value>), grid, dim3(256), 0, stream, p);
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
