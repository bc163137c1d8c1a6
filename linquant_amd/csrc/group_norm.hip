// lq_groupnorm_gated: group norm of each row, channels last, with a gate.
//   y = (x - mean) * rsqrt(var + eps) * weight + bias over groups of adjacent channels;  out = y * act(z), or act(y)
// HBM-bound: x and z once, out once.  A group stays in registers from its one read to its write, so the variance is that of the
// differences from the mean (a second pass over registers), not a difference of sums.
//
// TH threads have a group: 8 to 64 lanes of a wave where 8 NV entries a lane hold it, so that one wave has up to eight groups and sums are a
// few lane exchanges, else a workgroup.
#include "serve_common.h"

namespace {

struct NormParams {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* z;
  int64_t z_stride;
  const void* weight;
  const void* bias;
  int weight_dtype;
  uint16_t* out;
  float eps;
  int64_t groups;  // of all rows
  int num_groups, size, act;
};

LQ_DEV float activate(float v, int act) {
  if (act == 0) return v;
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
  return act == 1 ? v * s : s;
}

// sums over the TH threads of a group.  `turn` keeps two reductions of a workgroup apart.
template <int TH>
LQ_DEV float over_group(float v, float* lds, int turn) {
#pragma unroll
  for (int off = (TH > 64 ? 64 : TH) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (TH > 64) {
    float* s = lds + turn * (TH / 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) v += s[w];
  }
  return v;
}

// VEC: eight adjacent channels at a time (every group starts on a 16-byte boundary and has whole eights), else one at a time
template <typename T, int TH, int NV, bool VEC>
__global__ __launch_bounds__(256) void group_norm_kernel(NormParams p) {
  __shared__ float lds[2 * 4];
  const int tid = threadIdx.x % TH;
  const int64_t at = (int64_t)blockIdx.x * (256 / TH) + threadIdx.x / TH;
  const bool live = at < p.groups;  // (a whole wave's exchanges need all of its lanes)
  const int64_t gr = live ? at : p.groups - 1, row = gr / p.num_groups;
  const int grp = (int)(gr - row * p.num_groups), n = p.size;
  const int64_t ch = (int64_t)grp * n;
  const uint16_t* xp = p.x + row * p.x_stride + ch;
  const uint16_t* zp = p.z ? p.z + row * p.z_stride + ch : nullptr;
  uint16_t* op = p.out + row * ((int64_t)p.num_groups * n) + ch;
  constexpr int E = 8 * NV;
  // entry i of this thread
  auto index = [&](int i) { return VEC ? ((i >> 3) * TH + tid) * 8 + (i & 7) : i * TH + tid; };
  auto load = [&](const uint16_t* base, uint16_t (&raw)[E]) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const sv_v8u r = *(const sv_v8u*)(base + min((i * TH + tid) * 8, n - 8));
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[8 * i + e] = r[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = base[min(i * TH + tid, n - 1)];
    }
  };
  uint16_t xr[E], zr[E];
  load(xp, xr);
  if (zp) load(zp, zr);
  float x[E], s = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = index(i) < n ? T::to(xr[i]) : 0.0f, s += x[i];
  const float mean = over_group<TH>(s, lds, 0) / (float)n;
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x[i] = index(i) < n ? x[i] - mean : 0.0f;
    q = __builtin_fmaf(x[i], x[i], q);
  }
  const float rs = __builtin_amdgcn_rsqf(over_group<TH>(q, lds, 1) / (float)n + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint16_t o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = min(index(8 * i + e), n - 1);
      float y = x[8 * i + e] * rs;
      if (p.weight) y *= sv_load(p.weight, ch + c, p.weight_dtype);
      if (p.bias) y += sv_load(p.bias, ch + c, p.weight_dtype);
      o[e] = T::from(zp ? y * activate(T::to(zr[8 * i + e]), p.act) : activate(y, p.act));
    }
    if constexpr (VEC) {
      sv_v8u v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = o[e];
      if (live && (i * TH + tid) * 8 < n) *(sv_v8u*)(op + (i * TH + tid) * 8) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (live && index(8 * i + e) < n) op[index(8 * i + e)] = o[e];
    }
  }
}

}  // namespace

extern "C" int lq_groupnorm_gated(const lq_groupnorm_gated_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->out) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || a->rows <= 0 || a->dim <= 0 || a->num_groups <= 0 || a->dim % a->num_groups != 0 || a->act < 0 || a->act > 2) return LQ_ERR_SHAPE;
  const int size = a->dim / a->num_groups;
  if (size > 16384 || ((a->weight || a->bias) && !sv_float(a->weight_dtype))) return LQ_ERR_SHAPE;
  const int ws = a->weight || a->bias ? sv_size(a->weight_dtype) : 1;
  if (!sv_al(a->x, 2) || !sv_al(a->z, 2) || !sv_al(a->out, 2) || !sv_al(a->weight, ws) || !sv_al(a->bias, ws)) return LQ_ERR_SHAPE;
  NormParams p = {(const uint16_t*)a->x, a->x_stride, (const uint16_t*)a->z, a->z_stride, a->weight, a->bias, a->weight_dtype, (uint16_t*)a->out, a->eps,
                  (int64_t)a->rows * a->num_groups, a->num_groups, size, a->act};
  const bool vec = size % 8 == 0 && a->x_stride % 8 == 0 && (!a->z || a->z_stride % 8 == 0) && sv_al(a->x, 16) && sv_al(a->z, 16) && sv_al(a->out, 16);
  auto go = [&](auto t, auto th, auto nv, auto v) {
    constexpr int TH = decltype(th)::value;
    const int64_t wgs = (p.groups * TH + 255) / 256;
    if (!sv_fits(wgs, 256)) return (int)LQ_ERR_SHAPE;
    hipLaunchKernelGGL((group_norm_kernel<decltype(t), TH, decltype(nv)::value, decltype(v)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  auto sized = [&](auto t, auto v) {
    using std::integral_constant;
    const integral_constant<int, 1> one;
    if (size <= 64) return go(t, integral_constant<int, 8>{}, one, v);
    if (size <= 128) return go(t, integral_constant<int, 16>{}, one, v);
    if (size <= 256) return go(t, integral_constant<int, 32>{}, one, v);
    if (size <= 512) return go(t, integral_constant<int, 64>{}, one, v);
    if (size <= 1024) return go(t, integral_constant<int, 64>{}, integral_constant<int, 2>{}, v);
    if (size <= 2048) return go(t, integral_constant<int, 64>{}, integral_constant<int, 4>{}, v);
    if (size <= 4096) return go(t, integral_constant<int, 256>{}, integral_constant<int, 2>{}, v);
    if (size <= 8192) return go(t, integral_constant<int, 256>{}, integral_constant<int, 4>{}, v);
    return go(t, integral_constant<int, 256>{}, integral_constant<int, 8>{}, v);
  };
  auto with = [&](auto t) { return vec ? sized(t, std::true_type{}) : sized(t, std::false_type{}); };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
