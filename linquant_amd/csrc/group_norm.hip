// lq_groupnorm_gated: group norm of each row, channels last, with a gate.
//   y = (x - mean) * rsqrt(var + eps) * weight + bias over groups of adjacent channels;  out = y * act(z), or act(y)
// HBM-bound: x and z once, out once.  A group stays in registers from its one read to its write, so the variance is that of the
// differences from the mean (a second pass over registers), not a difference of sums.
//
// TH threads have a group: 8 to 64 lanes of a wave where 8 NV entries a lane hold it, so that one wave has up to eight groups and sums are a
// few lane exchanges, else a workgroup.
//
// 16384 rows of 32 heads of 128, fp16, gate and weights: 83 us, 4.8 TB/s of 5.2 that a copy reaches; 13622 rows of 16 of 256, no gate, 56 us, 4.0.
// Few rows are a launch and two round trips to memory: 16 rows of 32 of 128 4.8 us.
#include <algorithm>

#include "serve_common.h"

namespace {

constexpr int kWorkgroups = 256 * 8 * 2;

struct NormParams {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* z;
  int64_t z_stride;
  const void* weight;
  const void* bias;
  uint16_t* out;
  float eps;
  int64_t rows;
  int num_groups, size, act;
  int side, high;  // groups of a row that a workgroup has side by side, rows one behind the other
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
    __syncthreads();  // (two turns: what is read behind one is written again behind the other's)
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) v += s[w];
  }
  return v;
}

// Entries of one group in the order of a thread's registers.  VEC: eight adjacent channels at a time (every group starts on a 16-byte boundary
// and has whole eights), else one at a time.
template <int TH, int NV, bool VEC>
struct Part {
  static constexpr int E = 8 * NV;
  static LQ_DEV int index(int tid, int i) { return VEC ? ((i >> 3) * TH + tid) * 8 + (i & 7) : i * TH + tid; }
  static LQ_DEV void load(const uint16_t* base, int n, int tid, uint16_t (&raw)[E]) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const sv_v8u r = __builtin_nontemporal_load((const sv_v8u*)(base + min((i * TH + tid) * 8, n - 8)));
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[8 * i + e] = r[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) raw[i] = base[min(i * TH + tid, n - 1)];
    }
  }
  static LQ_DEV void store(uint16_t* base, int n, int tid, const uint16_t (&o)[E]) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        sv_v8u v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = o[8 * i + e];
        if ((i * TH + tid) * 8 < n) __builtin_nontemporal_store(v, (sv_v8u*)(base + (i * TH + tid) * 8));
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * TH + tid < n) base[i * TH + tid] = o[i];
    }
  }
  // scale or shift, `none` where there is none
  template <typename W>
  static LQ_DEV void weights(const void* p, int64_t at, int n, int tid, float none, float (&w)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int64_t c = at + min(index(tid, i), n - 1);
      if constexpr (std::is_same<W, float>::value) w[i] = p ? ((const float*)p)[c] : none;
      else w[i] = p ? W::to(((const uint16_t*)p)[c]) : none;
    }
  }
};

// A workgroup has some of the groups of some rows, then the same groups of the rows `stride` on: their scale and shift are read once.
template <typename T, typename W, int TH, int NV, bool VEC>
__global__ __launch_bounds__(256) void group_norm_kernel(NormParams p) {
  using P = Part<TH, NV, VEC>;
  constexpr int E = P::E;
  __shared__ float lds[2 * 4];
  const int tid = threadIdx.x % TH, place = threadIdx.x / TH, n = p.size;
  const int grp = min(blockIdx.y * (256 / TH) + place % p.side, p.num_groups - 1);
  const bool mine = (int)blockIdx.y * (256 / TH) + place % p.side < p.num_groups && place < p.side * p.high;
  const int64_t ch = (int64_t)grp * n, dim = (int64_t)p.num_groups * n;
  float w[E], b[E];
  P::template weights<W>(p.weight, ch, n, tid, 1.0f, w);
  P::template weights<W>(p.bias, ch, n, tid, 0.0f, b);
  for (int64_t row0 = (int64_t)blockIdx.x * p.high; row0 < p.rows; row0 += (int64_t)gridDim.x * p.high) {
    const int64_t at = row0 + place / p.side, row = min(at, p.rows - 1);  // (a whole wave's exchanges need all of its lanes)
    uint16_t xr[E], zr[E];
    P::load(p.x + row * p.x_stride + ch, n, tid, xr);
    if (p.z) P::load(p.z + row * p.z_stride + ch, n, tid, zr);
    float x[E], s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = P::index(tid, i) < n ? T::to(xr[i]) : 0.0f, s += x[i];
    const float mean = over_group<TH>(s, lds, 0) / (float)n;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] = P::index(tid, i) < n ? x[i] - mean : 0.0f;
      q = __builtin_fmaf(x[i], x[i], q);
    }
    const float rs = __builtin_amdgcn_rsqf(over_group<TH>(q, lds, 1) / (float)n + p.eps);
    uint16_t o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float y = x[i] * rs;
      if (p.weight) y *= w[i];
      if (p.bias) y += b[i];
      o[i] = T::from(p.z ? y * activate(T::to(zr[i]), p.act) : activate(y, p.act));
    }
    if (mine && at < p.rows) P::store(p.out + row * dim + ch, n, tid, o);
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
  NormParams p = {(const uint16_t*)a->x, a->x_stride, (const uint16_t*)a->z, a->z_stride, a->weight, a->bias, (uint16_t*)a->out, a->eps, a->rows, a->num_groups, size, a->act, 0, 0};
  const bool vec = size % 8 == 0 && a->x_stride % 8 == 0 && (!a->z || a->z_stride % 8 == 0) && sv_al(a->x, 16) && sv_al(a->z, 16) && sv_al(a->out, 16);
  auto go = [&](auto t, auto w, auto th, auto nv, auto v) {
    constexpr int TH = decltype(th)::value, places = 256 / TH;
    p.side = std::min(places, a->num_groups), p.high = places / p.side;
    const int64_t across = ((int64_t)a->num_groups + places - 1) / places, down = ((int64_t)a->rows + p.high - 1) / p.high;
    // as many workgroups as the card holds at a time, some times over: each goes on to further rows
    const int64_t most = std::max<int64_t>(1, kWorkgroups / across);
    if (across > 65535) return (int)LQ_ERR_SHAPE;
    const dim3 grid((unsigned)std::min(down, most), (unsigned)across);
    hipLaunchKernelGGL((group_norm_kernel<decltype(t), decltype(w), TH, decltype(nv)::value, decltype(v)::value>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  auto sized = [&](auto t, auto w, auto v) {
    using std::integral_constant;
    const integral_constant<int, 1> one;
    if (size <= 64) return go(t, w, integral_constant<int, 8>{}, one, v);
    if (size <= 128) return go(t, w, integral_constant<int, 16>{}, one, v);
    if (size <= 256) return go(t, w, integral_constant<int, 32>{}, one, v);
    if (size <= 512) return go(t, w, integral_constant<int, 64>{}, one, v);
    if (size <= 1024) return go(t, w, integral_constant<int, 64>{}, integral_constant<int, 2>{}, v);
    if (size <= 2048) return go(t, w, integral_constant<int, 64>{}, integral_constant<int, 4>{}, v);
    if (size <= 4096) return go(t, w, integral_constant<int, 256>{}, integral_constant<int, 2>{}, v);
    if (size <= 8192) return go(t, w, integral_constant<int, 256>{}, integral_constant<int, 4>{}, v);
    return go(t, w, integral_constant<int, 256>{}, integral_constant<int, 8>{}, v);
  };
  auto typed = [&](auto t, auto w) { return vec ? sized(t, w, std::true_type{}) : sized(t, w, std::false_type{}); };
  auto with = [&](auto t) {
    if (!a->weight && !a->bias) return typed(t, t);
    if (a->weight_dtype == LQ_DT_F32) return typed(t, 1.0f);
    return a->weight_dtype == LQ_DT_F16 ? typed(t, F16{}) : typed(t, BF16{});
  };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
