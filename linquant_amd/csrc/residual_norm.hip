// The residual stream between two blocks, and the quantizer with a scale for each row.
//   lq_residual_rmsnorm  u = x, or x * rsqrt(mean(x^2) + eps) * post_weight;  r = residual + scale * gate * u;
//                        y = r * rsqrt(mean(r^2) + eps) * weight -> 16 bits, or INT8 codes on a row's or a given scale
//   lq_quantize_rows     scale = max |x| / 127, codes = rint(x / scale)
// A row stays in registers from its one read to its writes: the norms need two passes over it, the codes a third.  HBM-bound; sums
// and everything between the inputs and the outputs is fp32.
//
// A wave per row (four rows to a workgroup, no barrier) where there are many rows, a workgroup of four waves per row where there are few
// or where a row does not fit a wave's registers.  32768 rows of 2560 in fp16 with a gate and both norms: 122 us, 5.5 TB/s of what has to
// move (a large copy reaches 5.1); the quantizer 50 us there, 5.0 TB/s; 16 rows: 3.5 us, a launch and two round trips to memory.
// With INT8 codes of each row from a stream in 32 bits, 32768 rows of 2560: 165 us, 5.6 TB/s.  Rows of 8193 entries and more that are off the
// 16-byte grid spill registers (one entry to a request): 4096 rows of 16383 226 us, 3.6 TB/s, of 16384 149.
#include "row_codes.h"

namespace {

struct RowsParams {
  const void* x;
  int64_t x_stride;
  const void* residual;
  int64_t residual_stride;
  const void* gate;
  int64_t gate_stride;
  int gate_rows;
  const void* post_weight;
  const void* weight;
  int weight_dtype;
  float scale, eps;
  void* residual_out;
  int64_t residual_out_stride;
  void* out;
  int64_t out_stride;
  int8_t* codes;
  int64_t codes_stride;
  const float* code_scale;
  float* row_scale;
  int rows, dim;
};

template <typename T, typename RT, int NV, int TH, bool VEC>
__global__ __launch_bounds__(256) void residual_norm_kernel(RowsParams p) {
  __shared__ float lds[3 * (256 / 64)];
  const int tid = threadIdx.x % TH;
  const int64_t row = (int64_t)blockIdx.x * (256 / TH) + threadIdx.x / TH;
  if (row >= p.rows) return;  // (whole waves, and whole workgroups where a row is one)
  const int dim = p.dim;
  using X = Row<T, NV, TH, VEC>;
  using R = Row<RT, NV, TH, VEC>;
  float u[8 * NV], w[8 * NV], r[8 * NV];
  auto weights = [&](const void* at) {
    if (p.weight_dtype == LQ_DT_F32) Row<F32, NV, TH, VEC>::load(at, 0, dim, tid, w);
    else if (p.weight_dtype == LQ_DT_F16) Row<F16, NV, TH, VEC>::load(at, 0, dim, tid, w);
    else Row<BF16, NV, TH, VEC>::load(at, 0, dim, tid, w);
  };
  X::load(p.x, row * p.x_stride, dim, tid, u);
  if (p.residual) {
    R::load(p.residual, row * p.residual_stride, dim, tid, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) r[i] = 0.0f;
  }
  if (p.post_weight) {
    weights(p.post_weight);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) s = __builtin_fmaf(u[i], u[i], s);
    s = over_row<TH>(s, plus, lds, 0);
    const float rs = __builtin_amdgcn_rsqf(s / (float)dim + p.eps);
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) u[i] = u[i] * rs * w[i];
  }
  if (p.gate) {
    X::load(p.gate, (row / p.gate_rows) * p.gate_stride, dim, tid, w);
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) u[i] = u[i] * w[i];
  }
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) r[i] = __builtin_fmaf(p.scale, u[i], r[i]);
  if (p.residual_out) R::store(p.residual_out, row * p.residual_out_stride, dim, tid, r);
  weights(p.weight);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) s = __builtin_fmaf(r[i], r[i], s);
  s = over_row<TH>(s, plus, lds, 1);
  const float rs = __builtin_amdgcn_rsqf(s / (float)dim + p.eps);
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) r[i] = r[i] * rs * w[i];
  if (p.out) X::store(p.out, row * p.out_stride, dim, tid, r);
  else if (p.code_scale) store_codes<NV, TH, VEC>(p.codes, row * p.codes_stride, dim, tid, r, *p.code_scale, -128.0f);
  else row_codes<NV, TH, VEC>(p.row_scale + row, p.codes, row * p.codes_stride, dim, tid, r, lds, 2);
}

template <typename T, int NV, int TH, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(RowsParams p) {
  __shared__ float lds[256 / 64];
  const int tid = threadIdx.x % TH;
  const int64_t row = (int64_t)blockIdx.x * (256 / TH) + threadIdx.x / TH;
  if (row >= p.rows) return;
  float v[8 * NV];
  Row<T, NV, TH, VEC>::load(p.x, row * p.x_stride, p.dim, tid, v);
  row_codes<NV, TH, VEC>(p.row_scale + row, p.codes, row * p.codes_stride, p.dim, tid, v, lds, 0);
}

constexpr int kMaxDim = 16384;

// A wave per row from here on, where the row fits 64 values a lane.  us, a wave / a workgroup to a row of 2560 in fp16: the quantizer with
// 512 rows 4.6 / 3.4, 4096 10.1 / 10.0, 16384 24 / 31; the norm of an fp32 stream with 512 rows 5.7 / 5.1, 4096 22.2 / 21.3, 16384 94 / 92;
// with two norms and a gate, 32768 rows, 122 / 130.
constexpr int kWaveRows = 8192;

template <typename T, typename RT, bool QUANT, bool VEC>
int launch_rows(const RowsParams& p, hipStream_t stream) {
  auto go = [&](auto nv, auto th) {
    constexpr int NV = decltype(nv)::value, TH = decltype(th)::value;
    const dim3 grid((unsigned)(((int64_t)p.rows * TH + 255) / 256));
    if (!sv_fits(grid.x, 256)) return (int)LQ_ERR_SHAPE;
    if constexpr (QUANT) hipLaunchKernelGGL((quantize_rows_kernel<T, NV, TH, VEC>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((residual_norm_kernel<T, RT, NV, TH, VEC>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  using std::integral_constant;
  const integral_constant<int, 64> wave;
  const integral_constant<int, 256> group;
  if constexpr (VEC) {
    if (p.rows >= kWaveRows && p.dim <= 4096) {
      const int n = (p.dim + 511) / 512;
      if (n <= 2) return go(integral_constant<int, 2>{}, wave);
      if (n <= 4) return go(integral_constant<int, 4>{}, wave);
      if (n <= 5) return go(integral_constant<int, 5>{}, wave);
      return go(integral_constant<int, 8>{}, wave);
    }
    if (p.dim <= 2048) return go(integral_constant<int, 1>{}, group);
    if (p.dim <= 4096) return go(integral_constant<int, 2>{}, group);
  }
  if (p.dim <= 8192) return go(integral_constant<int, 4>{}, group);
  return go(integral_constant<int, 8>{}, group);
}

}  // namespace

extern "C" int lq_quantize_rows(const lq_quantize_rows_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->codes || !a->scale) return LQ_ERR_NULL;
  if (a->rows <= 0 || a->cols <= 0 || a->cols > kMaxDim || !sv_float(a->dtype)) return LQ_ERR_SHAPE;
  if (!sv_al(a->x, sv_size(a->dtype)) || !sv_al(a->scale, 4)) return LQ_ERR_SHAPE;
  RowsParams p = {};
  p.x = a->x, p.x_stride = a->x_stride, p.codes = a->codes, p.codes_stride = a->codes_stride, p.row_scale = a->scale;
  p.rows = a->rows, p.dim = a->cols;
  const bool vec = a->cols % 8 == 0 && a->x_stride % 8 == 0 && a->codes_stride % 8 == 0 && sv_al(a->x, 16) && sv_al(a->codes, 8);
  auto go = [&](auto t) {
    using T = decltype(t);
    return vec ? launch_rows<T, T, true, true>(p, stream) : launch_rows<T, T, true, false>(p, stream);
  };
  if (a->dtype == LQ_DT_F32) return go(F32{});
  return a->dtype == LQ_DT_F16 ? go(F16{}) : go(BF16{});
}

extern "C" int lq_residual_rmsnorm(const lq_residual_rmsnorm_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->weight || (!a->out && !a->codes) || (a->codes && !a->code_scale && !a->row_scale)) return LQ_ERR_NULL;
  if (a->rows <= 0 || a->dim <= 0 || a->dim > kMaxDim || !sv_act(a->dtype) || !sv_float(a->weight_dtype)) return LQ_ERR_SHAPE;
  if ((a->out && a->codes) || (a->gate && a->gate_rows <= 0)) return LQ_ERR_SHAPE;
  const bool stream_out = a->residual || a->residual_out;
  if (stream_out && a->residual_dtype != a->dtype && a->residual_dtype != LQ_DT_F32) return LQ_ERR_SHAPE;
  const bool r32 = stream_out && a->residual_dtype == LQ_DT_F32;
  const int ws = sv_size(a->weight_dtype), rsz = r32 ? 4 : 2;
  if (!sv_al(a->x, 2) || !sv_al(a->gate, 2) || !sv_al(a->out, 2) || !sv_al(a->weight, ws) || !sv_al(a->post_weight, ws) || !sv_al(a->residual, rsz) ||
      !sv_al(a->residual_out, rsz) || !sv_al(a->code_scale, 4) || !sv_al(a->row_scale, 4))
    return LQ_ERR_SHAPE;
  RowsParams p;
  p.x = a->x, p.x_stride = a->x_stride, p.residual = a->residual, p.residual_stride = a->residual_stride;
  p.gate = a->gate, p.gate_stride = a->gate_stride, p.gate_rows = a->gate_rows;
  p.post_weight = a->post_weight, p.weight = a->weight, p.weight_dtype = a->weight_dtype, p.scale = a->scale, p.eps = a->eps;
  p.residual_out = a->residual_out, p.residual_out_stride = a->residual_out_stride, p.out = a->out, p.out_stride = a->out_stride;
  p.codes = a->codes, p.codes_stride = a->codes_stride, p.code_scale = a->code_scale, p.row_scale = a->row_scale;
  p.rows = a->rows, p.dim = a->dim;
  const void* ptrs[] = {a->x, a->residual, a->gate, a->post_weight, a->weight, a->residual_out, a->out};
  bool vec = a->dim % 8 == 0 && a->x_stride % 8 == 0 && sv_al(a->codes, 8);
  for (const void* q : ptrs) vec = vec && sv_al(q, 16);
  vec = vec && (!a->residual || a->residual_stride % 8 == 0) && (!a->gate || a->gate_stride % 8 == 0) &&
        (!a->residual_out || a->residual_out_stride % 8 == 0) && (!a->out || a->out_stride % 8 == 0) && (!a->codes || a->codes_stride % 8 == 0);
  auto go = [&](auto t, auto rt) {
    using T = decltype(t);
    using RT = decltype(rt);
    return vec ? launch_rows<T, RT, false, true>(p, stream) : launch_rows<T, RT, false, false>(p, stream);
  };
  if (a->dtype == LQ_DT_F16) return r32 ? go(F16{}, F32{}) : go(F16{}, F16{});
  return r32 ? go(BF16{}, F32{}) : go(BF16{}, BF16{});
}
