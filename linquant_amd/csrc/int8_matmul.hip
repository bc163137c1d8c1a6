// lq_int8_matmul: out[m,n] = (sum_k a[m,k] b[n,k]) * a_scale[m] * b_scale[n] + bias[n], INT8 in, the sum exact in 32 bits.
//
// The matrix instruction is v_mfma_i32_32x32x32_i8, which reaches 4.9 POPS here where the 16x16x64 form reaches 3.0.  Operands: lane l has
// row l & 31 and the 16 contraction bytes of half l >> 5; the result: column l & 31, rows 8 (r >> 2) + 4 (l >> 5) + (r & 3).
#include "serve_common.h"

namespace {

struct MatmulParams {
  const int8_t* a;
  int64_t a_stride;
  const int8_t* b;
  int64_t b_stride;
  const float* a_scale;
  const float* b_scale;
  int a_scale_rows, b_scale_cols;
  const void* bias;
  int bias_dtype;
  void* out;
  int64_t out_stride;
  int rows, cols, inner;
};

struct O32 {
  using type = float;
  static LQ_DEV float from(float f) { return f; }
};
template <typename T>
struct OutOf {
  using type = uint16_t;
};
template <>
struct OutOf<O32> {
  using type = float;
};

constexpr int kTile = 128, kStep = 128;  // rows of either operand in a tile, contraction bytes of a step

template <typename O>
__global__ __launch_bounds__(256) void int8_matmul_kernel(MatmulParams p) {
  __shared__ __align__(16) int8_t As[kTile * kStep], Bs[kTile * kStep];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  lq_v16i acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  for (int k0 = 0; k0 < p.inner; k0 += kStep) {
    lq_v4i ra[4], rb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pc = tid + 256 * i, r = pc >> 3, k = k0 + (pc & 7) * 16;
      const int kc = min(k, p.inner - 16);
      ra[i] = *(const lq_v4i*)(p.a + min(m0 + r, p.rows - 1) * p.a_stride + kc);
      rb[i] = *(const lq_v4i*)(p.b + min(n0 + r, p.cols - 1) * p.b_stride + kc);
      if (k >= p.inner) ra[i] = lq_v4i{0, 0, 0, 0};  // (a zero of one operand is enough)
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pc = tid + 256 * i, r = pc >> 3, at = r * kStep + ((pc ^ r) & 7) * 16;
      *(lq_v4i*)(As + at) = ra[i];
      *(lq_v4i*)(Bs + at) = rb[i];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      lq_v4i fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 32 * i + (lane & 31), c = 2 * s + (lane >> 5);
        fa[i] = *(const lq_v4i*)(As + (wm + r) * kStep + ((c ^ r) & 7) * 16);
        fb[i] = *(const lq_v4i*)(Bs + (wn + r) * kStep + ((c ^ r) & 7) * 16);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
  typename OutOf<O>::type* out = (typename OutOf<O>::type*)p.out;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 32 * j + (lane & 31);
    if (n >= p.cols) continue;
    const float sb = p.b_scale[p.b_scale_cols ? n : 0];
    const float bias = p.bias ? sv_load(p.bias, n, p.bias_dtype) : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + wm + 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (m >= p.rows) continue;
        const float sa = p.a_scale[p.a_scale_rows ? m : 0];
        out[m * p.out_stride + n] = O::from(__builtin_fmaf((float)acc[i][j][e], sa * sb, bias));
      }
  }
}

}  // namespace

extern "C" int lq_int8_matmul(const lq_int8_matmul_args* a, hipStream_t stream) {
  if (!a || !a->a || !a->b || !a->a_scale || !a->b_scale || !a->out) return LQ_ERR_NULL;
  if (a->rows <= 0 || a->cols <= 0 || a->inner <= 0 || a->inner % 16 != 0 || a->inner > 131056) return LQ_ERR_SHAPE;
  if (!sv_float(a->out_dtype) || (a->bias && !sv_float(a->bias_dtype))) return LQ_ERR_SHAPE;
  if (a->a_stride % 16 != 0 || a->b_stride % 16 != 0 || !sv_al(a->a, 16) || !sv_al(a->b, 16)) return LQ_ERR_SHAPE;
  if (!sv_al(a->out, sv_size(a->out_dtype)) || (a->bias && !sv_al(a->bias, sv_size(a->bias_dtype))) || !sv_al(a->a_scale, 4) || !sv_al(a->b_scale, 4))
    return LQ_ERR_SHAPE;
  MatmulParams p = {a->a, a->a_stride, a->b, a->b_stride, a->a_scale, a->b_scale, a->a_scale_rows, a->b_scale_cols, a->bias, a->bias_dtype,
                    a->out, a->out_stride, a->rows, a->cols, a->inner};
  const dim3 grid((unsigned)((a->cols + kTile - 1) / kTile), (unsigned)((a->rows + kTile - 1) / kTile));
  if (grid.y > 65535) return LQ_ERR_SHAPE;
  auto go = [&](auto o) {
    hipLaunchKernelGGL((int8_matmul_kernel<decltype(o)>), grid, dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  if (a->out_dtype == LQ_DT_F32) return go(O32{});
  return a->out_dtype == LQ_DT_F16 ? go(F16{}) : go(BF16{});
}
