// lq_adapter_down: the first half of low-rank adapters of many requests, h[m] = scaling[j] * (down[j] x[m]), j = ids[m], in fp32; the second
// half is the epilogue of lq_int8_matmul.
//
// Two kernels.  `rows`: few rows, each with a request of its own as a rule: a wave has two of a row's sums, so that the adapters stream from
// memory through many waves.  `tiles`: 16 rows of x to a workgroup, its waves share the contraction, and what meets the rows are the
// matrix instructions; the adapters that the 16 rows name are taken one after the other, each with all 16 rows, and a row keeps what its own
// gave (nothing is multiplied by zero: an infinity in one request's row or adapter stays there).  Rows of a prompt name one as a rule.
// v_mfma_f32_16x16x32: lane l has row l & 15 and the 8 contraction entries of quarter l >> 4; the result: column l & 15, rows 4 (l >> 4) + r.
// down is the operand of the rows, so that a lane holds four adjacent sums of one row of x.
//
// INT8 codes become 16 bits exactly; their scale multiplies the sum.  All sums are fp32.
#include "serve_common.h"

namespace {

struct DownParams {
  const void* x;
  int64_t x_stride;
  const float* x_scale;
  int x_scale_rows;
  const uint16_t* down;
  const float* scaling;
  const int32_t* ids;
  float* h;
  int rows, inner, padded, rank, count;
};

template <typename T>
LQ_DEV lq_v4f mfma16(lq_v4i a, lq_v4i b, lq_v4f c) {
  if constexpr (std::is_same<T, F16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lq_v8h, a), __builtin_bit_cast(lq_v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sv_v8bf, a), __builtin_bit_cast(sv_v8bf, b), c, 0, 0, 0);
}

// eight entries of a row from `k` on in T, zero behind the row's end.  (The last eight are read again there: inner is at least 8, or the row
// is read one by one.)
template <typename T, bool CODES>
LQ_DEV lq_v4i load8(const void* row, int k, int inner) {
  uint16_t v[8];
  if (inner % 8 == 0) {
    const int at = min(k, inner - 8);
    if constexpr (CODES) {
      const lq_v2i r = *(const lq_v2i*)((const int8_t*)row + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = T::from((float)lq_sbyte((uint32_t)r[e >> 2], e & 3));
    } else {
      const sv_v8u r = *(const sv_v8u*)((const uint16_t*)row + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k < inner ? v[e] : 0;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = min(k + e, inner - 1);
      uint16_t u;
      if constexpr (CODES) u = T::from((float)((const int8_t*)row)[at]);
      else u = ((const uint16_t*)row)[at];
      v[e] = k + e < inner ? u : 0;
    }
  }
  lq_v4i o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (int)(v[2 * i] | (uint32_t)v[2 * i + 1] << 16);
  return o;
}

template <typename T, bool CODES>
LQ_DEV const void* row_of(const DownParams& p, int m) {
  return (const char*)p.x + (int64_t)m * p.x_stride * (CODES ? 1 : 2);
}
template <bool CODES>
LQ_DEV float factor(const DownParams& p, int m, int id) {
  return CODES ? p.scaling[id] * p.x_scale[p.x_scale_rows ? m : 0] : p.scaling[id];
}

constexpr int kPer = 2;  // sums of a wave in `rows`

template <typename T, bool CODES>
__global__ __launch_bounds__(256) void down_rows_kernel(DownParams p) {
  const int m = blockIdx.x, lane = threadIdx.x & 63, r0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kPer;
  if (r0 >= p.rank) return;
  const int id = p.ids[m];
  float* h = p.h + (int64_t)m * p.rank + r0;
  if (id < 0 || id >= p.count) {
    if (lane < kPer) h[lane] = id < 0 ? 0.0f : __builtin_nanf("");
    return;
  }
  const void* x = row_of<T, CODES>(p, m);
  const uint16_t* d = p.down + ((int64_t)id * p.rank + r0) * p.padded;
  float s[kPer] = {};
  for (int k0 = 0; k0 < p.padded; k0 += 64 * 8 * 4) {
    lq_v4i xv[4], dv[4][kPer];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + (u * 64 + lane) * 8;
      xv[u] = load8<T, CODES>(x, k, p.inner);
#pragma unroll
      for (int r = 0; r < kPer; ++r) dv[u][r] = *(const lq_v4i*)(d + (int64_t)r * p.padded + min(k, p.padded - 8));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (k0 + (u * 64 + lane) * 8 >= p.inner) continue;
#pragma unroll
      for (int r = 0; r < kPer; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s[r] = __builtin_fmaf(T::to((uint16_t)((uint32_t)xv[u][e >> 1] >> (16 * (e & 1)))), T::to((uint16_t)((uint32_t)dv[u][r][e >> 1] >> (16 * (e & 1)))), s[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < kPer; ++r)
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s[r] += __shfl_xor(s[r], off, 64);
  const float f = factor<CODES>(p, m, id);
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < kPer; ++r) h[r] = s[r] * f;
  }
}

// RT tiles of 16 sums; W waves share the contraction in lines of 64 entries, side by side
template <typename T, bool CODES, int RT, int W>
__global__ __launch_bounds__(64 * W) void down_tiles_kernel(DownParams p) {
  __shared__ __align__(16) lq_v4f sums[W][RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
  const int m0 = blockIdx.x * 16, m = min(m0 + (lane & 15), p.rows - 1);
  const int id = p.ids[m];
  const void* x = row_of<T, CODES>(p, m);
  lq_v4f keep[RT];
  const float none = id < 0 ? 0.0f : __builtin_nanf("");
#pragma unroll
  for (int t = 0; t < RT; ++t) keep[t] = lq_v4f{none, none, none, none};
  uint64_t left = __ballot(id >= 0 && id < p.count);
  while (left) {
    const int j = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const bool mine = id == j;
    left &= ~__ballot(mine);
    const uint16_t* d = p.down + ((int64_t)j * p.rank + (lane & 15)) * p.padded;
    lq_v4f acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = lq_v4f{0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * 64; k0 < p.padded; k0 += 64 * W) {
      lq_v4i xv[2], dv[2][RT];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = k0 + 32 * u + 8 * quarter, kc = min(k, p.padded - 8);
        xv[u] = load8<T, CODES>(x, k, p.inner);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          dv[u][t] = *(const lq_v4i*)(d + (int64_t)16 * t * p.padded + kc);
          if (k >= p.padded) dv[u][t] = lq_v4i{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = mfma16<T>(dv[u][t], xv[u], acc[t]);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sv_settle(acc[t]);
      if (mine) keep[t] = acc[t];
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) sums[wave][t][lane] = keep[t];
  __syncthreads();
  for (int i = threadIdx.x; i < RT * 64; i += 64 * W) {
    const int t = i >> 6, l = i & 63, row = m0 + (l & 15);
    lq_v4f v = sums[0][t][l];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][t][l];
    if (row >= p.rows) continue;
    const int own = p.ids[row];
    const float f = own >= 0 && own < p.count ? factor<CODES>(p, row, own) : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= f;
    *(lq_v4f*)(p.h + (int64_t)row * p.rank + 16 * t + 4 * (l >> 4)) = v;
  }
}

constexpr int kFewRows = 256;

}  // namespace

extern "C" int lq_adapter_down(const lq_adapter_down_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->down || !a->scaling || !a->ids || !a->h || (a->x_dtype == LQ_DT_I8 && !a->x_scale)) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || (a->x_dtype != a->dtype && a->x_dtype != LQ_DT_I8)) return LQ_ERR_SHAPE;
  if (a->rows <= 0 || a->inner <= 0 || a->inner_padded < a->inner || a->inner_padded % 16 != 0 || a->count <= 0) return LQ_ERR_SHAPE;
  if (a->rank <= 0 || a->rank % 16 != 0 || a->rank > 128) return LQ_ERR_SHAPE;
  const bool codes = a->x_dtype == LQ_DT_I8;
  // (rows that are not whole eights of entries are read one by one)
  if (a->inner % 8 == 0 ? !sv_al(a->x, codes ? 8 : 16) || a->x_stride % 8 != 0 : !sv_al(a->x, codes ? 1 : 2)) return LQ_ERR_SHAPE;
  if (!sv_al(a->down, 16) || !sv_al(a->h, 16) || !sv_al(a->x_scale, 4) || !sv_al(a->scaling, 4) || !sv_al(a->ids, 4))
    return LQ_ERR_SHAPE;
  DownParams p = {a->x, a->x_stride, a->x_scale, a->x_scale_rows, (const uint16_t*)a->down, a->scaling, a->ids, a->h, a->rows, a->inner, a->inner_padded, a->rank, a->count};
  auto go = [&](auto t, auto c) {
    using T = decltype(t);
    constexpr bool C = decltype(c)::value;
    if (a->rows <= kFewRows) {
      hipLaunchKernelGGL((down_rows_kernel<T, C>), dim3((unsigned)a->rows, (unsigned)((a->rank + 4 * kPer - 1) / (4 * kPer))), dim3(256), 0, stream, p);
      return lq_check_launch();
    }
    auto tiles = [&](auto rt) {
      constexpr int RT = decltype(rt)::value, W = RT <= 4 ? 8 : 4;
      hipLaunchKernelGGL((down_tiles_kernel<T, C, RT, W>), dim3((unsigned)(((int64_t)a->rows + 15) / 16)), dim3(64 * W), 0, stream, p);
      return lq_check_launch();
    };
    if (!sv_fits(((int64_t)a->rows + 15) / 16, 512)) return (int)LQ_ERR_SHAPE;
    using std::integral_constant;
    switch (a->rank / 16) {
      case 1: return tiles(integral_constant<int, 1>{});
      case 2: return tiles(integral_constant<int, 2>{});
      case 3: return tiles(integral_constant<int, 3>{});
      case 4: return tiles(integral_constant<int, 4>{});
      case 5: return tiles(integral_constant<int, 5>{});
      case 6: return tiles(integral_constant<int, 6>{});
      case 7: return tiles(integral_constant<int, 7>{});
      default: return tiles(integral_constant<int, 8>{});
    }
  };
  auto with = [&](auto t) { return codes ? go(t, std::true_type{}) : go(t, std::false_type{}); };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
