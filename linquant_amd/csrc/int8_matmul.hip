// lq_int8_matmul: out[m,n] = (sum_k a[m,k] b[n,k]) * a_scale[m] * b_scale[n] + bias[n], INT8 in, the sum exact in 32 bits.
//
// Two kernels.  `tiles`: both operands go through LDS in stages of 128 contraction bytes, fetched straight from memory, and each wave has
// whole 32 x 32 tiles of the result.  `rows`: few rows of a (tokens that answer): a workgroup has 16 to 48 columns and its waves parts of
// the contraction, every operand straight to registers, so that the weights stream from memory once: 16 x 2560 x 10576 in 7.6 to
// 8.2 us by the kernel's own time, 3.4 to 3.6 TB/s.
//
// The matrix instruction of `tiles` is v_mfma_i32_32x32x32_i8, which reaches 4.9 POPS here where the 16x16x64 form reaches 3.0.  Operands:
// lane l has row l & 31 and the 16 contraction bytes of half l >> 5; the result: column l & 31, rows 8 (r >> 2) + 4 (l >> 5) + (r & 3).  b is
// the operand of the rows, so that a lane holds four adjacent columns of one row of `out`.
//
// What bounds `tiles`: the fetches and the way out.  A compute unit takes in 97 to 115 bytes/ns from its L2 in rows of 128 bytes (in rows of
// 64 half of that), a wave that waits to issue one issues no product either, and the result, twice the inputs at K = 2560, leaves at the
// memory's rate.  So a stage has one place in LDS and several workgroups share a compute unit: while one fetches or writes its result out,
// another multiplies.  32768 x 2560 x 10576: 913 to 1000 us by the card (1.94 to 1.77 POPS).  Rings of two to four stages with one workgroup of 256 x 256 to a compute
// unit, the next stages on their way during the products: 1120 to 1380 us; two workgroups of 128 x 256 with three stages of 64: 1080.
#include <algorithm>

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
  int vec;  // out's rows can be written 16 bytes at a time
};

struct F32 {
  using type = float;
  static LQ_DEV float from(float f) { return f; }
};
template <typename T>
struct OutOf {
  using type = uint16_t;
};
template <>
struct OutOf<F32> {
  using type = float;
};

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;

__device__ const lq_v4i zero16[1] = {{0, 0, 0, 0}};  // what a contraction past its end reads

constexpr int KB = 128, PC = KB / 16, FR = 64 / PC;  // contraction bytes of a stage, 16-byte pieces of its rows, rows of a fetch
// Piece c of a stage's row lies at place c ^ order(row): the 16 lanes that a read serves at once then touch each bank once.
LQ_DEV int order(int row) { return (row >> 1) & 7; }

// TM x TN of the result to KG groups of four waves, 2 x 2 of a tile; the groups have every KG-th stage each and are summed at the end.
template <int TM, int TN, int KG, typename O>
__global__ __launch_bounds__(256 * KG, KG == 1 && TM * TN <= 128 * 128 ? 3 : 2) void int8_tiles_kernel(MatmulParams p) {
  constexpr int MI = TM / 64, NI = TN / 64;          // 32-row tiles of a wave
  constexpr int PA = TM / FR / 4, PB = TN / FR / 4;  // fetches of a wave and stage
  constexpr int kStage = (TM + TN) * KB, SUB = KB / 32;
  constexpr int kOutRow = TN / 2 * (int)sizeof(typename OutOf<O>::type) + 16;  // bytes of a row of a wave's result on its way out
  constexpr int kLds = std::max(std::max(KG * kStage, 4 * 32 * kOutRow), KG / 2 * TM * TN * 4);
  __shared__ __align__(16) char lds[kLds];
  __shared__ __align__(16) float sb[2 * TN];  // the columns' scales and bias
  const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
  const int group = __builtin_amdgcn_readfirstlane(tid >> 8), wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
  // Workgroups go round the 8 XCDs in launch order; each XCD takes adjacent tiles of an order in which 32 of them are 8 x 4, so that what its
  // compute units read at one time is mostly the same and comes from its L2.
  const int nm = (p.rows + TM - 1) / TM, nn = (p.cols + TN - 1) / TN;
  int m0, n0;
  {
    const int i = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
    if (i >= nm * nn) return;
    const int band = i / (8 * nn), first = band * 8, high = min(8, nm - first), j = i - band * 8 * nn;
    m0 = (first + j % high) * TM, n0 = (j / high) * TN;
  }
  const int fr = lane / PC;
  uint32_t offa[PA], offb[PB];
  auto piece = [&](int row) { return 16 * ((lane & (PC - 1)) ^ order(row)); };
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int row = FR * (wave * PA + i) + fr;
    offa[i] = (uint32_t)min(row, p.rows - 1 - m0) * (uint32_t)p.a_stride + (uint32_t)piece(row);
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int row = FR * (wave * PB + i) + fr;
    offb[i] = (uint32_t)min(row, p.cols - 1 - n0) * (uint32_t)p.b_stride + (uint32_t)piece(row);
  }
  const int8_t* at = p.a + m0 * p.a_stride;
  const int8_t* bt = p.b + n0 * p.b_stride;
  const int ns = (p.inner + KB - 1) / KB;
  char* stage = lds + group * kStage;
  auto fetch = [&](int s) {
    const int8_t *as = at + s * KB, *bs = bt + s * KB;
    if ((s + 1) * KB <= p.inner) {
#pragma unroll
      for (int i = 0; i < PA; ++i) __builtin_amdgcn_global_load_lds((glb_void*)(as + offa[i]), (lds_void*)(stage + (wave * PA + i) * 1024), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < PB; ++i) __builtin_amdgcn_global_load_lds((glb_void*)(bs + offb[i]), (lds_void*)(stage + TM * KB + (wave * PB + i) * 1024), 16, 0, 0);
    } else {  // the last stage, cut short: zeros of either operand behind the contraction
      auto from = [&](const int8_t* q, uint32_t off, int row) { return s * KB + piece(row) < p.inner ? (const void*)(q + off) : (const void*)zero16; };
#pragma unroll
      for (int i = 0; i < PA; ++i)
        __builtin_amdgcn_global_load_lds((glb_void*)from(as, offa[i], FR * (wave * PA + i) + fr), (lds_void*)(stage + (wave * PA + i) * 1024), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < PB; ++i)
        __builtin_amdgcn_global_load_lds((glb_void*)from(bs, offb[i], FR * (wave * PB + i) + fr), (lds_void*)(stage + TM * KB + (wave * PB + i) * 1024), 16, 0, 0);
    }
  };
  const int wm = (wave >> 1) * (TM / 2), wn = (wave & 1) * (TN / 2);
  const int r0 = (lane & 31) * KB, x = order(lane & 31);
  auto read = [&](int k, lq_v4i (&fa)[MI], lq_v4i (&fb)[NI]) {
    const char* st = stage + r0 + (((2 * k + hh) ^ x) * 16);
#pragma unroll
    for (int i = 0; i < MI; ++i) fa[i] = *(const lq_v4i*)(st + (wm + 32 * i) * KB);
#pragma unroll
    for (int j = 0; j < NI; ++j) fb[j] = *(const lq_v4i*)(st + (TM + wn + 32 * j) * KB);
  };
  if (group < ns) fetch(group);
  float sa[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sa[i] = p.a_scale[p.a_scale_rows ? min(m0 + wm + 32 * i + (lane & 31), p.rows - 1) : 0];
  for (int i = tid; i < TN; i += 256 * KG) {
    const int n = min(n0 + i, p.cols - 1);
    sb[i] = p.b_scale[p.b_scale_cols ? n : 0];
    sb[TN + i] = p.bias ? sv_load(p.bias, n, p.bias_dtype) : 0.0f;
  }
  lq_v16i acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  auto multiply = [&](const lq_v4i (&fa)[MI], const lq_v4i (&fb)[NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
  };
  lq_v4i fa[2][MI], fb[2][NI];
  for (int s0 = 0; s0 < ns; s0 += KG) {
    const int s = s0 + group;
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");  // every wave's share of the stage has landed
    if (s < ns) {
      read(0, fa[0], fb[0]);
#pragma unroll
      for (int k = 0; k + 1 < SUB; ++k) {
        read(k + 1, fa[(k + 1) & 1], fb[(k + 1) & 1]);
        multiply(fa[k & 1], fb[k & 1]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave has read all of it
    if (s + KG < ns) fetch(s + KG);
    if (s < ns) multiply(fa[(SUB - 1) & 1], fb[(SUB - 1) & 1]);
  }
  // the groups' sums: each step halves how many there are, the upper ones' through LDS
  if constexpr (KG > 1) {
#pragma unroll
    for (int n = KG / 2; n >= 1; n /= 2) {
      int* at = (int*)lds + (group % n) * TM * TN + ((wave * 64 + lane) * 4);
      if (group >= n && group < 2 * n) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const lq_v4i v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
              *(lq_v4i*)(at + ((i * NI + j) * 4 + q) * 1024) = v;
            }
      }
      __syncthreads();
      if (group < n) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const lq_v4i v = *(const lq_v4i*)(at + ((i * NI + j) * 4 + q) * 1024);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
            }
      }
      __syncthreads();
    }
    if (group > 0) return;
  }
  // out: 32 rows of a wave's result at a time through LDS (nothing of it is read any more: the barrier behind the last stage's reads)
  using OT = typename OutOf<O>::type;
  char* my = lds + wave * 32 * kOutRow;
  OT* out = (OT*)p.out;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + wm + 32 * i;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = 32 * j + 8 * q + 4 * hh;
        const lq_v4f s4 = *(const lq_v4f*)(sb + wn + n), b4 = *(const lq_v4f*)(sb + TN + wn + n);
        typedef OT V4 __attribute__((ext_vector_type(4)));
        V4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = O::from(__builtin_fmaf((float)acc[i][j][4 * q + e], sa[i] * s4[e], b4[e]));
        *(V4*)(my + (lane & 31) * kOutRow + n * sizeof(OT)) = o;
      }
    // (a wave's LDS operations are in order)
    constexpr int kPieces = TN / 2 * (int)sizeof(OT) / 16, kRows = 64 / kPieces;  // 16-byte pieces of a row, rows written at a time
    constexpr int kPer = 16 / (int)sizeof(OT);
#pragma unroll
    for (int r = 0; r < 32; r += kRows) {
      const int row = r + lane / kPieces, pc = lane % kPieces, n = n0 + wn + pc * kPer;
      const lq_v4i v = *(const lq_v4i*)(my + row * kOutRow + pc * 16);
      if (m + row < p.rows) {
        OT* o = out + (m + row) * p.out_stride + n;
        if (p.vec && n + kPer <= p.cols) {
          *(lq_v4i*)o = v;
        } else {
          typedef OT VP __attribute__((ext_vector_type(kPer)));
          const VP e = __builtin_bit_cast(VP, v);
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (n + k < p.cols) o[k] = e[k];
        }
      }
    }
  }
}

// Few rows of a: 16 MT of them and 16 NT columns to a workgroup of W waves, which share the contraction in lines of 128 bytes, side by
// side (a wave that has a range of its own reads 8192 x 8192 a quarter slower).  The weights are read once, a's rows by every workgroup,
// and those cost as much: with 16 columns to a workgroup 16 x 2560 x 10576 takes 11.5 us, with one row of a 7.7.  So NT is taken such that
// there is one workgroup to a compute unit.  us, launch after launch in a graph (2 us above the kernel's own time), weights from memory, NT 1 / 2 / 3:
// 16 x 2560 x 10576 11.5 / 12.4 / 10.0, 64 rows 24.6 / 21.7 / 17.0, one row 7.7 / 10.3 / 8.7; 16 x 5120 x 2560, 160 tiles of 16 columns,
// 7.5 / 11.9 / 15.6.  Eight waves that request one line at a time are as good as any, but where results are many (MT 4, NT 2 or 3) four that
// request two: 64 x 2560 x 10576, NT 2: 21.7 and 22.7.
// v_mfma_i32_16x16x64_i8: lane l has row l & 15 and the 16 bytes of quarter l >> 4; the result: column l & 15, rows 4 (l >> 4) + r.
template <int MT, int NT, int W, int U, typename O>
__global__ __launch_bounds__(64 * W) void int8_rows_kernel(MatmulParams p) {
  __shared__ __align__(16) int sums[W][NT][MT][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * NT;
  const int8_t *b[NT], *a[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) b[j] = p.b + min(n0 + 16 * j + (lane & 15), p.cols - 1) * p.b_stride;
#pragma unroll
  for (int i = 0; i < MT; ++i) a[i] = p.a + min(16 * i + (lane & 15), p.rows - 1) * p.a_stride;
  lq_v4i acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = lq_v4i{0, 0, 0, 0};
  const int lines = (p.inner + 127) / 128;
  for (int s0 = wave; s0 < lines; s0 += W * U) {
    lq_v4i fb[U][2][NT], fa[U][2][MT];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + W * u < lines) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kc = min((s0 + W * u) * 128 + 64 * h + (lane >> 4) * 16, p.inner - 16);
#pragma unroll
          for (int j = 0; j < NT; ++j) fb[u][h][j] = *(const lq_v4i*)(b[j] + kc);
#pragma unroll
          for (int i = 0; i < MT; ++i) fa[u][h][i] = *(const lq_v4i*)(a[i] + kc);
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + W * u < lines) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = (s0 + W * u) * 128 + 64 * h + (lane >> 4) * 16 < p.inner;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            if (!in) fa[u][h][i] = lq_v4i{0, 0, 0, 0};  // (a zero of one operand is enough)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j][i] = lq_mfma_i8(fb[u][h][j], fa[u][h][i], acc[j][i]);
          }
        }
      }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) *(lq_v4i*)sums[wave][j][i][lane] = acc[j][i];
  __syncthreads();
  using OT = typename OutOf<O>::type;
  OT* out = (OT*)p.out;
  for (int t = threadIdx.x; t < NT * MT * 256; t += 64 * W) {  // adjacent threads: adjacent columns
    const int n = t & 15, j = (t >> 4) % NT, m = (t >> 4) / NT & 15, i = (t >> 4) / NT >> 4;
    int v = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) v += sums[w][j][i][(n >> 2) * 16 + m][n & 3];
    const int row = 16 * i + m, col = n0 + 16 * j + n;
    if (row < p.rows && col < p.cols) {
      const float s = p.a_scale[p.a_scale_rows ? row : 0] * p.b_scale[p.b_scale_cols ? col : 0];
      out[row * p.out_stride + col] = O::from(__builtin_fmaf((float)v, s, p.bias ? sv_load(p.bias, col, p.bias_dtype) : 0.0f));
    }
  }
}

template <typename O>
int launch(const MatmulParams& p, hipStream_t stream) {
  using std::integral_constant;
  if (p.rows <= 64) {
    if (!sv_fits(((int64_t)p.cols + 15) / 16, 512)) return LQ_ERR_SHAPE;
    const int mt = (p.rows + 15) / 16;
    // most tiles of 16 columns that a compute unit gets, n to a workgroup
    auto most = [&](int n) { return ((p.cols + 16 * n - 1) / (16 * n) + 255) / 256 * n; };
    const int nt = most(3) <= std::min(most(1), most(2)) ? 3 : (most(2) <= most(1) ? 2 : 1);
    auto go = [&](auto m, auto n) {
      constexpr int MT = decltype(m)::value, NT = decltype(n)::value, W = MT == 4 && NT > 1 ? 4 : 8;
      hipLaunchKernelGGL((int8_rows_kernel<MT, NT, W, 8 / W, O>), dim3((unsigned)((p.cols + 16 * NT - 1) / (16 * NT))), dim3(64 * W), 0, stream, p);
    };
    auto columns = [&](auto m) { nt == 1 ? go(m, integral_constant<int, 1>{}) : (nt == 2 ? go(m, integral_constant<int, 2>{}) : go(m, integral_constant<int, 3>{})); };
    mt == 1 ? columns(integral_constant<int, 1>{}) : (mt == 2 ? columns(integral_constant<int, 2>{}) : columns(integral_constant<int, 4>{}));
    return lq_check_launch();
  }
  auto tiles = [&](auto tm, auto tn, auto kg) {
    constexpr int TM = decltype(tm)::value, TN = decltype(tn)::value, KG = decltype(kg)::value;
    const int64_t n = (((int64_t)p.rows + TM - 1) / TM) * (((int64_t)p.cols + TN - 1) / TN);
    if (!sv_fits(n + 7, 256 * KG)) return LQ_ERR_SHAPE;
    hipLaunchKernelGGL((int8_tiles_kernel<TM, TN, KG, O>), dim3((unsigned)((n + 7) / 8 * 8)), dim3(256 * KG), 0, stream, p);
    return lq_check_launch();
  };
  auto count = [&](int tm, int tn) { return (((int64_t)p.rows + tm - 1) / tm) * (((int64_t)p.cols + tn - 1) / tn); };
  // The larger a tile, the less is fetched; the more tiles, the more compute units fetch, and two or three workgroups must share each.  Where
  // even small tiles are few, groups share their contraction.  us, rows x K x columns, for tiles of 128 x 256 / 128 x 128 / 64 x 128 in two
  // groups / 64 x 64 in four: 8192 x 2560 x 10576 248 / 249 / 329 / 428, 3001 x 2560 x 10576 92 / 99 / 122 / 162, 1000 x 2560 x 10576 42 / 40 /
  // 47 / 57, 2000 x 5120 x 2560 62 / 44 / 52 / 51, 1000 x 5120 x 2560 60 / 41 / 28 / 34, 300 x 2560 x 10576 34 / 24 / 19 / 23, 500 x 5120 x 2560
  // 60 / 41 / 26 / 20, 100 x 5120 x 2560 46 / 30 / 19 / 17.
  if (count(128, 256) >= 768) return tiles(integral_constant<int, 128>{}, integral_constant<int, 256>{}, integral_constant<int, 1>{});
  if (count(128, 128) >= 300) return tiles(integral_constant<int, 128>{}, integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (count(64, 64) > 512) return tiles(integral_constant<int, 64>{}, integral_constant<int, 128>{}, integral_constant<int, 2>{});
  return tiles(integral_constant<int, 64>{}, integral_constant<int, 64>{}, integral_constant<int, 4>{});
}

}  // namespace

extern "C" int lq_int8_matmul(const lq_int8_matmul_args* a, hipStream_t stream) {
  if (!a || !a->a || !a->b || !a->a_scale || !a->b_scale || !a->out) return LQ_ERR_NULL;
  if (a->rows <= 0 || a->cols <= 0 || a->inner <= 0 || a->inner % 16 != 0 || a->inner > 131056) return LQ_ERR_SHAPE;
  if (!sv_float(a->out_dtype) || (a->bias && !sv_float(a->bias_dtype))) return LQ_ERR_SHAPE;
  if (a->a_stride % 16 != 0 || a->b_stride % 16 != 0 || !sv_al(a->a, 16) || !sv_al(a->b, 16)) return LQ_ERR_SHAPE;
  if (a->a_stride < 0 || a->a_stride >= 1 << 23 || a->b_stride < 0 || a->b_stride >= 1 << 23) return LQ_ERR_SHAPE;  // a tile's rows are reached by 32-bit offsets
  if (!sv_al(a->out, sv_size(a->out_dtype)) || (a->bias && !sv_al(a->bias, sv_size(a->bias_dtype))) || !sv_al(a->a_scale, 4) || !sv_al(a->b_scale, 4))
    return LQ_ERR_SHAPE;
  const int per = 16 / sv_size(a->out_dtype);
  MatmulParams p = {a->a, a->a_stride, a->b, a->b_stride, a->a_scale, a->b_scale, a->a_scale_rows, a->b_scale_cols, a->bias, a->bias_dtype,
                    a->out, a->out_stride, a->rows, a->cols, a->inner, sv_al(a->out, 16) && a->out_stride % per == 0};
  if (a->out_dtype == LQ_DT_F32) return launch<F32>(p, stream);
  return a->out_dtype == LQ_DT_F16 ? launch<F16>(p, stream) : launch<BF16>(p, stream);
}
