// lq_adapter_down: the first half of low-rank adapters of many requests, h[m] = scaling[j] * (down[j] x[m]), j = ids[m], in fp32; the second
// half is the epilogue of lq_int8_matmul.
//
// Three kernels.  `rows`, few rows, each with a request of its own as a rule: a wave has two of a row's sums, so that the adapters stream
// from memory through many waves; the quantizer of the rows, if the call has one, runs in the same launch.  16 rows of 2560 entries, rank 16,
// 16 adapters, with the quantizer: 4.0 us, where the launch of an empty kernel takes 2.
// `staged`, and `tiles` for rows that are no whole 16-byte pieces: 16 rows of x to a workgroup, its waves share the contraction, and what meets
// the rows are the matrix instructions; the adapters that the 16 rows name are taken one after the other, each with all 16 rows, and a row keeps
// what its own gave (nothing is multiplied by zero: an infinity in one request's row or adapter stays there).  The bound is memory: 16384 rows of
// 2560 in 16 bits, 84 MB, rank 16, in 18 us 4.7 TB/s (some of it from the cache behind HBM, where the quantizer left it); 3001 rows of 5120 codes, rank 32, 14 us,
// where a workgroup's 10 stages one after the other are what it waits for.
// Rows that name adapters in turn would cost as many passes as there are adapters, so they are taken in an order (below).  us, 310 rows of 5120
// codes, rank 8, 8 adapters in turn: 44 in their own order, 13 ordered, 7 if all name one (and by `rows` 7); 1171 of 4096, rank 64, 16 adapters: 165, 29, 12.
// v_mfma_f32_16x16x32: lane l has row l & 15 and the 8 contraction entries of quarter l >> 4; the result: column l & 15, rows 4 (l >> 4) + r.
// down is the operand of the rows, so that a lane holds four adjacent sums of one row of x.
//
// INT8 codes become 16 bits exactly; their scale multiplies the sum.  All sums are fp32.
#include <algorithm>

#include "row_codes.h"

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
  int8_t* codes_out;  // NULL, or x's codes and scales as well
  float* scale_out;
  int32_t* order;  // NULL, or an order of the rows
};

// An order of the rows in which those that name one adapter lie together, within windows of 64 W rows; one thread has one row.  What a
// tile of 16 rows costs here, and one of 32 in the product's epilogue, is one pass for each adapter that it names.  A window with few changes
// between neighbours stays as it is.  Groups lie in the order of their first rows, a group's rows in their own: the same for the same ids, always.
constexpr int kWindow = 512, kFewChanges = 16;
template <int W>
struct Order {
  int key[64 * W], first[64 * W], start[W][64 * W], part[W];
};
template <int W>
LQ_DEV int window_place(const int32_t* ids, int n, int count, Order<W>& o) {  // the place of the window's row `threadIdx.x`; n: rows of the window
  constexpr int N = 64 * W;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const bool in = t < n;
  const int key = in ? max(-1, min(ids[t], count)) : -2;
  o.key[t] = key, o.first[t] = N;
#pragma unroll
  for (int w = 0; w < W; ++w) o.start[w][t] = 0;
  __syncthreads();
  if (__syncthreads_count(in && t > 0 && o.key[t - (t > 0)] != key) <= kFewChanges) return t;
  uint64_t same = 0;  // the wave's rows with this key
  for (uint64_t left = __ballot(in); left;) {
    const int k = __builtin_amdgcn_readlane(key, __builtin_ctzll(left));
    const uint64_t m = __ballot(key == k);
    if (key == k) same = m;
    left &= ~m;
  }
  const bool leads = in && __builtin_ctzll(same) == lane;
  // the key's first row in the window: at a place of the table that the key names; who finds another key's there tries others
  int first = -1;
  for (int round = 0;; ++round) {
    const int at = round == 0 ? key & (N - 1) : (int)(((uint32_t)key * (0x9e3779b1u + 2u * round)) >> 16) & (N - 1);
    if (leads && first < 0) atomicMin(&o.first[at], t);
    __syncthreads();
    if (leads && first < 0 && o.key[o.first[at]] == key) first = o.first[at];
    const bool open = __syncthreads_or(leads && first < 0);
    if (!open) break;
    o.first[t] = N;
    __syncthreads();
  }
  if (leads) o.start[wave][first] = __builtin_popcountll(same);
  __syncthreads();
  int rows[W], sum = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) rows[w] = o.start[w][t], sum += rows[w];
  int upto = sum;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(upto, off, 64);
    if (lane >= off) upto += v;
  }
  if (lane == 63) o.part[wave] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < wave; ++w) at += o.part[w];
#pragma unroll
  for (int w = 0; w < W; ++w) o.start[w][t] = at, at += rows[w];
  __syncthreads();
  const int f = __shfl(first, same ? __builtin_ctzll(same) : lane, 64);
  return in ? o.start[wave][f] + __builtin_popcountll(same & ((1ull << lane) - 1)) : t;
}
// The rows of the 16 places from m0 on, to LDS
template <int W>
LQ_DEV void ordered_rows(const DownParams& p, int m0, Order<W>& o, int (&rows)[16]) {
  const int w0 = m0 / (64 * W) * (64 * W), n = min(64 * W, p.rows - w0), i = w0 + window_place<W>(p.ids + w0, n, p.count, o) - m0, row = w0 + (int)threadIdx.x;
  if ((int)threadIdx.x < n && i >= 0 && i < 16) rows[i] = row;
  __syncthreads();
}

template <typename T>
LQ_DEV lq_v4f mfma16(lq_v4i a, lq_v4i b, lq_v4f c) {
  if constexpr (std::is_same<T, F16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lq_v8h, a), __builtin_bit_cast(lq_v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sv_v8bf, a), __builtin_bit_cast(sv_v8bf, b), c, 0, 0, 0);
}

// Eight codes in T, exactly: nothing is rounded, so bits may be cut off
template <typename T>
LQ_DEV lq_v4i from_codes(lq_v2i r) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)lq_sbyte((uint32_t)r[e >> 2], e & 3);
  lq_v4i o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, F16>::value) o[i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_pkrtz(f[2 * i], f[2 * i + 1]));
    else o[i] = (int)__builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302);
  }
  return o;
}
// Eight entries of a row from `k` on in T, zero behind the row's end.  EIGHTS: rows of whole eights on boundaries of eight entries, of which the
// last are read again behind the end; else one by one.
template <typename T, bool CODES, bool EIGHTS>
LQ_DEV lq_v4i load8(const void* row, int k, int inner) {
  if constexpr (EIGHTS && !CODES) {
    const lq_v4i zero = {0, 0, 0, 0}, r = *(const lq_v4i*)((const uint16_t*)row + min(k, inner - 8));
    return k < inner ? r : zero;
  } else {
    if constexpr (EIGHTS) {
      lq_v2i r = *(const lq_v2i*)((const int8_t*)row + min(k, inner - 8));
      if (k >= inner) r = lq_v2i{0, 0};
      return from_codes<T>(r);
    }
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = min(k + e, inner - 1);
      uint16_t u;
      if constexpr (CODES) u = T::from((float)((const int8_t*)row)[at]);
      else u = ((const uint16_t*)row)[at];
      v[e] = k + e < inner ? u : 0;
    }
    lq_v4i o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (int)(v[2 * i] | (uint32_t)v[2 * i + 1] << 16);
    return o;
  }
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

// QV: 0, or the workgroups in front of the others quantize the rows, each thread 8 QV entries of one
template <typename T, bool CODES, bool EIGHTS, int QV>
__global__ __launch_bounds__(256) void down_rows_kernel(DownParams p) {
  int m = blockIdx.x, lane = threadIdx.x & 63;
  if (p.order) {  // the first workgroups: the order
    const int windows = (p.rows + 255) / 256, w0 = m * 256;
    if (m < windows) {
      __shared__ Order<4> o;
      const int n = min(256, p.rows - w0), at = window_place<4>(p.ids + w0, n, p.count, o);
      if ((int)threadIdx.x < n) p.order[w0 + at] = w0 + (int)threadIdx.x;
      return;
    }
    m -= windows;
  }
  if constexpr (QV > 0) {
    if (m < p.rows) {
      __shared__ float lds[4];
      float v[8 * QV];
      Row<T, QV, 256, true>::load(p.x, m * p.x_stride, p.inner, threadIdx.x, v);
      row_codes<QV, 256, true>(p.scale_out + m, p.codes_out, (int64_t)m * p.inner, p.inner, threadIdx.x, v, lds, 0);
      return;
    }
    m -= p.rows;
  }
  const int groups = (p.rank + 4 * kPer - 1) / (4 * kPer), r0 = (m % groups * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kPer;
  m /= groups;
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
      xv[u] = load8<T, CODES, EIGHTS>(x, k, p.inner);
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

// the waves' sums together, and out
template <bool CODES, int RT, int W>
LQ_DEV void down_finish(const DownParams& p, int m0, const int (&rows)[16], const lq_v4f (&keep)[RT], lq_v4f (&sums)[W][RT][64]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p.order && threadIdx.x < 16 && m0 + (int)threadIdx.x < p.rows) p.order[m0 + threadIdx.x] = rows[threadIdx.x];
#pragma unroll
  for (int t = 0; t < RT; ++t) sums[wave][t][lane] = keep[t];
  __syncthreads();
  for (int i = threadIdx.x; i < RT * 64; i += 64 * W) {
    const int t = i >> 6, l = i & 63;
    lq_v4f v = sums[0][t][l];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][t][l];
    if (m0 + (l & 15) >= p.rows) continue;
    const int row = rows[l & 15];
    const int own = p.ids[row];
    const float f = own >= 0 && own < p.count ? factor<CODES>(p, row, own) : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= f;
    *(lq_v4f*)(p.h + (int64_t)row * p.rank + 16 * t + 4 * (l >> 4)) = v;
  }
}

// RT tiles of 16 sums; W waves share the contraction in lines of 64 entries, side by side, U of them requested at a time
template <typename T, bool CODES, bool EIGHTS, int RT, int W>
__global__ __launch_bounds__(64 * W) void down_tiles_kernel(DownParams p) {
  constexpr int U = RT <= 2 ? 4 : RT <= 4 ? 2 : 1;
  __shared__ __align__(16) lq_v4f sums[W][RT][64];
  __shared__ Order<W> order;
  __shared__ int rows[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
  const int m0 = blockIdx.x * 16;
  ordered_rows<W>(p, m0, order, rows);
  const int m = rows[min(lane & 15, p.rows - 1 - m0)];
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
    for (int k0 = wave * 64; k0 < p.padded; k0 += 64 * W * U) {
      lq_v4i xv[U][2], dv[U][2][RT];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = k0 + 64 * W * u + 32 * h + 8 * quarter;
          xv[u][h] = load8<T, CODES, EIGHTS>(x, k, p.inner);
#pragma unroll
          for (int t = 0; t < RT; ++t) dv[u][h][t] = *(const lq_v4i*)(d + (int64_t)16 * t * p.padded + min(k, p.padded - 8));
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            if (k0 + 64 * W * u + 32 * h + 8 * quarter >= p.padded) dv[u][h][t] = lq_v4i{0, 0, 0, 0};  // (an infinity of the row's last)
            acc[t] = mfma16<T>(dv[u][h][t], xv[u][h], acc[t]);
          }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sv_settle(acc[t]);
      if (mine) keep[t] = acc[t];
    }
  }
  down_finish<CODES, RT, W>(p, m0, rows, keep, sums);
}

// The same, x and down through LDS in stages of SE entries, each row's whole 16-byte pieces fetched side by side: as operands they are read
// from memory 64 bytes of a row at a time, at half the rate.  Piece c of row r lies at place c ^ r % 16, so that the 16 rows that a read serves
// at once touch each bank once.  ST places, of which all but one are filled while that one is multiplied.
template <typename T, bool CODES, int RT>
struct Staged {
  static constexpr int SE = RT <= 2 ? 512 : 256, bytes = (16 * (CODES ? 1 : 2) + RT * 16 * 2) * SE, deep = std::min(4, 150 * 1024 / bytes);
};
template <typename T, bool CODES, int RT, int ST>
__global__ __launch_bounds__(512) void down_staged_kernel(DownParams p) {
  constexpr int W = 8, SE = Staged<T, CODES, RT>::SE, XB = SE * (CODES ? 1 : 2), DB = SE * 2;  // bytes of a stage's row of x and of down
  constexpr int XR = 1024 / XB, DR = 1024 / DB;                             // rows of a fetch
  constexpr int XF = 16 / XR, DF = RT * 16 / DR, kStage = 16 * XB + RT * 16 * DB;  // fetches of a stage
  constexpr int XW = (XF + W - 1) / W, DW = (DF + W - 1) / W;               // of each wave (of those left over the last one again)
  constexpr int H = SE / (32 * W);                                          // products of a wave and stage
  static_assert(2 * kStage >= W * RT * 1024 && 2 * kStage >= sizeof(Order<W>) && kWindow == 64 * W && kStage == Staged<T, CODES, RT>::bytes);
  __shared__ __align__(1024) char lds[ST][kStage];
  __shared__ int rows[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4, r16 = lane & 15;
  const int m0 = blockIdx.x * 16, w0 = m0 / kWindow * kWindow;
  ordered_rows<W>(p, m0, *(Order<W>*)lds, rows);
  auto row_at = [&](int i) { return rows[min(i, min(15, p.rows - 1 - m0))]; };
  const int m = row_at(r16);
  const int id = p.ids[m];
  const char* x = (const char*)p.x + w0 * p.x_stride * (CODES ? 1 : 2);  // (the window's rows by 32-bit offsets)
  // a wave's fetches: the i-th one's number, this lane's row and piece of it
  struct Piece { int fetch, row, at; };
  auto of_x = [&](int i) { const int f = min(i * W + wave, XF - 1), row = f * XR + lane / (64 / XR); return Piece{f, row, ((lane % (64 / XR)) ^ (row & 15)) * 16}; };
  auto of_down = [&](int i) { const int f = min(i * W + wave, DF - 1), row = f * DR + lane / (64 / DR); return Piece{f, row, ((lane % (64 / DR)) ^ (row & 15)) * 16}; };
  uint32_t xoff[XW], doff[DW];
#pragma unroll
  for (int i = 0; i < XW; ++i) xoff[i] = (uint32_t)(row_at(of_x(i).row) - w0) * (uint32_t)p.x_stride * (CODES ? 1u : 2u) + of_x(i).at;
#pragma unroll
  for (int i = 0; i < DW; ++i) doff[i] = (uint32_t)of_down(i).row * (uint32_t)p.padded * 2u + of_down(i).at;
  lq_v4f keep[RT];
  const float none = id < 0 ? 0.0f : __builtin_nanf("");
#pragma unroll
  for (int t = 0; t < RT; ++t) keep[t] = lq_v4f{none, none, none, none};
  const int stages = (p.inner + SE - 1) / SE, xlast = (p.inner - (CODES ? 16 : 8)) * (CODES ? 1 : 2), dlast = (p.padded - 8) * 2;
  uint64_t left = __ballot(id >= 0 && id < p.count);
  while (left) {
    const int j = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const bool mine = id == j;
    left &= ~__ballot(mine);
    const char* d = (const char*)(p.down + (int64_t)j * p.rank * p.padded);
    auto fetch = [&](int s) {
      char* to = lds[s % ST];
      const bool whole = (s + 1) * SE <= p.inner;  // (else behind a row's end its last piece again: down is zero there as an operand)
#pragma unroll
      for (int i = 0; i < XW; ++i)
        sv_fetch16(x + s * XB, xoff[i] - (whole ? 0u : (uint32_t)max(s * XB + of_x(i).at - xlast, 0)), to + of_x(i).fetch * 1024);
#pragma unroll
      for (int i = 0; i < DW; ++i)
        sv_fetch16(d + s * DB, doff[i] - (whole ? 0u : (uint32_t)max(s * DB + of_down(i).at - dlast, 0)), to + 16 * XB + of_down(i).fetch * 1024);
    };
    lq_v4f acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = lq_v4f{0.f, 0.f, 0.f, 0.f};
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (from here on only fetches are counted)
    for (int s = 0; s < min(ST - 1, stages); ++s) fetch(s);
    for (int s = 0; s < stages; ++s) {
      // the stage is there, and the one in front of it is read (fetches end in order: all but those of the ST - 2 stages behind it)
      if (s + ST - 2 < stages) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((ST - 2) * (XW + DW)) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const char* st = lds[s % ST];
      // A fetch takes some 100 cycles to go out: behind the operands' reads if they are few.  3001 rows of 5120 codes, rank 32, 14.3 us, in front
      // 15.0; 1171 of 4096, rank 64, 12.6 and 11.4.
      auto ahead = [&] { if (s + ST - 1 < stages) fetch(s + ST - 1); };
      if constexpr (RT > 2) ahead();
      lq_v2i xc[H];
      lq_v4i xv[H], dv[H][RT];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int k = (wave * H + h) * 32 + 8 * quarter;  // of the stage
        if constexpr (CODES) xc[h] = *(const lq_v2i*)(st + r16 * XB + (((k >> 4) ^ r16) << 4) + (k & 8));
        else xv[h] = *(const lq_v4i*)(st + r16 * XB + (((k >> 3) ^ r16) << 4));
#pragma unroll
        for (int t = 0; t < RT; ++t) dv[h][t] = *(const lq_v4i*)(st + 16 * XB + (16 * t + r16) * DB + (((k >> 3) ^ r16) << 4));
      }
      if constexpr (RT <= 2) ahead();
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const bool in = s * SE + (wave * H + h) * 32 + 8 * quarter < p.inner;
        if constexpr (CODES) xv[h] = from_codes<T>(xc[h]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (!in) dv[h][t] = lq_v4i{0, 0, 0, 0};
          acc[t] = mfma16<T>(dv[h][t], xv[h], acc[t]);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sv_settle(acc[t]);
      if (mine) keep[t] = acc[t];
    }
  }
  down_finish<CODES, RT, W>(p, m0, rows, keep, *(lq_v4f(*)[W][RT][64])lds);  // (nothing of a stage is read any more)
}

// How many rows `rows` takes: their adapters are read for each, at the caches' rate.  Whole calls, us, 2560 entries to 1024 columns, one adapter / 16 in
// turn, `rows` and `staged`: rank 16, 256 rows 16 / 16 and 20 / 22, 1024 21 / 22 and 21 / 24; rank 64, 256 rows 22 / 24 and 25 / 29, 512 28 / 30 and
// 26 / 29.  From codes, where there is no quantizer to take along: rank 16, 512 rows 15 / 16 and 15 / 17, 1024 18 / 20 and 15 / 18; rank 32, 320 rows
// 16 / 20 and 16 / 22, 512 18 / 20 and 16 / 19.
int few_rows(int rank, bool codes) { return std::max(256, (codes ? 8192 : 16384) / rank); }

}  // namespace

extern "C" int lq_adapter_down(const lq_adapter_down_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->down || !a->scaling || !a->ids || !a->h || (a->x_dtype == LQ_DT_I8 && !a->x_scale)) return LQ_ERR_NULL;
  if (!sv_act(a->dtype) || (a->x_dtype != a->dtype && a->x_dtype != LQ_DT_I8)) return LQ_ERR_SHAPE;
  if (a->rows <= 0 || a->inner <= 0 || a->inner_padded < a->inner || a->inner_padded % 16 != 0 || a->count <= 0) return LQ_ERR_SHAPE;
  if (a->rank <= 0 || a->rank % 16 != 0 || a->rank > 128) return LQ_ERR_SHAPE;
  const bool codes = a->x_dtype == LQ_DT_I8;
  // (rows that are not whole eights of entries are read one by one)
  if (a->inner % 8 == 0 ? !sv_al(a->x, codes ? 8 : 16) || a->x_stride % 8 != 0 : !sv_al(a->x, codes ? 1 : 2)) return LQ_ERR_SHAPE;
  if (!sv_al(a->down, 16) || !sv_al(a->h, 16) || !sv_al(a->x_scale, 4) || !sv_al(a->scaling, 4) || !sv_al(a->ids, 4) || !sv_al(a->order, 4))
    return LQ_ERR_SHAPE;
  DownParams p = {a->x, a->x_stride, a->x_scale, a->x_scale_rows, (const uint16_t*)a->down, a->scaling, a->ids, a->h, a->rows, a->inner, a->inner_padded, a->rank, a->count,
                  a->codes_out, a->scale_out, a->order};
  const bool eights = a->inner % 8 == 0;
  if (a->codes_out && (!a->scale_out || codes || !eights || a->inner > 16384 || !sv_al(a->codes_out, 8) || !sv_al(a->scale_out, 4))) return LQ_ERR_SHAPE;
  using std::integral_constant;
  auto rows = [&](auto t, auto c, auto e, auto qv) {
    const int64_t wgs = (int64_t)a->rows * ((a->rank + 4 * kPer - 1) / (4 * kPer)) + (decltype(qv)::value ? a->rows : 0) + (a->order ? (a->rows + 255) / 256 : 0);
    hipLaunchKernelGGL((down_rows_kernel<decltype(t), decltype(c)::value, decltype(e)::value, decltype(qv)::value>), dim3((unsigned)wgs), dim3(256), 0, stream, p);
    return lq_check_launch();
  };
  auto go = [&](auto t, auto c, auto e) {
    using T = decltype(t);
    constexpr bool C = decltype(c)::value, E = decltype(e)::value;
    if constexpr (!C && E) {
      if (a->codes_out && a->rows <= few_rows(a->rank, codes)) {
        if (a->inner <= 2048) return rows(t, c, e, integral_constant<int, 1>{});
        if (a->inner <= 4096) return rows(t, c, e, integral_constant<int, 2>{});
        if (a->inner <= 8192) return rows(t, c, e, integral_constant<int, 4>{});
        return rows(t, c, e, integral_constant<int, 8>{});
      }
      if (a->codes_out) {
        lq_quantize_rows_args q = {a->x, a->x_stride, a->x_dtype, a->codes_out, a->inner, a->scale_out, a->rows, a->inner};
        const int rc = lq_quantize_rows(&q, stream);
        if (rc != LQ_OK) return rc;
      }
    }
    if (a->rows <= few_rows(a->rank, codes)) return rows(t, c, e, integral_constant<int, 0>{});
    // whole 16-byte pieces of both
    const bool pieces = E && a->inner % (C ? 16 : 8) == 0 && a->x_stride % (C ? 16 : 8) == 0 && sv_al(a->x, 16) && a->x_stride >= 0 && a->x_stride < 1 << 22;
    auto tiles = [&](auto rt) {
      constexpr int RT = decltype(rt)::value, W = RT <= 4 ? 8 : 4;
      if (pieces) {
        // Where a compute unit has one workgroup at most, that one has more of its stages on their way: 1171 rows of 4096 codes, rank 64, one
        // adapter 11.9 us, with two places 13.9, 16 adapters in turn 30.5 and 36.7; 3001 of 5120, rank 32, 16.1 and 16.8.
        const dim3 grid((unsigned)(((int64_t)a->rows + 15) / 16)), threads(512);
        if (grid.x <= 256) hipLaunchKernelGGL((down_staged_kernel<T, C, RT, Staged<T, C, RT>::deep>), grid, threads, 0, stream, p);
        else hipLaunchKernelGGL((down_staged_kernel<T, C, RT, 2>), grid, threads, 0, stream, p);
        return lq_check_launch();
      }
      hipLaunchKernelGGL((down_tiles_kernel<T, C, E, RT, W>), dim3((unsigned)(((int64_t)a->rows + 15) / 16)), dim3(64 * W), 0, stream, p);
      return lq_check_launch();
    };
    if (!sv_fits(((int64_t)a->rows + 15) / 16, 512)) return (int)LQ_ERR_SHAPE;
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
  auto with = [&](auto t, auto c) { return eights ? go(t, c, std::true_type{}) : go(t, c, std::false_type{}); };
  auto typed = [&](auto t) { return codes ? with(t, std::true_type{}) : with(t, std::false_type{}); };
  return a->dtype == LQ_DT_F16 ? typed(F16{}) : typed(BF16{});
}
