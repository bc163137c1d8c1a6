// lq_ssm_prompt: the selective state space scan over prompts of any lengths, from and into an fp32 state.
//   S_t = exp(d_t A) S_{t-1} + d_t x_t B_t^T,   y_t = S_t C_t + D x_t
// in chunks of 64 tokens.  With c_t = sum of d A up to t inside a chunk and S the state in front of it,
//   y_t = exp(c_t) S C_t + sum_{s <= t} exp(c_t - c_s) d_s (C_t . B_s) x_s + D x_t
//   S'  = exp(c_63) S + sum_s exp(c_63 - c_s) d_s x_s B_s^T
// which are products of matrices.  Three kernels:
//   operands   per chunk and group: C, B^T and C B^T in the order in which the matrix instruction takes them, shared by the group's
//              heads; per chunk and head: d, c (in powers of two) and exp(c_63 - c_s) d_s
//   states     per segment of a prompt, or piece of one: the state at its end if it starts from zero, and what it multiplies an earlier
//              one by;
//   join       walks the segments: the state in front of each.  (states and join: only where prompts are cut into segments, because
//              prompts times heads are too few for 256 compute units)
//   chunks     walks a segment chunk by chunk, the state in registers
//
// Precision.  Activations enter the matrix products as they are, all sums are fp32, and so is the state.  What is formed in fp32 on the way
// and reaches only y, which is rounded to the activations' type itself (weighted C B^T, the state that C multiplies), enters rounded to
// that type, to the nearest: half a step of each term.  What the state gathers over a prompt (weighted x) enters as two pieces of the type:
// off by 2^-18 of itself (bf16) or 2^-22 (fp16).  bf16 has the range of fp32.  fp16: after a multiplication by a power of two that brings the
// largest of what is multiplied (a channel's state; its state and weighted x; a row of weighted C B^T) below 2^14, so no size of
// activations overflows.  Below 2^-14 fp16 is evenly spaced: a state or weight 2^27 below its largest starts to lose bits, weighted x
// (whose second piece is 2^11 smaller) 2^16 below its channel's.  A unit for 32 channels and 64 tokens together (2 % less time) lost a
// channel beside one 2^26 above it, and the state that a chunk's first tokens read where a later one was as far above them.
//
// What bounds it.  4 prompts of 8192 tokens, 80 heads of 64 channels, 128 state columns, fp16: 408 to 426 us by the card, call after
// call (the kernels' own least times: operands 27, states 99, join 16, chunks 287; the profiler's medians are up to 14 % above them), 1.7 TB/s of
// what has to move and 254 to 265 TFLOP/s of the recurrence's operations.  In the last kernel the vector unit is
// busy 53 % of the time (scaling, rounding and splitting operands, 774 instructions to 32 channels and 64 tokens), the matrix unit 22 %, and
// the clock falls from 2.4 to 2.1 GHz; two waves to a SIMD is what the state in registers (64 of 256) and 81 KB of LDS leave.  Few or
// ragged prompts are a chain of chunks, about 4 us each: 384 tokens 36 us, 6949 in 10 prompts of up to 2047, 64 heads in 8 groups, bf16, 140.
// Tried: C B^T formed by each workgroup (its product is the group's, so 80 heads made it 80 times); one piece of a state's additions (a state
// gathers the rounding of a whole prompt); a higher priority for the younger of two workgroups, which the older one holds up (3 % less here,
// 3 % more for ragged prompts).
#include <algorithm>
#include <cmath>

#include "serve_common.h"

namespace {

constexpr int Q = 64;             // tokens of a chunk
constexpr int kCB = 6 * 2 * 1024;  // bytes of a chunk's C B^T: six operands (32 rows, 16 tokens) on and below the diagonal, fp32
constexpr float kLog2e = 1.44269504088896340736f;

struct PromptParams {
  const uint16_t* x;
  int64_t sx_b, sx_l, sx_h;
  const void* dt;
  int64_t sdt_b, sdt_l, sdt_h;
  int dt_dtype;
  const float* A;
  const uint16_t* B;
  int64_t sB_b, sB_l, sB_g;
  const uint16_t* C;
  int64_t sC_b, sC_l, sC_g;
  const float* D;
  int D_has_hdim;
  const float* dt_bias;
  int softplus;
  float dt_min, dt_max;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, H, P, G, N;
  // workspace
  char* tables;     // [unit][group] operands
  float* steps;     // [unit][head][d, c, w, most][64]
  float* rows;      // [unit][group][64]: largest |C B^T| of each row
  float* seg_state;  // [segment][piece][H][P][N], or NULL: prompts are not cut
  float* seg_decay;  // [segment][piece][H]
  int units, segs, seg_chunks, pieces, per_group;  // (seg_chunks a multiple of pieces)
};

typedef float v16f __attribute__((ext_vector_type(16)));
template <typename T>
LQ_DEV v16f mfma(lq_v4i a, lq_v4i b, v16f c) {
  if constexpr (std::is_same<T, F16>::value) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lq_v8h, a), __builtin_bit_cast(lq_v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(sv_v8bf, a), __builtin_bit_cast(sv_v8bf, b), c, 0, 0, 0);
}
LQ_DEV uint32_t pack_bf16(float a, float b) {
  const sv_v2bf v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
// eight numbers, or products, rounded to T
template <typename T>
LQ_DEV lq_v4i round8(const float (&a)[8]) {
  lq_v4i r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, F16>::value) {
      typedef _Float16 v2h __attribute__((ext_vector_type(2)));
      typedef float v2f __attribute__((ext_vector_type(2)));
      const v2f f = {a[2 * i], a[2 * i + 1]};
      r[i] = __builtin_bit_cast(int, __builtin_convertvector(f, v2h));
    } else {
      r[i] = (int)pack_bf16(a[2 * i], a[2 * i + 1]);
    }
  }
  return r;
}
template <typename T>
LQ_DEV lq_v4i round8(const float (&a)[8], const float (&b)[8]) {
  if constexpr (std::is_same<T, F16>::value) {  // one mixed-precision instruction each
    lq_v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)__builtin_fmaf(a[i], b[i], 0.0f);
    return __builtin_bit_cast(lq_v4i, h);
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a[i] * b[i];
    return round8<T>(v);
  }
}
// two products as two pieces each: fp16, hi = RN(a b), lo = RN(a b - hi), one mixed-precision instruction a piece; bf16 likewise from the
// rounded product
template <typename T>
LQ_DEV void split2(float a0, float b0, float a1, float b1, int& hi, int& lo) {
  if constexpr (std::is_same<T, F16>::value) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h h = {(_Float16)__builtin_fmaf(a0, b0, 0.0f), (_Float16)__builtin_fmaf(a1, b1, 0.0f)};
    const v2h l = {(_Float16)__builtin_fmaf(a0, b0, -(float)h[0]), (_Float16)__builtin_fmaf(a1, b1, -(float)h[1])};
    hi = __builtin_bit_cast(int, h), lo = __builtin_bit_cast(int, l);
  } else {
    const float u = a0 * b0, v = a1 * b1;
    const uint32_t h = pack_bf16(u, v);
    hi = (int)h, lo = (int)pack_bf16(u - __uint_as_float(h << 16), v - __uint_as_float(h & 0xffff0000u));
  }
}
// The power of two that brings m below 2^(TOP + 1) (and not below 2^TOP), within 2^LO and 2^HI
template <int TOP, int LO, int HI>
LQ_DEV float scale_for(float m) {
  const int e = (int)((__float_as_uint(m) >> 23) & 255u) - 127;  // (0: -127)
  return __uint_as_float((uint32_t)(127 + min(max(TOP - e, LO), HI)) << 23);
}
// the largest of a wave's non-negative values, by lane permutations of the vector unit; the same for the whole wave
// (whole numbers order like them, and their maximum takes a permuted operand)
LQ_DEV float wave_top(float f) {
  uint32_t v = __float_as_uint(f);
#define LQ_TOP(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false))
  LQ_TOP(0xB1);   // lanes 1 0 3 2
  LQ_TOP(0x4E);   // lanes 2 3 0 1
  LQ_TOP(0x141);  // mirrored halves of a row of 16
  LQ_TOP(0x140);  // mirrored rows
  LQ_TOP(0x142);  // the last lane of a row to the next row
  LQ_TOP(0x143);  // the last lane of the first half of the wave to the second
#undef LQ_TOP
  return __int_as_float(__builtin_amdgcn_readlane((int)v, 63));
}
LQ_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
LQ_DEV float lane63(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
// the larger of a lane's and the lane's of the other half, which has the same channel (by their bits: non-negative numbers)
LQ_DEV uint32_t channel_top(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}
LQ_DEV float channel_top(float v) { return __uint_as_float(channel_top(__float_as_uint(v))); }
// a power of two's reciprocal
LQ_DEV float pow2_inverse(float v) { return __uint_as_float(0x7f000000u - __float_as_uint(v)); }
// Four rows of 16 entries of 16 bits, given by the 16 lanes of a quarter of the wave as four pieces a row, come back by columns: lane i has
// entry i of the rows
LQ_DEV lq_v2i read_columns(const void* at) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  return __builtin_bit_cast(lq_v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
}
// LDS reads stay where they are written (everything else may move): as the compiler orders them, most stand right in front of their use
LQ_DEV void reads_stay() { __builtin_amdgcn_sched_barrier(0xf); }
// |v|, or 0 for what is no number and must not set a scale
LQ_DEV float finite_size(float v) {
  const float a = __builtin_fabsf(v);
  return a < __builtin_inff() ? a : 0.0f;
}
LQ_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The order of a contraction of 64: step ks, half hh of the wave and slot i stand for entry 16 ks + 8 (i / 4) + 4 hh + i % 4, in which the
// accumulators of v_mfma_f32_32x32x16 hold their rows.  The state's and C B^T's accumulators then are operands as they are.
LQ_DEV int entry(int ks, int hh, int i) { return 16 * ks + 8 * (i >> 2) + 4 * hh + (i & 3); }

// sizes of a (chunk, group)'s operands.  NT: tiles of 32 state columns
template <int NT>
struct Table {
  static constexpr int kC = NT * 4 * 1024, kB = NT * 4 * 1024, kBytes = kCB + kC + kB;
};

// which unit (chunk) of which sequence
LQ_DEV Unit unit_of(const PromptParams& p, int u) {
  if (p.starts) return sv_locate<Q>(p.starts, p.nseq, p.tokens, u);
  const int per = (p.seqlen + Q - 1) / Q;
  Unit r;
  r.seq = u / per, r.index = u - r.seq * per, r.begin = 0, r.end = p.seqlen;
  return r;
}

// ---------------------------------------------------------------------------------------------------------------- operands
template <typename T, int NT>
LQ_DEV void operands(const PromptParams& p, const Unit& u, int unit, int g, uint16_t* smem, float* top) {
  constexpr int LD = 32 * NT + 8;  // halves of a row in LDS
  uint16_t *Bs = smem, *Cs = smem + Q * LD;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const int64_t seq = p.starts ? 0 : u.seq, t0 = u.begin + (int64_t)u.index * Q;
  const int rem = min(Q, u.end - u.begin - u.index * Q);
  const uint16_t* Bg = p.B + seq * p.sB_b + t0 * p.sB_l + g * p.sB_g;
  const uint16_t* Cg = p.C + seq * p.sC_b + t0 * p.sC_l + g * p.sC_g;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int pc = tid + 256 * i, t = pc / (4 * NT), n = (pc % (4 * NT)) * 8;
    const bool in = t < rem && n < p.N;
    const int tc = min(t, rem - 1), nc = min(n, p.N - 8);
    const lq_v4i zero = {0, 0, 0, 0};
    const lq_v4i b = *(const lq_v4i*)(Bg + tc * p.sB_l + nc), c = *(const lq_v4i*)(Cg + tc * p.sC_l + nc);
    *(lq_v4i*)(Bs + t * LD + n) = in ? b : zero;
    *(lq_v4i*)(Cs + t * LD + n) = in ? c : zero;
  }
  __syncthreads();
  char* out = p.tables + ((int64_t)unit * p.G + g) * Table<NT>::kBytes;
  if (wave < 3) {  // C B^T of rows t (columns of the product) and tokens s (its rows); fp32 sums of exact products
    const int tt = wave > 0, st = wave > 1;
    v16f acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2 * NT; ++k) {
      const lq_v4i b = *(const lq_v4i*)(Bs + (32 * st + (lane & 31)) * LD + 16 * k + 8 * hh);
      const lq_v4i c = *(const lq_v4i*)(Cs + (32 * tt + (lane & 31)) * LD + 16 * k + 8 * hh);
      acc = mfma<T>(b, c, acc);
    }
    float m = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {  // nothing above the diagonal
      if (tt == st && entry(r >> 3, hh, r & 7) > (lane & 31)) acc[r] = 0.0f;
      m = fmaxf(m, finite_size(acc[r]));
    }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (lane < 32) top[32 * wave + lane] = m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // operand 2 wave + r / 2, its slots 4 (r % 2) ..
      const lq_v4f v = {acc[4 * r], acc[4 * r + 1], acc[4 * r + 2], acc[4 * r + 3]};
      *(lq_v4f*)(out + ((2 * wave + (r >> 1)) * 2 + (r & 1)) * 1024 + lane * 16) = v;
    }
  }
  __syncthreads();
  if (tid < Q) p.rows[((int64_t)unit * p.G + g) * Q + tid] = tid < 32 ? top[tid] : fmaxf(top[tid], top[tid + 32]);
  auto put = [&](const uint16_t (&v)[8], char* at) {
    lq_v4i o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (int)(v[2 * i] | (uint32_t)v[2 * i + 1] << 16);
    *(lq_v4i*)(at + lane * 16) = o;
  };
#pragma unroll
  for (int i = 0; i < NT; ++i) {  // C: operand (tt, nt, q): rows t, state columns 32 nt + entry(q, ..)
    const int op = wave + 4 * i, tt = op / (2 * NT), k = op % (2 * NT);
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = Cs[(32 * tt + (lane & 31)) * LD + entry(k, hh, e)];
    put(v, out + kCB + op * 1024);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {  // B^T: operand (nt, ks): rows n, tokens entry(ks, ..)
    const int op = wave + 4 * i, nt = op >> 2, ks = op & 3;
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = Bs[entry(ks, hh, e) * LD + 32 * nt + (lane & 31)];
    put(v, out + kCB + Table<NT>::kC + op * 1024);
  }
}

constexpr int kHeads = 16;  // heads of a workgroup that forms step sizes

LQ_DEV void step_sizes(const PromptParams& p, const Unit& u, int unit, int h0, float* tile) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t seq = p.starts ? 0 : u.seq, t0 = u.begin + (int64_t)u.index * Q;
  const int rem = min(Q, u.end - u.begin - u.index * Q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = (tid + 256 * i) / kHeads, h = (tid + 256 * i) % kHeads;
    tile[t * (kHeads + 1) + h] = sv_load(p.dt, seq * p.sdt_b + (t0 + min(t, rem - 1)) * p.sdt_l + min(h0 + h, p.H - 1) * p.sdt_h, p.dt_dtype);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kHeads / 4; ++i) {
    const int h = h0 + wave * (kHeads / 4) + i;
    if (h >= p.H) break;
    float d = sv_step_size(tile[lane * (kHeads + 1) + h - h0], p.dt_bias ? p.dt_bias[h] : 0.0f, p.softplus, p.dt_min, p.dt_max);
    if (lane >= rem) d = 0.0f;  // a token behind the prompt changes nothing
    // one factor of 2^-160 is zero in 32 bits, and sums of larger ones would cost the tokens behind them their last bits
    const float e = d * (p.A[h] * kLog2e), a = e < -160.0f ? -160.0f : e;
    float c = a, r = __shfl_down(a, 1, 64);  // sums up to and with this token; behind it (summed from the end: near it they are small and exact)
    if (lane == 63) r = 0.0f;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float up = __shfl_up(c, off, 64), down = __shfl_down(r, off, 64);
      if (lane >= off) c += up;
      if (lane + off < 64) r += down;
    }
    // the largest weight exp(c_t - c_s) |d_s| of a row of C B^T: a running maximum of log2 |d_s| - c_s
    float most = __builtin_amdgcn_logf(finite_size(d)) - c;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float up = __shfl_up(most, off, 64);
      if (lane >= off) most = fmaxf(most, up);
    }
    float* o = p.steps + ((int64_t)unit * p.H + h) * (4 * Q) + lane;
    o[0] = d, o[Q] = c, o[2 * Q] = exp2_fast(r) * d, o[3 * Q] = exp2_fast(most + c);
  }
}

template <typename T, int NT>
__global__ __launch_bounds__(256) void ssm_operands_kernel(PromptParams p) {
  __shared__ __align__(16) uint16_t smem[2 * Q * (32 * NT + 8)];
  __shared__ float top[96];
  const int unit = blockIdx.x;
  const Unit u = unit_of(p, unit);
  if (u.seq < 0) return;
  if ((int)blockIdx.y < p.G) operands<T, NT>(p, u, unit, blockIdx.y, smem, top);
  else step_sizes(p, u, unit, ((int)blockIdx.y - p.G) * kHeads, (float*)smem);
}

// ---------------------------------------------------------------------------------------------------------------- segments
struct Segment {
  int seq, begin, len;      // tokens of the sequence
  int chunk0, chunks, unit0;  // its first chunk in the sequence, how many, and the unit of the first
  bool first, last;
};
LQ_DEV Segment segment_of(const PromptParams& p, int sg) {
  Segment r;
  r.seq = -1;
  if (!p.starts) {
    const int nc = (p.seqlen + Q - 1) / Q, per = (nc + p.seg_chunks - 1) / p.seg_chunks;
    r.seq = sg / per;
    r.begin = 0, r.len = p.seqlen, r.chunk0 = (sg - r.seq * per) * p.seg_chunks, r.unit0 = r.seq * nc + r.chunk0;
    r.chunks = min(p.seg_chunks, nc - r.chunk0);
    r.first = r.chunk0 == 0, r.last = r.chunk0 + r.chunks == nc;
    return r;
  }
  const int lane = threadIdx.x & 63;
  int before = 0, ubefore = 0;
  for (int s0 = 0; s0 < p.nseq; s0 += 64) {
    const int s = s0 + lane;
    int b = 0, e = 0;
    if (s < p.nseq) b = p.starts[s], e = p.starts[s + 1];
    if (b < 0 || e > p.tokens || e < b) b = e = 0;
    const int units = (int)(((uint32_t)(e - b) + (Q - 1)) / Q), n = (units + p.seg_chunks - 1) / p.seg_chunks;
    int sum = n, usum = units;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(sum, off, 64), v = __shfl_up(usum, off, 64);
      sum += lane >= off ? o : 0, usum += lane >= off ? v : 0;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (sg < before + total) {
      const int l = __builtin_ctzll(__ballot(sg < before + sum));
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int nc = of(units);
      r.seq = s0 + l, r.begin = of(b), r.len = of(e) - r.begin;  // (scalar already)
      r.chunk0 = (sg - before - of(sum - n)) * p.seg_chunks;
      r.unit0 = ubefore + of(usum - units) + r.chunk0;
      r.chunks = min(p.seg_chunks, nc - r.chunk0);
      r.first = r.chunk0 == 0, r.last = r.chunk0 + r.chunks == nc;
      return r;
    }
    before += total, ubefore += __builtin_amdgcn_readlane(usum, 63);
    if (ubefore > p.units) break;
  }
  return r;
}

// Which segment and which part of a group's heads a workgroup of the flat grid has.  Workgroups go round the 8 XCDs in launch order; the
// parts of one segment read the same operands, so each XCD gets adjacent ones.  (A whole number of segments to an XCD instead left four of
// the eight with twice the others' work.)
LQ_DEV void place(const PromptParams& p, int& sg, int& part) {
  const int parts = p.G * p.per_group, i = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  sg = i / parts, part = i - sg * parts;
}

constexpr int W = 4;  // waves of a workgroup

// A wave has 32 channels of one head: the state's N x 32 as accumulators (rows n, columns the channels).  STATES: only the segment's
// state and decay.  A workgroup's waves share the chunk's operands in LDS, fetched there as they lie in memory; each wave's x comes the same
// way, 64 tokens x 32 channels, a chunk ahead into one of two places, and its y leaves through the same place.  Two workgroups share a
// compute unit, so that one computes while the other's operands are on their way.
template <typename T, int NT, bool STATES>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(NT == 8 ? 1 : 2, NT == 8 ? 1 : 2))) void ssm_chunks_kernel(PromptParams p) {
  constexpr bool kHalf = std::is_same<T, F16>::value;
  using Tab = Table<NT>;
  constexpr int kSkip = STATES ? kCB + Tab::kC : 0, kLoad = Tab::kBytes - kSkip;  // bytes of a chunk's operands that are needed
  __shared__ __align__(16) char bufs[STATES ? 2 : 1][kLoad];
  __shared__ __align__(256) uint16_t xbuf[2][W][Q * 32];
  __shared__ __align__(16) float tok[W][3 * Q];  // each wave's q (or d), w, exp2(c) (fp16: scaled)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5, col = lane & 31;
  int sg, part;
  place(p, sg, part);
  // (what is the same for the whole wave goes to scalar registers: a division leaves it in vector ones, and every address made of it too)
  sg = uniform(sg), part = uniform(part);
  int at = 0;  // STATES: which piece of which segment
  if (STATES) {
    const int piece = sg % p.pieces;
    sg /= p.pieces;
    if (!p.starts) sg += sg / max(p.segs / p.nseq - 1, 1);  // (as many segments to each prompt, the last ones left out)
    sg = uniform(sg), at = uniform(sg * p.pieces + piece);
  }
  if (sg >= p.segs) return;
  Segment s = segment_of(p, sg);
  // (starts that do not ascend can name the same tokens twice: what is behind the tables' end is left out)
  if (s.seq < 0 || s.unit0 + s.chunks > p.units || (STATES && s.last)) return;
  if (STATES) {  // (a segment that is not a prompt's last one has all its chunks)
    s.chunks = p.seg_chunks / p.pieces;
    const int skip = (at - sg * p.pieces) * s.chunks;
    s.chunk0 += skip, s.unit0 += skip;
  }
  s.seq = uniform(s.seq), s.begin = uniform(s.begin), s.len = uniform(s.len), s.chunk0 = uniform(s.chunk0), s.chunks = uniform(s.chunks), s.unit0 = uniform(s.unit0);
  const int g = uniform(part / p.per_group), pblocks = (p.P + 31) >> 5, hpg = uniform(p.H / p.G);
  const int block = (part - g * p.per_group) * W + wave;
  const bool live = block < hpg * pblocks;  // a wave without channels only helps to fetch the operands
  const int h = uniform(g * hpg + (live ? block / pblocks : 0)), ch0 = uniform((live ? block % pblocks : 0) * 32), ch = ch0 + col;
  const int chc = min(ch, p.P - 1);
  const int slot = p.state || p.slots ? uniform(sv_slot(p.slots, s.seq, p.num_slots)) : kSlotPad;
  const bool keeps = p.state && slot >= 0;
  const int64_t row0 = (p.starts ? s.begin : (int64_t)s.seq * p.seqlen);  // of the dense output
  uint16_t* os = p.out + (row0 * p.H + h) * p.P + ch0;
  const int64_t ostride = (int64_t)p.H * p.P;

  v16f S[NT];
  const int64_t sbase = ((int64_t)h * p.P + chc) * p.N;
  {
    const float* src = STATES ? nullptr : (p.seg_state && !(s.first && s.last)) ? p.seg_state + (int64_t)sg * p.pieces * p.H * p.P * p.N + sbase : keeps ? p.state + slot * p.ss_s + sbase : nullptr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = 32 * nt + 8 * j + 4 * hh;
        lq_v4f v = {0.f, 0.f, 0.f, 0.f};
        if (src && n < p.N) v = *(const lq_v4f*)(src + n);
#pragma unroll
        for (int e = 0; e < 4; ++e) S[nt][4 * j + e] = v[e];
      }
  }
  float unit_S = 1.0f;  // fp16: S holds the channel's state times this power of two
  const float Dv = !STATES && p.D ? p.D[p.D_has_hdim ? h * p.P + chc : h] : 0.0f;
  const bool bad = slot == kSlotBad;

  // what a chunk needs, requested while the one in front of it is worked on.  x: four rows of 16 bytes a lane, 8 channels each; tokens
  // behind the prompt read its last one again (at weight zero), channels behind the head its last eight.
  const char* tab = p.tables + ((int64_t)s.unit0 * p.G + g) * Tab::kBytes + kSkip;
  const uint16_t* xs = p.x + (p.starts ? s.begin * p.sx_l : s.seq * p.sx_b) + h * p.sx_h + ch0 + (int64_t)s.chunk0 * Q * p.sx_l;
  const float* steps = p.steps + ((int64_t)s.unit0 * p.H + h) * (4 * Q);
  const float* rows = p.rows + ((int64_t)s.unit0 * p.G + g) * Q;
  int left = s.len - s.chunk0 * Q;  // tokens that are not requested yet
  const uint32_t xcol = (uint32_t)min(8 * (lane & 3), p.P - 8 - ch0);
  uint32_t xoff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) xoff[i] = ((uint32_t)(16 * i + (lane >> 2)) * (uint32_t)p.sx_l + xcol) * 2u;
  float dv = 0.f, cv = 0.f, wv = 0.f, mv = 0.f, rv = 0.f;
  auto fetch = [&](int c) {  // chunk c's operands, one chunk after the other
    char* buf = bufs[STATES ? c & 1 : 0];
#pragma unroll
    for (int k = 0; k < kLoad / (1024 * W); ++k) sv_fetch16(tab + (k * W + wave) * 1024, (uint32_t)lane * 16u, buf + (k * W + wave) * 1024);
    tab += (int64_t)p.G * Tab::kBytes;
  };
  static_assert(kLoad % (1024 * W) == 0);
  auto request = [&](int c) {  // the next chunk's x and step sizes
    uint16_t* to = xbuf[c & 1][wave];
    if (left >= Q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sv_fetch16(xs, xoff[i], to + 16 * 32 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) sv_fetch16(xs, ((uint32_t)min(16 * i + (lane >> 2), left - 1) * (uint32_t)p.sx_l + xcol) * 2u, to + 16 * 32 * i);
    }
    uint32_t l = (uint32_t)lane;
    asm volatile("" : "+v"(l));  // (a scalar base and this offset: sums of both kept over the loop are registers that it lacks)
    dv = steps[l], cv = steps[l + Q], wv = steps[l + 2 * Q];
    if (kHalf && !STATES) mv = steps[l + 3 * Q], rv = rows[l];
    xs += Q * p.sx_l, steps += (int64_t)p.H * (4 * Q), rows += (int64_t)p.G * Q, left -= Q;
  };
  // Everything is there; or all but the last four stores (memory operations end in order), which are not waited for.
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" : "+v"(dv), "+v"(cv), "+v"(wv), "+v"(mv), "+v"(rv)::"memory"); };
  auto all_but_stores = [&] { asm volatile("s_waitcnt vmcnt(4)" ::: "memory"); };
  // every wave has read all of a chunk's operands: the next chunk's take their place
  auto taken = [&](int c) {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (c + 1 < s.chunks) fetch(c + 1);
  };
  fetch(0);
  if (live) request(0);
  arrived();
  // What a chunk's products need of the wave's own: x in registers, step sizes in LDS, the state's unit.  Done at the end of the chunk in
  // front, whose operands' successors are then on their way.
  float decay = 0.0f;
  float* my = tok[wave];
  lq_v4i xp[4];  // this lane's channel, tokens in the order of an operand
  auto x = [&](int ks, int i) { return T::to((uint16_t)((uint32_t)xp[ks][i >> 1] >> (16 * (i & 1)))); };
  float sum64 = 0.0f, step = 0.0f, all = 0.0f, row = 1.0f, lrow = 0.0f;
  float rescale = 1.0f, read = 1.0f, unread = 1.0f;  // fp16: to the state's new unit; what C multiplies is S times `read`, 1 / unread of the state
  uint32_t units = 0;                                // fp16: the power of two of x that enters the state, twice
  bool apart = false;
  auto begin = [&](int c) {
    const uint16_t* xl = xbuf[c & 1][wave] + (4 * hh + ((lane & 15) >> 2)) * 32 + (lane & 16) + 4 * (lane & 3);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const lq_v2i lo = read_columns(xl + 16 * ks * 32), hi = read_columns(xl + (16 * ks + 8) * 32);
      xp[ks] = lq_v4i{lo[0], lo[1], hi[0], hi[1]};
    }
    sum64 = cv, step = dv;  // (the next chunk's are requested soon)
    const float last = lane63(cv);
    all = exp2_fast(last);
    decay += last;
    float uw = 1.0f;
    if constexpr (kHalf) {
      // Units of the channel, from its largest entry of the state and of x.  What C multiplies has one of its own: what the chunk adds can be
      // far above the state that its first tokens read.
      float m = 0.0f;  // (no number where the lane has one that is none: its scale does not matter then)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(S[nt][e]));
      uint32_t top = 0;  // both halves of a dword at once: magnitudes order like whole numbers
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          typedef uint16_t v2u __attribute__((ext_vector_type(2)));
          top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u, top), __builtin_bit_cast(v2u, (uint32_t)xp[ks][i] & 0x7fff7fffu)));
        }
      const float mx = channel_top(finite_size(T::to((uint16_t)max(top & 0xffffu, top >> 16)))), ms = channel_top(finite_size(m));
      const float mw = wave_top(finite_size(wv)), iu = pow2_inverse(unit_S);
      // The state's new unit is uw, which brings the weights below 1, times that of x: within fp16, and such that weighted x is below 2^14 and
      // the state too, unless it is 2^38 above x (it is kept in 32 bits: nothing overflows)
      uw = scale_for<-1, -60, 24>(mw);
      const float k = fminf(fmaxf(scale_for<13, -100, 24>(fmaxf(ms * iu, mx * mw)) * pow2_inverse(uw), 0x1p-24f), 0x1p15f);
      const uint32_t k16 = F16::from(k);
      units = k16 | k16 << 16;
      if (!STATES) read = scale_for<13, -100, 100>(ms), unread = pow2_inverse(read) * iu;
      unit_S = uw * k, rescale = unit_S * iu;
      if (!STATES) {
        row = scale_for<13, -100, 24>(rv * mv);  // brings the token's row of weighted C B^T below 2^14
        lrow = (float)((int)(__float_as_uint(row) >> 23) - 127);
      }
    }
    // The weight exp(c_t - c_s) d_s of an entry of C B^T.  Where no eight tokens decay by 2^60, it is r q: r = exp(c_t - c) for each row and
    // block of eight tokens, c that in front of the block, and q = exp(c - c_s) d_s, at most 2^60 d_s: twelve exponentials a lane instead of
    // 48, and what r rounds to zero is below 2^-66.  Nor may c rise (negative steps), for r is cut off at 2^30: half a unit of it to a block
    // is the rounding of its sums, and what eight blocks add up to then stays below 2^28 with the row's unit, 2^24 at most.
    const float before = __shfl(cv, (lane & 56) - 1, 64), ahead = (lane < 8 ? 0.0f : before) - cv;
    apart = !STATES && __ballot(!(__builtin_fabsf(ahead - 29.75f) < 30.25f)) == 0;
    my[lane] = apart ? exp2_fast(ahead) * dv : dv;
    my[Q + lane] = kHalf ? wv * uw : wv, my[2 * Q + lane] = kHalf ? exp2_fast(cv) * row : exp2_fast(cv);
  };
  if (live) begin(0);
  for (int c = 0; c < s.chunks; ++c) {
    const bool more = c + 1 < s.chunks;
    // every wave's share of this chunk's operands is there
    if (STATES) taken(c);  // (and the chunk's before the last are read: the next one's on their way into that place)
    else asm volatile("s_barrier" ::: "memory");
    const char* buf = bufs[STATES ? c & 1 : 0];
    if (live) {
      if (more) request(c + 1);
      const lq_v4i* op = (const lq_v4i*)buf + lane;
      const lq_v4i* opB = op + (STATES ? 0 : (kCB + Tab::kC) / 16);
      v16f Y[2];
      if constexpr (!STATES) {  // exp(c_t) S C_t
        const lq_v4i* opC = op + kCB / 16;
        lq_v4i cc[3][2];
        auto ask = [&](int k) {
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) cc[k % 3][tt] = opC[(tt * 2 * NT + k) * 64];
        };
        ask(0);
        ask(1);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int e = 0; e < 16; ++e) Y[tt][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * NT; ++k) {
          if (k + 2 < 2 * NT) ask(k + 2);
          __builtin_amdgcn_sched_barrier(0);  // (all of S converted ahead is registers that it lacks)
          float v[8], r[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = S[k >> 1][8 * (k & 1) + i], r[i] = read;
          const lq_v4i sh = kHalf ? round8<T>(v, r) : round8<T>(v);
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) Y[tt] = mfma<T>(cc[k % 3][tt], sh, Y[tt]);
        }
      }
      if constexpr (!STATES) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          lq_v4f e4[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e4[j] = *(const lq_v4f*)(my + 2 * Q + 32 * tt + 8 * j + 4 * hh);
#pragma unroll
          for (int e = 0; e < 16; ++e) Y[tt][e] *= kHalf ? e4[e >> 2][e & 3] * unread : e4[e >> 2][e & 3];
        }
      }
      // the state behind the chunk
      {
        // Ahead: what the next products need is formed between these (one issued behind another of the same tile waits for it, and the
        // vector unit is free): 384 tokens in fp16 36.4 -> 35.3 us (before each channel had a unit).  bf16 lacks the registers from 65
        // state columns on (ragged prompts 140 -> 191, ten spilled); so does fp16 from 129 on, where it spills ten (4 prompts of 8192 tokens at
        // 256 columns: 1021 us, bf16 797).
        constexpr bool kAhead = kHalf || NT < 4;
        lq_v4i bb[3], wh[2], wl[2];
        lq_v4f w4[2][2];
        auto ask = [&](int i) { bb[i % 3] = opB[(4 * (i % NT) + i / NT) * 64]; };  // operand i = NT ks + nt
        auto ask_w = [&](int ks) {
#pragma unroll
          for (int j = 0; j < 2; ++j) w4[ks & 1][j] = *(const lq_v4f*)(my + Q + 16 * ks + 8 * j + 4 * hh);
        };
        auto pair = [&](int ks, int q) {  // a quarter of step ks' weighted x
          const lq_v4f& w = w4[ks & 1][q >> 1];
          float x0 = x(ks, 2 * q), x1 = x(ks, 2 * q + 1);
          if constexpr (kHalf) {
            typedef _Float16 v2h __attribute__((ext_vector_type(2)));
            const int two = xp[ks][q];  // (an element's bits are not cast in place)
            const v2h x2 = __builtin_bit_cast(v2h, two) * __builtin_bit_cast(v2h, units);
            x0 = (float)x2[0], x1 = (float)x2[1];
          }
          int h, l;
          split2<T>(w[2 * (q & 1)], x0, w[2 * (q & 1) + 1], x1, h, l);
          wh[kAhead ? ks & 1 : 0][q] = h, wl[kAhead ? ks & 1 : 0][q] = l;
        };
        ask_w(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) ask(i);
        reads_stay();
        const float f = kHalf ? all * rescale : all;
        if (kAhead) {
#pragma unroll
          for (int q = 0; q < 4; ++q) pair(0, q);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 16; ++e) S[nt][e] *= f;
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int i = NT * ks + nt;
            if (i + 2 < 4 * NT) ask(i + 2);
            if (nt == (kAhead ? 0 : NT - 1) && ks < 3) ask_w(ks + 1);
            if (kAhead && ks == 0) {
#pragma unroll
              for (int e = 0; e < 16; ++e) S[nt][e] *= f;
            }
            if (!kAhead) {
              reads_stay();
              if (nt == 0) {
#pragma unroll
                for (int q = 0; q < 4; ++q) pair(ks, q);
              }
            }
            if (kAhead) __builtin_amdgcn_sched_barrier(0);
            S[nt] = mfma<T>(bb[i % 3], wh[kAhead ? ks & 1 : 0], S[nt]);
            if (kAhead) __builtin_amdgcn_sched_barrier(0);
            if (kAhead && ks < 3 && nt >= NT - 2) {
              const int q = NT == 1 ? 0 : 2 * (nt - (NT - 2));
              pair(ks + 1, q);
              if (NT == 1) pair(ks + 1, q + 1);
            }
            if (kAhead) __builtin_amdgcn_sched_barrier(0);
            S[nt] = mfma<T>(bb[i % 3], wl[kAhead ? ks & 1 : 0], S[nt]);
            if (kAhead) __builtin_amdgcn_sched_barrier(0);
            if (kAhead && ks < 3 && nt >= NT - 2) {
              const int q = NT == 1 ? 2 : 2 * (nt - (NT - 2)) + 1;
              pair(ks + 1, q);
              if (NT == 1) pair(ks + 1, q + 1);
            }
          }
        }
      }
      if constexpr (!STATES) {
        // An activation that is no number must not reach the tokens in front of it, which the product below multiplies by zero: the state,
        // which all of the chunk's tokens reach, tells.  Then such tokens are left out and every output from them on is NaN.
        const bool odd = bad || __ballot(S[0][0] != S[0][0]) != 0;
        int from = bad ? -4 : Q;  // counted from token 4 hh, as this lane's entries are
        if (odd) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!(__builtin_fabsf(x(ks, i)) < __builtin_inff())) {
                from = min(from, entry(ks, 0, i));
                xp[ks][i >> 1] &= i & 1 ? 0xffff : 0xffff0000;
              }
          from = min(from, __shfl_xor(from, 32, 64) + (hh ? -4 : 4));
        }
        const lq_v4f* cb = (const lq_v4f*)buf + lane;
        if (kHalf) my[Q + lane] = pow2_inverse(row);
        float ct[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) ct[tt] = __shfl(sum64 + lrow, 32 * tt + col, 64);
        // six steps: rows tt, tokens ks (above the diagonal C B^T is stored as zero)
        constexpr int kT[6] = {0, 1, 0, 1, 1, 1}, kS[6] = {0, 0, 1, 1, 2, 3};
        auto add = [&](int n, const float (&f)[8], const float (&a)[8]) {
          Y[kT[n]] = mfma<T>(round8<T>(f, a), xp[kS[n]], Y[kT[n]]);
        };
        if (apart && !odd) {
          lq_v4f f4[2][2], q4[2][2];  // (the q of a ks serve two steps)
          auto ask = [&](int n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              f4[n & 1][j] = cb[((kT[n] * 2 + kS[n]) * 2 + j) * 64];
              if (n == 0 || kS[n] != kS[n - 1]) q4[kS[n] & 1][j] = *(const lq_v4f*)(my + 16 * kS[n] + 8 * j + 4 * hh);
            }
          };
          ask(0);
#pragma unroll
          for (int n = 0; n < 6; ++n) {
            if (n < 5) ask(n + 1);
            reads_stay();
            float f[8], a[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int kb = 2 * kS[n] + j;
              // (rows in front of the block, whose entries are zero, must not overflow)
              const float r = exp2_fast(fminf(ct[kT[n]] - (kb ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum64), 8 * kb - 1)) : 0.0f), 30.0f));
#pragma unroll
              for (int i = 0; i < 4; ++i) f[4 * j + i] = f4[n & 1][j][i], a[4 * j + i] = r * q4[kS[n] & 1][j][i];
            }
            add(n, f, a);
          }
        } else {
          my[lane] = step, my[2 * Q + lane] = sum64;
#pragma unroll
          for (int n = 0; n < 6; ++n) {
            __builtin_amdgcn_sched_barrier(0);  // (a seldom way: nothing of it is worth a register elsewhere)
            int t = col;
            asm volatile("" : "+v"(t));
            float f[8], a[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const lq_v4f f4 = cb[((kT[n] * 2 + kS[n]) * 2 + j) * 64];
              const lq_v4f c4 = *(const lq_v4f*)(my + 2 * Q + 16 * kS[n] + 8 * j + 4 * hh), d4 = *(const lq_v4f*)(my + 16 * kS[n] + 8 * j + 4 * hh);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float m = exp2_fast(ct[kT[n]] - c4[i]) * d4[i];
                f[4 * j + i] = f4[i], a[4 * j + i] = kS[n] >= 2 * kT[n] && entry(kS[n] - 2 * kT[n], hh, 4 * j + i) > t ? 0.0f : m;
              }
            }
            add(n, f, a);
          }
        }
        arrived();  // (requested at the chunk's beginning)
        taken(c);
        if (odd) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (entry(ks, 0, i) >= from) Y[ks >> 1][8 * (ks & 1) + i] = __builtin_nanf("");
        }
        // Out through the place of x (the wave's own, and in registers since the chunk's beginning): [channel][block of four tokens], block b
        // at place b ^ channel % 16, and back by columns, 16 tokens of eight channels a lane.
        char* yw = (char*)xbuf[c & 1][wave];
        const uint32_t y0 = (uint32_t)(col * 128 + ((hh ^ (col & 15)) * 8));
        lq_v4f r4[4][2];
        if (kHalf) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) r4[ks][j] = *(const lq_v4f*)(my + Q + 16 * ks + 8 * j + 4 * hh);
        }
        reads_stay();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            sv_v4u y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = Y[ks >> 1][8 * (ks & 1) + 4 * j + i], xi = x(ks, 4 * j + i);
              y[i] = T::from(kHalf ? __builtin_fmaf(v, r4[ks][j][i], __builtin_fmaf(Dv, xi, 0.0f)) : __builtin_fmaf(Dv, xi, v));
            }
            *(sv_v4u*)(yw + (y0 ^ (32 * ks + 16 * j))) = y;
          }
        lq_v4i yo[4];
        {
          const int q8 = 8 * (lane >> 4) + ((lane & 15) >> 2);  // channels q8 and q8 + 4 of this lane's pieces
          const uint32_t a0 = (uint32_t)(q8 * 128 + (((lane & 3) ^ (q8 & 15)) * 8)), a1 = (uint32_t)((q8 + 4) * 128 + (((lane & 3) ^ ((q8 + 4) & 15)) * 8));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const lq_v2i lo = read_columns(yw + (a0 ^ (32 * i))), hi = read_columns(yw + (a1 ^ (32 * i)));
            yo[i] = lq_v4i{lo[0], lo[1], hi[0], hi[1]};
          }
        }
        const int rem = s.len - (s.chunk0 + c) * Q;
        uint16_t* oc = os + (int64_t)(s.chunk0 + c) * Q * ostride;
        const uint32_t o0 = (uint32_t)(lane & 15) * (uint32_t)ostride + 8 * (lane >> 4);
        if (rem >= Q && ch0 + 32 <= p.P) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *(lq_v4i*)(oc + 16 * i * ostride + o0) = yo[i];
          if (more) begin(c + 1);
          all_but_stores();
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * i + (lane & 15) < rem && ch0 + 8 * (lane >> 4) < p.P) *(lq_v4i*)(oc + 16 * i * ostride + o0) = yo[i];
          if (more) begin(c + 1);
          arrived();
        }
      } else {
        arrived();
        if (more) begin(c + 1);
      }
    } else {
      if (!STATES) taken(c);
      arrived();
    }
  }
  float* dst = STATES ? p.seg_state + (int64_t)at * p.H * p.P * p.N + sbase : s.last && keeps ? p.state + slot * p.ss_s + sbase : nullptr;
  if (dst && live && ch < p.P) {
    const float ui = kHalf ? 1.0f / unit_S : 1.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = 32 * nt + 8 * j + 4 * hh;
        lq_v4f v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = kHalf ? S[nt][4 * j + e] * ui : S[nt][4 * j + e];
        if (n < p.N) *(lq_v4f*)(dst + n) = v;
      }
  }
  if (STATES && live && lane == 0 && ch0 == 0) p.seg_decay[(int64_t)at * p.H + h] = exp2_fast(decay);
}

// The state in front of each segment, in the place of what its first piece adds to one (what the last segment adds is not there).  A
// workgroup has 1024 entries of one head's state.
__global__ __launch_bounds__(256) void ssm_join_kernel(PromptParams p) {
  const int64_t per = (int64_t)p.P * p.N;
  const int h = blockIdx.y, at = (blockIdx.z * 256 + threadIdx.x) * 4, seq = blockIdx.x;
  // the sequence's segments, and how many there are in front of them
  auto segments = [&](int i) {
    int b = 0, e = p.seqlen;
    if (p.starts) {
      b = p.starts[i], e = p.starts[i + 1];
      if (b < 0 || e > p.tokens || e < b) b = e = 0;
    }
    return ((int)(((uint32_t)(e - b) + (Q - 1)) / Q) + p.seg_chunks - 1) / p.seg_chunks;
  };
  const int n = segments(seq);
  if (n < 2) return;
  int first = 0;
  if (p.starts) {
    // (starts that do not ascend can name far more than there are, and their sum must not wrap: one too many is enough to know)
    for (int i = threadIdx.x & 63; i < seq; i += 64) first = min(first + segments(i), p.segs + 1);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) first += __shfl_xor(first, off, 64);
  } else {
    first = seq * n;
  }
  if (at >= per || first > p.segs - n) return;
  const int slot = p.state || p.slots ? sv_slot(p.slots, seq, p.num_slots) : kSlotPad;
  lq_v4f v = {0.f, 0.f, 0.f, 0.f};
  if (p.state && slot >= 0) v = *(const lq_v4f*)(p.state + slot * p.ss_s + h * per + at);
  // four pieces requested at a time: a chain of one load after the other was most of this kernel
  constexpr int U = 4;
  float* base = p.seg_state + ((int64_t)first * p.pieces * p.H + h) * per + at;
  const float* dec = p.seg_decay + (int64_t)first * p.pieces * p.H + h;
  const int64_t next = (int64_t)p.H * per;
  const int all = (n - 1) * p.pieces;
  for (int i = 0, piece = 0; i <= all; i += U) {
    lq_v4f add[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(i + u, all - 1);
      add[u] = *(const lq_v4f*)(base + k * next), d[u] = dec[(int64_t)k * p.H];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u > all) break;
      if (piece == 0) *(lq_v4f*)(base + (i + u) * next) = v;
      piece = piece + 1 == p.pieces ? 0 : piece + 1;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(d[u], v[e], add[u][e]);  // (behind the last one: not used)
    }
  }
}

int check_dims(const lq_ssm_prompt_args* a) {
  if (a->nseq <= 0 || a->nheads <= 0 || a->ngroups <= 0 || a->nheads % a->ngroups != 0) return LQ_ERR_SHAPE;
  if (a->headdim <= 0 || a->headdim % 8 != 0 || a->dstate <= 0 || a->dstate % 8 != 0 || a->dstate > 256) return LQ_ERR_SHAPE;
  if ((a->seq_starts ? a->tokens <= 0 : a->seqlen <= 0) || !sv_act(a->dtype)) return LQ_ERR_SHAPE;
  if ((int64_t)a->nheads * a->headdim > 1 << 23 || a->ngroups + a->nheads / kHeads > 65000) return LQ_ERR_SHAPE;
  return LQ_OK;
}

int table_bytes(const lq_ssm_prompt_args* a) {
  return kCB + (a->dstate <= 32 ? 1 : a->dstate <= 64 ? 2 : a->dstate <= 128 ? 4 : 8) * 8 * 1024;
}

// How a call is cut: the units, the chunks of a segment.
struct Plan {
  int64_t units, segs, tables, steps, rows, states, decays, bytes;
  int per_group, seg_chunks, pieces, cut;
};
bool plan(const lq_ssm_prompt_args* a, Plan& r) {
  const int64_t nseq = a->nseq, most = ((int64_t)(a->seq_starts ? a->tokens : a->seqlen) + Q - 1) / Q;  // chunks of the longest prompt there can be
  r.units = a->seq_starts ? (int64_t)a->tokens / Q + nseq : nseq * most;
  const int64_t blocks = (int64_t)(a->nheads / a->ngroups) * ((a->headdim + 31) / 32);
  r.per_group = (int)((blocks + W - 1) / W);
  const int64_t parts = (int64_t)a->ngroups * r.per_group;
  // Tenths of a microsecond.  A chunk's step takes 43 where a compute unit has one workgroup and 72 where it has two; one of the states'
  // takes 17 and 27 (the younger one's: the older goes first), or 22 where others follow, and a piece of them 40 more; the join moves every piece's state and each segment's twice at 3 TB/s, and it and two
  // more launches come to 250.  Prompts of one length end with the fullest compute unit; of packed ones only a few are long, and mostly
  // alone.  Their lengths are not known here: the longest is taken to be two and a half times the mean.  Measured, 80 heads of 64 by 128: 4
  // prompts of 8192 tokens in 3 segments of one piece 303 us and the states 120, of two pieces 99 (of four 93, but the join takes longer), in 2
  // segments 397; 10 packed prompts of 6949 tokens, the longest 2047, 64 heads in 8 groups, 140 us uncut, 155 in segments of 12 chunks.
  // All of it at 128 state columns; at others the steps are shorter or longer, and above 128 a compute unit has one workgroup.  Where one packed
  // prompt is most of the tokens the guess is far off: 8000 tokens and 63 single ones are not cut, 661 to 684 us for 125 to 128 of the long one alone.
  const double mean = (double)r.units / nseq, chain = a->seq_starts ? std::min<double>((double)most, 2.5 * mean) : (double)most;
  auto step = [&](double wgs, double one, double two) {
    if (wgs <= 256) return one;
    return a->seq_starts && wgs <= 512 ? one + (two - one) * (wgs / 256 - 1) : two * std::ceil(wgs / 512);
  };
  double best = chain * step((double)nseq * parts, 43, 72);
  r.seg_chunks = (int)most, r.pieces = 1, r.cut = 0;
  int64_t last[3] = {0, 0, 0};        // (many numbers of segments come to the same chunks in each: those cost what the first of them does)
  for (int64_t k = 2; k <= 256; ++k)  // segments of the longest
    for (int64_t pieces = 1; pieces <= 2; ++pieces) {
      const int64_t n = (std::max<int64_t>(1, (int64_t)std::ceil(chain / k)) + pieces - 1) / pieces * pieces;
      if (n == last[pieces]) continue;
      last[pieces] = n;
      const double segs = a->seq_starts ? (double)r.units / n + 0.5 * nseq : (double)(nseq * ((most + n - 1) / n)), ahead = std::max(0.0, segs - nseq) * pieces;
      const double cost = n * step(segs * parts, 43, 72) + n / pieces * step(ahead * parts, 17, ahead * parts <= 512 ? 27 : 22) + 40 * std::ceil(ahead * parts / 512) +
                          (ahead + 2 * segs) * a->nheads * a->headdim * a->dstate * 4 / 3e5 + 250;
      if (n < most && cost < best) best = cost, r.seg_chunks = (int)n, r.pieces = (int)pieces, r.cut = 1;
    }
  const int64_t per = (most + r.seg_chunks - 1) / r.seg_chunks;
  r.segs = a->seq_starts ? std::min<int64_t>(r.units / r.seg_chunks + nseq, r.units) : nseq * per;
  if (!r.cut) r.segs = nseq;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  r.tables = 0;
  r.steps = up(r.units * a->ngroups * table_bytes(a));
  r.rows = r.steps + up(r.units * a->nheads * (4 * Q * 4));
  r.states = r.rows + up(r.units * a->ngroups * (Q * 4));
  r.decays = r.states + (r.cut ? up(r.segs * r.pieces * a->nheads * a->headdim * a->dstate * 4) : 0);
  r.bytes = r.decays + (r.cut ? up(r.segs * r.pieces * a->nheads * 4) : 0);
  return sv_fits(r.units, 256) && sv_fits(nseq, 256) && sv_fits(r.segs * r.pieces * parts + 7, 64 * W);
}

}  // namespace

extern "C" int lq_ssm_prompt_workspace_bytes(const lq_ssm_prompt_args* a, int64_t* bytes) {
  if (!a || !bytes) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  Plan pl;
  if (rc != LQ_OK) return rc;
  if (!plan(a, pl)) return LQ_ERR_SHAPE;
  *bytes = pl.bytes;
  return LQ_OK;
}

extern "C" int lq_ssm_prompt_plan(const lq_ssm_prompt_args* a, int64_t* out) {
  if (!a || !out) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  Plan pl;
  if (rc != LQ_OK) return rc;
  if (!plan(a, pl)) return LQ_ERR_SHAPE;
  out[0] = pl.segs, out[1] = pl.seg_chunks, out[2] = pl.cut ? pl.pieces : 0;
  return LQ_OK;
}

extern "C" int lq_ssm_prompt(const lq_ssm_prompt_args* a, hipStream_t stream) {
  if (!a || !a->x || !a->dt || !a->A || !a->B || !a->C || !a->out || !a->workspace) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc != LQ_OK) return rc;
  if (!sv_float(a->dt_dtype) || (a->state && a->num_slots <= 0)) return LQ_ERR_SHAPE;
  for (const int64_t s : {a->B_stride_b, a->B_stride_l, a->B_stride_g, a->C_stride_b, a->C_stride_l, a->C_stride_g})
    if (s % 8 != 0) return LQ_ERR_SHAPE;
  if (a->x_stride_l < 0 || a->x_stride_l >= 1 << 24) return LQ_ERR_SHAPE;  // a chunk's rows are reached by 32-bit offsets
  if (a->x_stride_b % 8 != 0 || a->x_stride_l % 8 != 0 || a->x_stride_h % 8 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->x, 16) || !sv_al(a->B, 16) || !sv_al(a->C, 16) || !sv_al(a->out, 16) || !sv_al(a->state, 16) || a->state_stride_s % 4 != 0 ||
      !sv_al(a->dt, sv_size(a->dt_dtype)) || !sv_al(a->A, 4) || !sv_al(a->D, 4) || !sv_al(a->dt_bias, 4) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4))
    return LQ_ERR_SHAPE;
  Plan pl;
  if (!plan(a, pl) || a->workspace_bytes < pl.bytes || !sv_al(a->workspace, 256)) return LQ_ERR_SHAPE;
  char* ws = (char*)a->workspace;
  PromptParams p = {(const uint16_t*)a->x, a->x_stride_b, a->x_stride_l, a->x_stride_h, a->dt, a->dt_stride_b, a->dt_stride_l, a->dt_stride_h, a->dt_dtype, a->A,
                    (const uint16_t*)a->B, a->B_stride_b, a->B_stride_l, a->B_stride_g, (const uint16_t*)a->C, a->C_stride_b, a->C_stride_l, a->C_stride_g,
                    a->D, a->D_has_hdim, a->dt_bias, a->dt_softplus, a->dt_min, a->dt_max, (uint16_t*)a->out, a->state, a->state_stride_s, a->slots,
                    a->seq_starts, a->num_slots, a->nseq, a->seqlen, a->tokens, a->nheads, a->headdim, a->ngroups, a->dstate,
                    ws + pl.tables, (float*)(ws + pl.steps), (float*)(ws + pl.rows), pl.cut ? (float*)(ws + pl.states) : nullptr, pl.cut ? (float*)(ws + pl.decays) : nullptr,
                    (int)pl.units, (int)pl.segs, pl.seg_chunks, pl.pieces, pl.per_group};
  const dim3 pre((unsigned)pl.units, (unsigned)(a->ngroups + (a->nheads + kHeads - 1) / kHeads));
  auto grid_of = [&](int64_t segs) { return dim3((unsigned)((segs * a->ngroups * pl.per_group + 7) / 8 * 8)); };
  const dim3 grid = grid_of(pl.segs), pieces = grid_of((a->seq_starts ? pl.segs : pl.segs - a->nseq) * pl.pieces), threads(64 * W);
  const int64_t per = (int64_t)a->headdim * a->dstate;
  const dim3 join((unsigned)a->nseq, (unsigned)a->nheads, (unsigned)((per + 1023) / 1024));
  if (join.y > 65535 || join.z > 65535) return LQ_ERR_SHAPE;
  auto go = [&](auto t, auto k) {
    using T = decltype(t);
    constexpr int NT = decltype(k)::value;
    hipLaunchKernelGGL((ssm_operands_kernel<T, NT>), pre, dim3(256), 0, stream, p);
    if (pl.cut) {
      hipLaunchKernelGGL((ssm_chunks_kernel<T, NT, true>), pieces, threads, 0, stream, p);
      hipLaunchKernelGGL(ssm_join_kernel, join, dim3(256), 0, stream, p);
    }
    hipLaunchKernelGGL((ssm_chunks_kernel<T, NT, false>), grid, threads, 0, stream, p);
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
