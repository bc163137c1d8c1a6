// lq_linear_attention_prompt: linear attention over prompts of any lengths, from and into an fp32 state.
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t
// in chunks of 64 tokens.  With c_t = sum of g up to t inside a chunk and S the state in front of it,
//   o_t = scale (exp(c_t) S^T q_t + sum_{s <= t} exp(c_t - c_s) (q_t . k_s) v_s)
//   S'  = exp(c_63) S + sum_s exp(c_63 - c_s) k_s v_s^T
// which are products of matrices.  Three kernels:
//   states     per segment of a prompt: the state at its end if it starts from zero, and what it multiplies an earlier one by;
//   join       walks the segments: the state in front of each.  (states and join: only where prompts are cut into segments, because
//              prompts times heads are too few for 256 compute units)
//   chunks     walks a segment chunk by chunk, the state in registers
//
// Precision.  Activations enter the matrix products as they are, all sums are fp32, and so is the state.  What is formed in fp32 on the way
// and reaches only o, which is rounded to the activations' type itself (weighted q . k, the state that q multiplies), enters rounded to
// that type: half a step of each term.  What the state gathers over a prompt (weighted v) enters as two (fp16) or three (bf16) pieces of the
// type: off by 2^-22 of itself, or not at all (two of bf16: the state 2.4e-6 off, here and in fp16 below 1e-6).  bf16 has the range of fp32.  fp16: after a multiplication by a power of two that brings the largest of what
// is multiplied (a channel's state; its state and v; a row of 32 weighted q . k) below 2^14, so no size of activations overflows.
#include <algorithm>
#include <cmath>

#include "serve_common.h"

namespace {

constexpr int Q = 64;  // tokens of a chunk
constexpr float kLog2e = 1.44269504088896340736f;

struct PromptParams {
  const uint16_t* q;
  int64_t sq_b, sq_l, sq_h;
  const uint16_t* k;
  int64_t sk_b, sk_l, sk_h;
  const uint16_t* v;
  int64_t sv_b, sv_l, sv_h;
  const void* g;
  int64_t sg_b, sg_l, sg_h;
  int g_dtype, g_same;  // g_same: one decay for all tokens of a head
  float scale;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, H, K, V;
  float* seg_state;  // [segment][H][K][V], or NULL: prompts are not cut
  float* seg_decay;  // [segment][H]
  int segs, seg_chunks, parts;
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
// eight numbers, or products with one, rounded to T
template <typename T>
LQ_DEV lq_v4i round8(const float (&a)[8]) {
  lq_v4i r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, F16>::value) {
      typedef _Float16 v2h __attribute__((ext_vector_type(2)));
      const v2h h = {(_Float16)a[2 * i], (_Float16)a[2 * i + 1]};
      r[i] = __builtin_bit_cast(int, h);
    } else {
      r[i] = (int)pack_bf16(a[2 * i], a[2 * i + 1]);
    }
  }
  return r;
}
template <typename T>
LQ_DEV lq_v4i round8(const float (&a)[8], float b) {
  lq_v8h h;  // (fp16: one mixed-precision instruction each)
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (_Float16)__builtin_fmaf(a[i], b, 0.0f);
  return __builtin_bit_cast(lq_v4i, h);
}
// two products as pieces of T, each what the ones before leave of it, rounded: fp16 two (the product's own, and one mixed-precision instruction
// a piece), bf16 three, which hold all 24 bits of the rounded product
template <typename T>
LQ_DEV void split2(float a0, float b0, float a1, float b1, int (&o)[3]) {
  if constexpr (std::is_same<T, F16>::value) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h h = {(_Float16)__builtin_fmaf(a0, b0, 0.0f), (_Float16)__builtin_fmaf(a1, b1, 0.0f)};
    const v2h l = {(_Float16)__builtin_fmaf(a0, b0, -(float)h[0]), (_Float16)__builtin_fmaf(a1, b1, -(float)h[1])};
    o[0] = __builtin_bit_cast(int, h), o[1] = __builtin_bit_cast(int, l);
  } else {
    float u = a0 * b0, v = a1 * b1;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t h = pack_bf16(u, v);
      o[i] = (int)h, u -= __uint_as_float(h << 16), v -= __uint_as_float(h & 0xffff0000u);
    }
  }
}
// The power of two that brings m below 2^(TOP + 1) (and not below 2^TOP), within 2^LO and 2^HI
template <int TOP, int LO, int HI>
LQ_DEV float scale_for(float m) {
  const int e = (int)((__float_as_uint(m) >> 23) & 255u) - 127;  // (0: -127)
  return __uint_as_float((uint32_t)(127 + min(max(TOP - e, LO), HI)) << 23);
}
LQ_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
LQ_DEV float lane_of(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
// the larger of a lane's and the lane's of the other half, which has the same channel (by their bits: non-negative numbers)
LQ_DEV float channel_top(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(max((uint32_t)r[0], (uint32_t)r[1]));
}
// a power of two's reciprocal
LQ_DEV float pow2_inverse(float v) { return __uint_as_float(0x7f000000u - __float_as_uint(v)); }
// Four rows of 16 entries of 16 bits, given by the 16 lanes of a quarter of the wave as four pieces a row, come back by columns: lane i has
// entry i of the rows
LQ_DEV lq_v2i read_columns(const void* at) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  return __builtin_bit_cast(lq_v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
}
// |v|, or 0 for what is no number and must not set a scale
LQ_DEV float finite_size(float v) {
  const float a = __builtin_fabsf(v);
  return a < __builtin_inff() ? a : 0.0f;
}
// LDS reads stay where they are written (everything else may move): as the compiler orders them, most stand right in front of their use
LQ_DEV void reads_stay() { __builtin_amdgcn_sched_barrier(0xf); }
LQ_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
template <int CTRL, int ROWS>
LQ_DEV float shifted(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true)); }
// sums over the wave: up to and with each lane; behind each lane (summed from the end: near it they are small and exact)
LQ_DEV float sums_upto(float v) {
  v += shifted<0x111, 0xf>(v), v += shifted<0x112, 0xf>(v), v += shifted<0x114, 0xf>(v), v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v), v += shifted<0x143, 0xc>(v);
  return v;
}
LQ_DEV float sums_behind(float v, int lane) {
  float r = shifted<0x101, 0xf>(v);  // the next lane's of the row of 16
  r += shifted<0x101, 0xf>(r), r += shifted<0x102, 0xf>(r), r += shifted<0x104, 0xf>(r), r += shifted<0x108, 0xf>(r);
  const float all = r + v;  // (a row's first lane: the whole row)
  const float r3 = lane_of(all, 48), r2 = r3 + lane_of(all, 32), r1 = r2 + lane_of(all, 16);
  return r + (lane < 16 ? r1 : lane < 32 ? r2 : lane < 48 ? r3 : 0.0f);
}

// The order of a contraction over tokens: step ks, half hh of the wave and slot i stand for token 16 ks + 8 (i / 4) + 4 hh + i % 4, in which the
// accumulators of v_mfma_f32_32x32x16 hold their rows: those of k q^T then are operands as they are.  The state's accumulators are too, over
// channels of k: the row that is token x above is channel x with bits 2 and 3 exchanged, so that eight slots are eight adjacent channels.
LQ_DEV int entry(int ks, int hh, int i) { return 16 * ks + 8 * (i >> 2) + 4 * hh + (i & 3); }
LQ_DEV int channel(int nt, int hh, int r) { return 32 * nt + 16 * (r >> 3) + 8 * hh + (r & 7); }

// Rows of q and k in LDS: 16-byte piece c of a row lies at place c ^ order(row).  The 16 rows at one piece that a read of 16 bytes serves at
// once, and the four rows at four pieces that a read by columns does, then touch each bank once.
template <int NT>
LQ_DEV int order(int row) {
  if constexpr (NT == 1) return (row >> 2) & 3;
  else if constexpr (NT == 2) return (row << 1 & 4) | (row >> 2 & 3);
  else return (row << 2 & 12) | (row >> 2 & 3);
}

struct Segment {
  int seq, begin, len;  // tokens of the sequence
  int chunk0, chunks;   // its first chunk in the sequence, how many
  bool first, last;
};
LQ_DEV Segment segment_of(const PromptParams& p, int sg) {
  Segment r;
  if (p.starts) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    r.seq = -1;
    for (int s0 = 0; s0 < p.nseq; s0 += 64) {
      const int s = s0 + lane;
      int b = 0, e = 0;
      if (s < p.nseq) b = p.starts[s], e = p.starts[s + 1];
      if (b < 0 || e > p.tokens || e < b) b = e = 0;
      const int chunks = (int)(((uint32_t)(e - b) + (Q - 1)) / Q), n = (chunks + p.seg_chunks - 1) / p.seg_chunks;
      int sum = n;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(sum, off, 64);
        sum += lane >= off ? o : 0;
      }
      const int total = __builtin_amdgcn_readlane(sum, 63);
      if (sg < before + total) {
        const int l = __builtin_ctzll(__ballot(sg < before + sum));
        r.seq = s0 + l, r.begin = __builtin_amdgcn_readlane(b, l), r.len = __builtin_amdgcn_readlane(e, l) - r.begin;
        r.chunk0 = (sg - before - __builtin_amdgcn_readlane(sum - n, l)) * p.seg_chunks;
        break;
      }
      before += total;
      if (before >= p.segs) break;  // (starts that do not ascend can name far more than there are, and their sum must not wrap)
    }
  } else {
    const int per = ((p.seqlen + Q - 1) / Q + p.seg_chunks - 1) / p.seg_chunks;
    r.seq = sg / per, r.begin = 0, r.len = p.seqlen, r.chunk0 = (sg - r.seq * per) * p.seg_chunks;
  }
  if (r.seq >= 0) {
    const int nc = (r.len + Q - 1) / Q;
    r.chunks = min(p.seg_chunks, nc - r.chunk0), r.first = r.chunk0 == 0, r.last = r.chunk0 + r.chunks == nc;
  }
  return r;
}

// A wave has 32 channels of v of a head: the state's K x 32 as accumulators (rows channels of k, columns those of v).  STATES: only the
// segment's state and decay.  A workgroup's waves, up to W, share the chunk's q and k in LDS and the 32 x 32 tiles of weighted q . k that each
// of them forms one or two of; each wave's v comes the same way, a chunk ahead into one of two places, and its o leaves through the other.
template <typename T, int NT, int W, bool STATES>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(NT == 8 ? 1 : 2, NT == 8 ? 1 : 2))) void linear_attention_chunks_kernel(PromptParams p) {
  constexpr bool kHalf = std::is_same<T, F16>::value;
  constexpr int RB = 64 * NT, PR = 4 * NT, kTile = Q * RB;  // bytes and pieces of a row of q or k, bytes of a chunk's
  constexpr int kFetch = kTile / (1024 * W), kRows = 1024 / RB;  // fetches of a wave, rows of each
  constexpr int PT = W == 2 ? 2 : 1;                           // tiles of q . k of a wave
  __shared__ __align__(1024) char kbuf[STATES ? 2 : 1][kTile];
  __shared__ __align__(1024) char qbuf[STATES ? 16 : kTile];
  __shared__ __align__(256) uint16_t vbuf[2][W][Q * 32];
  __shared__ __align__(16) char pbuf[STATES ? 16 : 8 * 1024];  // weighted q . k, operands 4 tt + ks; (0, 2) and (0, 3) are zero
  __shared__ __align__(16) float punit[kHalf && !STATES ? 4 * 32 : 4];  // fp16: 1 / unit of each tile's rows t, tiles 2 tt + st
  __shared__ int podd[4];                                       // fp16: whether a tile has a unit that is not 1
  __shared__ __align__(16) float tok[W][3 * Q];                 // each wave's c, exp2(c_63 - c), exp2(c) scale
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), hh = lane >> 5, col = lane & 31;
  // Workgroups go round the 8 XCDs in launch order; the parts of one head, which read the same q and k, and the heads of one segment, whose
  // rows lie side by side, go to one.
  const int at = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3), per = p.H * p.parts;
  int sg = uniform(at / per);
  const int h = uniform((at - sg * per) / p.parts), part = uniform(at - sg * per - h * p.parts);
  if (STATES && !p.starts) sg = uniform(sg + sg / max(p.segs / p.nseq - 1, 1));  // (as many segments to each prompt, the last ones left out)
  if (sg >= p.segs) return;
  Segment s = segment_of(p, sg);
  if (s.seq < 0 || (STATES && s.last)) return;
  s.seq = uniform(s.seq), s.begin = uniform(s.begin), s.len = uniform(s.len), s.chunk0 = uniform(s.chunk0), s.chunks = uniform(s.chunks);
  const int ch0 = (part * W + wave) * 32, ch = ch0 + col, chc = min(ch, p.V - 1);
  const bool live = ch0 < p.V;  // a wave without channels only helps
  const int slot = p.state || p.slots ? uniform(sv_slot(p.slots, s.seq, p.num_slots)) : kSlotPad;
  const bool keeps = p.state && slot >= 0, bad = slot == kSlotBad;
  const int64_t row0 = p.starts ? s.begin : (int64_t)s.seq * p.seqlen;  // of the dense output
  const int64_t ostride = (int64_t)p.H * p.V, first = (int64_t)s.chunk0 * Q;
  uint16_t* os = p.out + (row0 * p.H + h) * p.V + ch0;
  const int64_t b = p.starts ? 0 : s.seq, l0 = (p.starts ? s.begin : 0) + first;
  const uint16_t* qs = p.q + b * p.sq_b + l0 * p.sq_l + h * p.sq_h;
  const uint16_t* ks_ = p.k + b * p.sk_b + l0 * p.sk_l + h * p.sk_h;
  const uint16_t* vs = p.v + b * p.sv_b + l0 * p.sv_l + h * p.sv_h + (live ? ch0 : 0);
  const int64_t g0 = b * p.sg_b + l0 * p.sg_l + h * p.sg_h;

  v16f S[NT];
  const int64_t sbase = (int64_t)h * p.K * p.V + chc;
  {
    const float* src = STATES ? nullptr : (p.seg_state && !(s.first && s.last)) ? p.seg_state + (int64_t)sg * p.H * p.K * p.V + sbase : keeps ? p.state + slot * p.ss_s + sbase : nullptr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = channel(nt, hh, r);
        S[nt][r] = src && n < p.K ? src[(int64_t)n * p.V] : 0.0f;
      }
  }
  float unit_S = 1.0f;  // fp16: S holds the channel's state times this power of two

  if (!STATES) {
    const lq_v4i zero = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < 128; i += 64 * W) *(lq_v4i*)(pbuf + (2 * 64 + i) * 16) = zero;  // (read behind two barriers)
  }
  // channels behind K: zeros, left there for good (nothing is fetched over them)
  const bool whole = p.K == 32 * NT;
  if (!whole) {
    const lq_v4i zero = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < kTile / 16; i += 64 * W) {
      *(lq_v4i*)(kbuf[0] + i * 16) = zero;
      if (STATES) *(lq_v4i*)(kbuf[STATES ? 1 : 0] + i * 16) = zero;
      else *(lq_v4i*)(qbuf + i * 16) = zero;
    }
    __syncthreads();
  }
  // chunk by chunk: rows behind the prompt are its last one again (at weight zero)
  // (addresses are made of a lane number that the compiler does not know to be the same: kept over the loop they are registers that it lacks)
  auto fresh = [&] {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };
  auto rows_of = [&](const uint16_t* base, int64_t stride, char* to, int left) {
    const int lane = fresh();
#pragma unroll
    for (int i = 0; i < kFetch; ++i) {
      const int f = wave * kFetch + i, row = f * kRows + lane / PR, c = (lane % PR) ^ order<NT>(row);
      const uint32_t off = (uint32_t)min(row, left - 1) * (uint32_t)stride * 2u + (uint32_t)c * 16u;
      if (whole || c * 8 < p.K) sv_fetch16(base, off, to + f * 1024);
    }
  };
  int kleft = s.len - (int)first, vleft = kleft;
  auto fetch = [&](int c) {  // a chunk's k and q
    rows_of(ks_, p.sk_l, kbuf[STATES ? c & 1 : 0], kleft);
    if (!STATES) rows_of(qs, p.sq_l, qbuf, kleft);
    ks_ += Q * p.sk_l, qs += Q * p.sq_l, kleft -= Q;
  };
  float gv = 0.0f;
  int64_t gat = g0;
  auto request = [&](int c) {  // a chunk's v and decays
    uint16_t* to = vbuf[c & 1][wave];
    const int lane = fresh();
    if (live) {
      const uint32_t vcol = (uint32_t)min(8 * (lane & 3), p.V - 8 - ch0);
#pragma unroll
      for (int i = 0; i < 4; ++i) sv_fetch16(vs, ((uint32_t)min(16 * i + (lane >> 2), vleft - 1) * (uint32_t)p.sv_l + vcol) * 2u, to + 16 * 32 * i);
    }
    if (p.g && !p.g_same) gv = sv_load(p.g, gat + min(lane, vleft - 1) * p.sg_l, p.g_dtype);
    vs += Q * p.sv_l, gat += Q * p.sg_l, vleft -= Q;
  };
  if (p.g && p.g_same) gv = sv_load(p.g, g0, p.g_dtype);
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" : "+v"(gv)::"memory"); };
  auto all_but_stores = [&] { asm volatile("s_waitcnt vmcnt(4)" ::: "memory"); };
  auto meet = [&] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  fetch(0);
  request(0);
  arrived();

  // What a chunk's products need of the wave's own: v in registers, decays in LDS, the state's unit.
  float* my = tok[wave];
  lq_v4i xp[4] = {};  // this lane's channel, tokens in the order of an operand
  auto x = [&](int ks, int i) { return T::to((uint16_t)((uint32_t)xp[ks][i >> 1] >> (16 * (i & 1)))); };
  float total = 0.0f, all = 1.0f;                   // the segment's decay so far; the chunk's
  float rescale = 1.0f, read = 1.0f, unread = 1.0f;  // fp16: to the state's new unit; what q multiplies is S times `read`, 1 / unread of the state
  uint32_t units = 0;                                // fp16: the power of two of v that enters the state, twice
  auto begin = [&](int c) {
    const int lane = fresh(), hh = lane >> 5;
    const int rem = s.len - (s.chunk0 + c) * Q;
    {
      // one factor of 2^-160 is zero in 32 bits, and sums of larger ones would cost the tokens behind them their last bits
      const float e = sv_decay(gv) * kLog2e, one = e < -160.0f ? -160.0f : e;
      float cs, behind;
      if (p.g_same) {
        cs = one * (float)min(lane + 1, rem), behind = one * (float)max(min(rem, Q) - 1 - lane, 0);
      } else {
        const float a = lane < rem ? one : 0.0f;
        cs = sums_upto(a), behind = sums_behind(a, lane);
      }
      const float last = lane_of(cs, 63);
      all = exp2_fast(last);
      total += last;
      my[lane] = cs, my[Q + lane] = lane < rem ? exp2_fast(behind) : 0.0f;
      if (!STATES) my[2 * Q + lane] = exp2_fast(cs) * p.scale;
    }
    if (!live) return;
    const uint16_t* xl = vbuf[c & 1][wave] + (4 * hh + ((lane & 15) >> 2)) * 32 + (lane & 16) + 4 * (lane & 3);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const lq_v2i lo = read_columns(xl + 16 * ks * 32), hi = read_columns(xl + (16 * ks + 8) * 32);
      xp[ks] = lq_v4i{lo[0], lo[1], hi[0], hi[1]};
    }
    if constexpr (kHalf) {
      // Units of the channel, from its largest entry of the state and of v.  What q multiplies has one of its own: what the chunk adds can be
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
      const float mx = channel_top(finite_size(T::to((uint16_t)max(top & 0xffffu, top >> 16)))), ms = channel_top(finite_size(m)), iu = pow2_inverse(unit_S);
      // Weights are at most 1.  Weighted v is below 2^14 and the state too, unless it is 2^38 above v (it is kept in 32 bits: nothing overflows)
      const float k = fminf(fmaxf(scale_for<13, -100, 15>(fmaxf(ms * iu, mx)), 0x1p-24f), 0x1p15f);
      const uint32_t k16 = F16::from(k);
      units = k16 | k16 << 16;
      if (!STATES) read = scale_for<13, -100, 100>(ms), unread = pow2_inverse(read) * iu;
      unit_S = k, rescale = k * iu;
    }
  };
  begin(0);
  // this lane's place in the rows of q and k as operands: row lane & 31, pieces 2 ks + hh; and in k by columns (see `channel`)
  auto k_columns = [&](const char* buf, int lane, int nt, int ks) {
    const int hh = lane >> 5, r4 = (lane & 15) >> 2, nb = (lane >> 4) & 1, p4 = lane & 3;
    lq_v2i o[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = 8 * half + 4 * hh + r4;  // (order: the same 16 rows on)
      o[half] = read_columns(buf + (16 * ks + row) * RB + (((4 * nt + 2 * nb + (p4 & 1)) ^ order<NT>(row)) << 4) + 8 * (p4 >> 1));
    }
    return lq_v4i{o[0][0], o[0][1], o[1][0], o[1][1]};
  };
  // tiles of q . k: columns t of tile tt, rows s of tile st.  Y[0] has the rows of tile ta, Y[1] of the other
  const int ta = wave == 0 && W == 4 ? 0 : 1;
  for (int c = 0; c < s.chunks; ++c) {
    const int lane = fresh(), hh = lane >> 5, col = lane & 31;
    const bool more = c + 1 < s.chunks;
    meet();  // every wave's share of this chunk's q and k is there (STATES: and the chunk's in front is read)
    const char* kb = kbuf[STATES ? c & 1 : 0];
    if (STATES && more) fetch(c + 1);
    if (more) request(c + 1);
    v16f Y[2];
    if constexpr (!STATES) {
      v16f P[PT];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        Y[0][e] = Y[1][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < PT; ++i) P[i][e] = 0.0f;
      }
      // W = 4: waves 0, 1, 2 have (st, tt) = (0, 0), (0, 1), (1, 1), the last one has none.  W = 2: wave 0 (0, 1) and (0, 0), wave 1 (1, 1)
      const int st = W == 4 ? wave == 2 : wave;
      const char *qa = qbuf + ta * 32 * RB, *qz = qbuf + (1 - ta) * 32 * RB, *kx = kb + st * 32 * RB;
      const int a0 = col * RB + ((hh ^ order<NT>(col)) << 4);
      lq_v4i q0[3], q1[3], k0[3];
      auto ask = [&](int ks) {
        const int o = a0 ^ (ks << 5);
        q0[ks % 3] = *(const lq_v4i*)(qa + o), q1[ks % 3] = *(const lq_v4i*)(qz + o), k0[ks % 3] = *(const lq_v4i*)(kx + o);
      };
      ask(0);
      ask(1);
#pragma unroll
      for (int ks = 0; ks < 2 * NT; ++ks) {
        if (ks + 2 < 2 * NT) ask(ks + 2);
        __builtin_amdgcn_sched_barrier(0);  // (operands of all steps read ahead are registers that it lacks)
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = S[ks >> 1][8 * (ks & 1) + i];
        lq_v4i sh;
        if constexpr (kHalf) sh = round8<T>(v, read);
        else sh = round8<T>(v);
        P[0] = mfma<T>(k0[ks % 3], q0[ks % 3], P[0]);
        if constexpr (PT == 2) P[1] = mfma<T>(k0[ks % 3], q1[ks % 3], P[1]);
        Y[0] = mfma<T>(q0[ks % 3], sh, Y[0]);
        Y[1] = mfma<T>(q1[ks % 3], sh, Y[1]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int tt = y == 0 ? ta : 1 - ta;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const lq_v4f e4 = *(const lq_v4f*)(my + 2 * Q + 32 * tt + 8 * j + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) Y[y][4 * j + e] *= kHalf ? e4[e] * unread : e4[e];
        }
      }
      // weighted q . k, rounded, for all of the workgroup's waves
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        const int tt = i == 0 ? ta : 1 - ta;
        if ((W == 4 && wave == 3) || (W == 2 && i == 1 && wave == 1)) continue;
        const float ct = my[32 * tt + col];
        float w[16], m = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const lq_v4f c4 = *(const lq_v4f*)(my + 32 * st + 8 * j + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = P[i][4 * j + e] * (exp2_fast(ct - c4[e]) * p.scale);
            w[4 * j + e] = st == tt && 8 * j + 4 * hh + e > col ? 0.0f : f;
            if (kHalf) m = fmaxf(m, finite_size(w[4 * j + e]));
          }
        }
        if constexpr (kHalf) {
          m = channel_top(m);
          const bool plain = m == 0.0f || (m >= 0x1p-5f && m < 0x1p15f);
          const float u = plain ? 1.0f : scale_for<13, -100, 100>(m);
          const bool odd = __ballot(!plain) != 0;
          if (lane == 0) podd[2 * tt + st] = odd;
          if (odd) {
            if (lane < 32) punit[(2 * tt + st) * 32 + lane] = pow2_inverse(u);
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] *= u;
          }
        }
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = w[8 * k2 + e];
          *(lq_v4i*)(pbuf + (4 * tt + 2 * st + k2) * 1024 + lane * 16) = round8<T>(v);
        }
      }
    }
    // the state behind the chunk
    const int kl = fresh();
    const float f = kHalf ? all * rescale : all;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 16; ++e) S[nt][e] *= f;
    __builtin_amdgcn_sched_barrier(0);
    {
      constexpr int N = kHalf ? 2 : 3;
      lq_v4i kt[3], w[N];
      lq_v4f w4[2][2];
      auto ask = [&](int i) { kt[i % 3] = k_columns(kb, kl, i % NT, i / NT); };  // operand i = NT ks + nt
      auto ask_w = [&](int ks) {
#pragma unroll
        for (int j = 0; j < 2; ++j) w4[ks & 1][j] = *(const lq_v4f*)(my + Q + 16 * ks + 8 * j + 4 * hh);
      };
      ask_w(0);
      ask(0);
      ask(1);
      reads_stay();
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int i = NT * ks + nt;
          if (i + 2 < 4 * NT) ask(i + 2);
          if (nt == NT - 1 && ks < 3) ask_w(ks + 1);
          reads_stay();
          if (nt == 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const lq_v4f& f = w4[ks & 1][q >> 1];
              float x0 = x(ks, 2 * q), x1 = x(ks, 2 * q + 1);
              if constexpr (kHalf) {
                typedef _Float16 v2h __attribute__((ext_vector_type(2)));
                const int two = xp[ks][q];  // (an element's bits are not cast in place)
                const v2h x2 = __builtin_bit_cast(v2h, two) * __builtin_bit_cast(v2h, units);
                x0 = (float)x2[0], x1 = (float)x2[1];
              }
              int o[3];
              split2<T>(f[2 * (q & 1)], x0, f[2 * (q & 1) + 1], x1, o);
#pragma unroll
              for (int n = 0; n < N; ++n) w[n][q] = o[n];
            }
          }
#pragma unroll
          for (int n = 0; n < N; ++n) S[nt] = mfma<T>(kt[i % 3], w[n], S[nt]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!STATES) {
      arrived();  // (requested at the chunk's beginning)
      meet();     // every wave has read the chunk's q and k, and the weighted q . k is there
      if (more) fetch(c + 1);
      bool four = false;  // whether this wave has stored four times
      if (live) {
        const int lane = fresh(), hh = lane >> 5, col = lane & 31;
        // A v that is no number must not reach the tokens in front of it, which the product below multiplies by zero: the state, which all of
        // the chunk's tokens reach, tells.  Then such tokens are left out and every output from them on is NaN.
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
        bool apart = false;
        if constexpr (kHalf) apart = uniform(podd[0] | podd[2] | podd[3]) != 0;
        auto weighted = [&](int tt, int ks) { return *(const lq_v4i*)(pbuf + (4 * tt + ks) * 1024 + lane * 16); };
        if (!apart) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int y = 0; y < 2; ++y) Y[y] = mfma<T>(weighted(y == 0 ? ta : 1 - ta, ks), xp[ks], Y[y]);
        } else if constexpr (kHalf) {  // units of their own for the rows of a tile
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tt = y == 0 ? ta : 1 - ta;
            for (int st = 0; st <= tt; ++st) {
              v16f d = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              d = mfma<T>(weighted(tt, 2 * st), st ? xp[2] : xp[0], d);
              d = mfma<T>(weighted(tt, 2 * st + 1), st ? xp[3] : xp[1], d);
              sv_settle(d);
              const bool own = podd[2 * tt + st] != 0;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const lq_v4f u4 = *(const lq_v4f*)(punit + (2 * tt + st) * 32 + 8 * j + 4 * hh);
#pragma unroll
                for (int e = 0; e < 4; ++e) Y[y][4 * j + e] = __builtin_fmaf(d[4 * j + e], own ? u4[e] : 1.0f, Y[y][4 * j + e]);
              }
            }
          }
        }
        if (odd) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (32 * (y == 0 ? ta : 1 - ta) + entry(e >> 3, 0, e & 7) >= from) Y[y][e] = __builtin_nanf("");
        }
        // Out through the place of v (the wave's own, and in registers since the chunk's beginning): [channel][block of four tokens], block b
        // at place b ^ channel % 16, and back by columns, 16 tokens of eight channels a lane.
        char* yw = (char*)vbuf[c & 1][wave];
        const uint32_t y0 = (uint32_t)(col * 128 + ((hh ^ (col & 15)) * 8));
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t yt = y0 ^ (uint32_t)(64 * (y == 0 ? ta : 1 - ta));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sv_v4u o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = T::from(Y[y][4 * j + i]);
            *(sv_v4u*)(yw + (yt ^ (16 * j))) = o;
          }
        }
        lq_v4i yo[4];
        {
          const int q8 = 8 * (lane >> 4) + ((lane & 15) >> 2);  // channels q8 and q8 + 4 of this lane's pieces
          const uint32_t b0 = (uint32_t)(q8 * 128 + (((lane & 3) ^ (q8 & 15)) * 8)), b1 = (uint32_t)((q8 + 4) * 128 + (((lane & 3) ^ ((q8 + 4) & 15)) * 8));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const lq_v2i lo = read_columns(yw + (b0 ^ (32 * i))), hi = read_columns(yw + (b1 ^ (32 * i)));
            yo[i] = lq_v4i{lo[0], lo[1], hi[0], hi[1]};
          }
        }
        const int rem = s.len - (s.chunk0 + c) * Q;
        uint16_t* oc = os + (int64_t)(s.chunk0 + c) * Q * ostride;
        const uint32_t o0 = (uint32_t)(lane & 15) * (uint32_t)ostride + 8 * (lane >> 4);
        four = rem >= Q && ch0 + 32 <= p.V;
        if (four) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *(lq_v4i*)(oc + 16 * i * ostride + o0) = yo[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * i + (lane & 15) < rem && ch0 + 8 * (lane >> 4) < p.V) *(lq_v4i*)(oc + 16 * i * ostride + o0) = yo[i];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (more) begin(c + 1);
      if (four) all_but_stores();
      else arrived();
    } else {
      arrived();
      if (more) begin(c + 1);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) sv_settle(S[nt]);
  float* dst = STATES ? p.seg_state + (int64_t)sg * p.H * p.K * p.V + sbase : s.last && keeps ? p.state + slot * p.ss_s + sbase : nullptr;
  if (dst && ch < p.V) {
    const float ui = kHalf ? 1.0f / unit_S : 1.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = channel(nt, hh, r);
        if (n < p.K) dst[(int64_t)n * p.V] = kHalf ? S[nt][r] * ui : S[nt][r];
      }
  }
  if (STATES && threadIdx.x == 0 && part == 0) p.seg_decay[(int64_t)sg * p.H + h] = exp2_fast(total);
}

// The state in front of each segment, in the place of what it adds to one.  A workgroup has 1024 entries of one head's state.
__global__ __launch_bounds__(256) void linear_attention_join_kernel(PromptParams p) {
  const int64_t per = (int64_t)p.K * p.V;
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
    for (int off = 32; off >= 1; off >>= 1) first = min(first + __shfl_xor(first, off, 64), p.segs + 1);
  } else {
    first = seq * n;
  }
  if (at >= per || first > p.segs - n) return;
  const int slot = p.state || p.slots ? sv_slot(p.slots, seq, p.num_slots) : kSlotPad;
  lq_v4f v = {0.f, 0.f, 0.f, 0.f};
  if (p.state && slot >= 0) v = *(const lq_v4f*)(p.state + slot * p.ss_s + h * per + at);
  constexpr int U = 4;  // requested at a time: a chain of one load after the other would be most of this kernel
  float* base = p.seg_state + ((int64_t)first * p.H + h) * per + at;
  const float* dec = p.seg_decay + (int64_t)first * p.H + h;
  const int64_t next = (int64_t)p.H * per;
  for (int i = 0; i < n; i += U) {
    lq_v4f add[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(i + u, n - 2);
      add[u] = *(const lq_v4f*)(base + k * next), d[u] = dec[(int64_t)k * p.H];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= n) break;
      *(lq_v4f*)(base + (i + u) * next) = v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(d[u], v[e], add[u][e]);  // (behind the last one: not used)
    }
  }
}

int check_dims(const lq_linear_attention_prompt_args* a) {
  if (a->nseq <= 0 || a->nheads <= 0 || a->kdim <= 0 || a->kdim % 8 != 0 || a->kdim > 256 || a->vdim <= 0 || a->vdim % 8 != 0) return LQ_ERR_SHAPE;
  if ((a->seq_starts ? a->tokens <= 0 : a->seqlen <= 0) || !sv_act(a->dtype)) return LQ_ERR_SHAPE;
  if ((int64_t)a->nheads * a->vdim > 1 << 23 || a->nheads > 65535 || (int64_t)a->kdim * a->vdim > 1024 * 65535ll) return LQ_ERR_SHAPE;
  return LQ_OK;
}

// How a call is cut: the chunks of a segment.
struct Plan {
  int64_t segs, decays, bytes;
  int waves, parts, seg_chunks, cut;
};
bool plan(const lq_linear_attention_prompt_args* a, Plan& r) {
  const int64_t nseq = a->nseq, most = ((int64_t)(a->seq_starts ? a->tokens : a->seqlen) + Q - 1) / Q;  // chunks of the longest prompt there can be
  const int64_t units = a->seq_starts ? (int64_t)a->tokens / Q + nseq : nseq * most;
  r.waves = a->vdim <= 64 ? 2 : 4;
  r.parts = (a->vdim + 32 * r.waves - 1) / (32 * r.waves);
  const int64_t parts = (int64_t)a->nheads * r.parts;
  // Packed prompts' lengths are not known here: the longest is taken to be two and a half times the mean.
  const double mean = (double)units / nseq, chain = a->seq_starts ? std::min<double>((double)most, 2.5 * mean) : (double)most;
  auto step = [&](double wgs, double one, double two) {
    if (wgs <= 256) return one;
    return a->seq_starts && wgs <= 512 ? one + (two - one) * (wgs / 256 - 1) : two * std::ceil(wgs / 512);
  };
  double best = chain * step((double)nseq * parts, 30, 50);
  r.seg_chunks = (int)most, r.cut = 0;
  int64_t seen = 0;
  for (int64_t k = 2; k <= 256; ++k) {  // segments of the longest
    const int64_t n = std::max<int64_t>(1, (int64_t)std::ceil(chain / k));
    if (n == seen) continue;
    seen = n;
    const double segs = a->seq_starts ? (double)units / n + 0.5 * nseq : (double)(nseq * ((most + n - 1) / n)), ahead = std::max(0.0, segs - nseq);
    const double cost = n * step(segs * parts, 30, 50) + n * step(ahead * parts, 15, 25) + (ahead + 2 * segs) * a->nheads * a->kdim * a->vdim * 4 / 3e5 + 150;
    if (n < most && cost < best) best = cost, r.seg_chunks = (int)n, r.cut = 1;
  }
  const int64_t per = (most + r.seg_chunks - 1) / r.seg_chunks;
  r.segs = a->seq_starts ? std::min<int64_t>(units / r.seg_chunks + nseq, units) : nseq * per;
  if (!r.cut) r.segs = nseq;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  r.decays = r.cut ? up(r.segs * a->nheads * a->kdim * a->vdim * 4) : 0;
  r.bytes = r.decays + (r.cut ? up(r.segs * a->nheads * 4) : 0);
  return sv_fits(nseq, 256) && sv_fits(r.segs * parts + 7, 256) && r.segs * parts < 0x7fffffff;
}

}  // namespace

extern "C" int lq_linear_attention_prompt_workspace_bytes(const lq_linear_attention_prompt_args* a, int64_t* bytes) {
  if (!a || !bytes) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  Plan pl;
  if (rc != LQ_OK) return rc;
  if (!plan(a, pl)) return LQ_ERR_SHAPE;
  *bytes = pl.bytes;
  return LQ_OK;
}

extern "C" int lq_linear_attention_prompt(const lq_linear_attention_prompt_args* a, hipStream_t stream) {
  if (!a || !a->q || !a->k || !a->v || !a->out) return LQ_ERR_NULL;
  const int rc = check_dims(a);
  if (rc != LQ_OK) return rc;
  if ((a->g && !sv_float(a->g_dtype)) || (a->state && a->num_slots <= 0)) return LQ_ERR_SHAPE;
  for (const int64_t s : {a->q_stride_l, a->k_stride_l, a->v_stride_l})
    if (s < 0 || s >= 1 << 24) return LQ_ERR_SHAPE;  // a chunk's rows are reached by 32-bit offsets
  for (const int64_t s : {a->q_stride_b, a->q_stride_l, a->q_stride_h, a->k_stride_b, a->k_stride_l, a->k_stride_h, a->v_stride_b, a->v_stride_l, a->v_stride_h})
    if (s % 8 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->q, 16) || !sv_al(a->k, 16) || !sv_al(a->v, 16) || !sv_al(a->out, 16) || !sv_al(a->state, 16) || a->state_stride_s % 4 != 0 ||
      (a->g && !sv_al(a->g, sv_size(a->g_dtype))) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4))
    return LQ_ERR_SHAPE;
  Plan pl;
  if (!plan(a, pl) || a->workspace_bytes < pl.bytes || !sv_al(a->workspace, 256)) return LQ_ERR_SHAPE;
  if (pl.bytes && !a->workspace) return LQ_ERR_NULL;
  char* ws = (char*)a->workspace;
  PromptParams p = {(const uint16_t*)a->q, a->q_stride_b, a->q_stride_l, a->q_stride_h, (const uint16_t*)a->k, a->k_stride_b, a->k_stride_l, a->k_stride_h,
                    (const uint16_t*)a->v, a->v_stride_b, a->v_stride_l, a->v_stride_h, a->g, a->g_stride_b, a->g_stride_l, a->g_stride_h, a->g_dtype,
                    !a->g || (a->g_stride_b == 0 && a->g_stride_l == 0), a->scale, (uint16_t*)a->out, a->state, a->state_stride_s, a->slots, a->seq_starts,
                    a->num_slots, a->nseq, a->seqlen, a->tokens, a->nheads, a->kdim, a->vdim, pl.cut ? (float*)ws : nullptr,
                    pl.cut ? (float*)(ws + pl.decays) : nullptr, (int)pl.segs, pl.seg_chunks, pl.parts};
  auto grid_of = [&](int64_t segs) { return dim3((unsigned)((segs * a->nheads * pl.parts + 7) / 8 * 8)); };
  const dim3 grid = grid_of(pl.segs), ahead = grid_of(a->seq_starts ? pl.segs : pl.segs - a->nseq), threads(64 * pl.waves);
  const dim3 join((unsigned)a->nseq, (unsigned)a->nheads, (unsigned)(((int64_t)a->kdim * a->vdim + 1023) / 1024));
  auto go = [&](auto t, auto k, auto w) {
    using T = decltype(t);
    constexpr int NT = decltype(k)::value, W = decltype(w)::value;
    if (pl.cut) {
      hipLaunchKernelGGL((linear_attention_chunks_kernel<T, NT, W, true>), ahead, threads, 0, stream, p);
      hipLaunchKernelGGL(linear_attention_join_kernel, join, dim3(256), 0, stream, p);
    }
    hipLaunchKernelGGL((linear_attention_chunks_kernel<T, NT, W, false>), grid, threads, 0, stream, p);
    return lq_check_launch();
  };
  using std::integral_constant;
  auto waves = [&](auto t, auto k) { return pl.waves == 2 ? go(t, k, integral_constant<int, 2>{}) : go(t, k, integral_constant<int, 4>{}); };
  auto with = [&](auto t) {
    if (a->kdim <= 32) return waves(t, integral_constant<int, 1>{});
    if (a->kdim <= 64) return waves(t, integral_constant<int, 2>{});
    if (a->kdim <= 128) return waves(t, integral_constant<int, 4>{});
    return waves(t, integral_constant<int, 8>{});
  };
  return a->dtype == LQ_DT_F16 ? with(F16{}) : with(BF16{});
}
