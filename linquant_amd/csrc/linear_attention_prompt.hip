// lq_linear_attention_prompt: linear attention over prompts of any lengths, from and into an fp32 state.
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t
// in chunks of 64 tokens.  With c_t = sum of g up to t inside a chunk and S the state in front of it,
//   o_t = scale (exp(c_t) S^T q_t + sum_{s <= t} exp(c_t - c_s) (q_t . k_s) v_s)
//   S'  = exp(c_63) S + sum_s exp(c_63 - c_s) k_s v_s^T
// which are products of matrices.  Three kernels:
//   states     per segment of a prompt but the last: the state at its end if it starts from zero, and what it multiplies an earlier one by;
//   join       walks the segments: the state in front of each.  (states and join: only where prompts are cut into segments, because
//              prompts times heads are too few for 256 compute units)
//   chunks     walks a segment chunk by chunk, the state in registers
// A workgroup has 128 columns of a head's state (64 where there are no more), a wave 32 of them over all K: the state and the chunk's products
// with it never leave the wave.  q, k and v come to LDS by fetches that pass no registers, the next chunk's while one is multiplied.
//
// What bounds it.  2 prompts of 8192, 32 heads of 128 by 128, fp16: chunks 129 us for 537 MB (4.2 TB/s), states 66 for half of that once more,
// join 13; a copy's rate for what has to move is 103.  10 packed prompts of 6949 tokens, 16 heads: 52, 26 and 8, by steps one after the other (up to
// 32 chunks in a prompt, 6 to a segment).  500 tokens of 16 heads, bf16: 9.7, 7.6 and 3.9, three launches and a chunk's step in each of two.  In a step of
// the long prompts (fp16, two workgroups to a compute unit, 11300 cycles): waiting for the chunk 450, its successor's fetches 1200, q k 1190, weights and
// rounding 1130, meeting 850, the state 1950, outputs 3100, operands of v 1490.  Units that go by weighted v and outputs formed 2^8 times as large (fp16,
// below) are 110 and 130 of these; with v's own sizes the calls took 1 to 4 % less.
// Tried and no faster: fetches spread between the products, outputs' products between the state's, segments in the other order (so that the
// caches still have what the states read last), a segment's own state as two pieces of 16 bits.
//
// Precision.  Activations enter the matrix products as they are, all sums are fp32, and so is the state.  What is formed in fp32 on the way
// and reaches only o, which is rounded to the activations' type itself (weighted q . k, the state that q multiplies), enters rounded to
// that type: half a step of each term.  What the state gathers over a prompt (weighted v) enters as two (fp16) or three (bf16) pieces of the
// type: off by 2^-22 of itself, or not at all (two of bf16: the state 2.4e-6 off, here and in fp16 below 1e-6).  bf16 has the range of fp32.
// fp16: after a multiplication by a power of two that brings the largest of what is multiplied (a channel's state; its weighted v; a row of 32 weighted
// q . k) below 2^15, so no size of activations overflows.  Below 2^-14 fp16 is evenly spaced, which bounds what is far below that largest: weighted v is
// off by 2^-26 of the channel's largest weighted v of its chunk (by the largest v itself, which may have decayed to nothing, states were 0.3 off), weighted
// q . k by 2^-29 of the largest of its 32 (old tokens of large v still count there: 2^-17, with outputs formed at their own size, cost outputs five
// times that half step), the state that q multiplies by 2^-25 of its channel's largest.
// Decays are summed over a chunk in 32 bits, each a factor of 2^-160 at least: behind 32 tokens that decay to nothing the weights of the chunk's others are
// off by up to 3.4e-4 of themselves, behind 52 of them by 9e-4 (half a step of fp16 is 4.9e-4); the state's weights, summed from the end, are not.  Sums of
// whole parts and of fractions by themselves, where a chunk's decays are that large, would make every call 1 % longer.
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
  const float* g;
  int64_t sg_b, sg_l, sg_h;
  int g_same;  // g_same: one decay for all tokens of a head
  float log_scale;  // of its size over post, a power of two
  float post;       // outputs are multiplied by it at the end: a power of two, one where the scale is of ordinary size
  int negative;
  uint16_t* out;
  float* state;
  int64_t ss_s;
  const int32_t* slots;
  const int32_t* starts;
  int num_slots, nseq, seqlen, tokens, H, K, V;
  float* seg_state;  // [place][H][K][V], or NULL: prompts are not cut
  float* seg_decay;  // [place][H]
  int segs, seg_chunks, parts;
  int blocks, places;  // packed prompts: STATES' units, and places of the workspace
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
// the largest of the first 32 lanes' non-negative values (whole numbers order like them)
LQ_DEV float first_half_top(float f) {
  uint32_t v = __float_as_uint(f);
#define LQ_TOP(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false))
  LQ_TOP(0xB1);   // lanes 1 0 3 2
  LQ_TOP(0x4E);   // lanes 2 3 0 1
  LQ_TOP(0x141);  // mirrored halves of a row of 16
  LQ_TOP(0x140);  // mirrored rows
  LQ_TOP(0x142);  // the last lane of a row to the next row
#undef LQ_TOP
  return __int_as_float(__builtin_amdgcn_readlane((int)v, 31));
}
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

// Segments have places in the workspace if their prompt has more than one.  Packed prompts, w tokens to a segment: prompt r of those that have more
// than w, from token b on, has its places from b / w + r on, a segment each.  Ascending prompts so have places of their own, and however many short prompts
// there are, places are no more than tokens / w and the prompts that can be longer than w.  (Starts that do not ascend could lead beyond them: `fit` tells.)
struct Segment {
  int seq, begin, len;  // tokens of the sequence
  int chunk0, chunks;   // its first chunk in the sequence, how many
  int place;            // of the segment
  bool first, last, fit;
};
LQ_DEV int tokens_of(const PromptParams& p, int s, int& begin) {  // 0 for what is no prompt
  int b = 0, e = 0;
  if (s < p.nseq) b = p.starts[s], e = p.starts[s + 1];
  if (b < 0 || e > p.tokens || e < b) b = e = 0;
  begin = b;
  return e - b;
}
LQ_DEV int segments_of(const PromptParams& p, int len) { return ((int)(((uint32_t)len + (Q - 1)) / Q) + p.seg_chunks - 1) / p.seg_chunks; }
// STATES: the segment, not a prompt's last one, that starts at a token of sg w .. sg w + w - 1.  There is one at most, and its prompt has token sg w + w too.
template <bool STATES>
LQ_DEV Segment segment_of(const PromptParams& p, int sg) {
  Segment r;
  int index = 0, base = 0;  // of the prompt's segments; the first one's place
  if (p.starts) {
    const int lane = threadIdx.x & 63;
    const uint32_t w = (uint32_t)p.seg_chunks * Q;
    const int64_t behind = (int64_t)(sg + 1) * w;
    int before = 0, cut = 0;
    r.seq = -1;
    for (int s0 = 0; s0 < p.nseq; s0 += 64) {
      int b;
      const int len = tokens_of(p, s0 + lane, b);
      uint64_t found;
      int n = 0, sum = 0, total = 0;
      if (STATES) {
        found = __ballot(b < behind && behind < (int64_t)b + len);
      } else {
        sum = n = segments_of(p, len);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int o = __shfl_up(sum, off, 64);
          sum += lane >= off ? o : 0;
        }
        total = __builtin_amdgcn_readlane(sum, 63);
        found = sg < before + total ? __ballot(sg < before + sum) : 0;
      }
      const uint64_t longer = __ballot((uint32_t)len > w);
      if (found) {
        const int l = __builtin_ctzll(found);
        r.seq = s0 + l, r.begin = __builtin_amdgcn_readlane(b, l), r.len = __builtin_amdgcn_readlane(len, l);
        const int at = (int)((uint32_t)r.begin / w);
        index = STATES ? sg - at : sg - before - __builtin_amdgcn_readlane(sum - n, l), base = at + cut + __builtin_popcountll(longer & ((1ull << l) - 1));
        break;
      }
      before += total, cut += __builtin_popcountll(longer);
      if (before >= p.segs) break;  // (starts that do not ascend can name far more than there are, and their sum must not wrap)
    }
  } else {
    const int per = segments_of(p, p.seqlen);
    r.seq = sg / per, r.begin = 0, r.len = p.seqlen, base = r.seq * per, index = sg - base;
  }
  if (r.seq >= 0) {
    const int nc = (r.len + Q - 1) / Q;
    r.chunk0 = index * p.seg_chunks, r.place = base + index;
    r.chunks = min(p.seg_chunks, nc - r.chunk0), r.first = r.chunk0 == 0, r.last = r.chunk0 + r.chunks >= nc;
    r.fit = !p.starts || (r.first && r.last) || base <= p.places - segments_of(p, r.len);
  }
  return r;
}

// A wave has 32 channels of v of a head: the state's K x 32 as accumulators (rows channels of k, columns those of v).  STATES: only the
// segment's state and decay.  A workgroup's waves, up to W, share the chunk's q and k in LDS and the 32 x 32 tiles of weighted q . k that each
// of them forms one or two of; each wave's v comes the same way, a chunk ahead.  o is formed with channels as rows, so that a lane has 32
// bytes of a token's row between two exchanges of its halves and stores them from registers.
//
// The state's accumulators are not multiplied by the decay of every chunk: they hold the state over 2^total, which multiplies the rows of q S
// (with exp(c_t)) and divides the weights of v, until total falls below kFloor.
template <typename T, int NT, int W, bool STATES>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(NT == 8 ? 1 : 2, NT == 8 ? 1 : 2))) void linear_attention_chunks_kernel(PromptParams p) {
  constexpr bool kHalf = std::is_same<T, F16>::value;
  constexpr int kLift = kHalf ? 8 : 0;  // outputs are formed 2^kLift times as large: weighted q . k below 2^-14 of that would be evenly spaced
  constexpr float kFloor = kHalf ? -6.0f : 0.0f;  // (bf16: no room above the formula's range, which weights above one would need)
  constexpr float kUnit = kHalf ? 16.0f : 1.0f;  // of v and the state where they are of ordinary size
  constexpr int RB = 64 * NT, PR = 4 * NT, kTile = Q * RB;  // bytes and pieces of a row of q or k, bytes of a chunk's
  constexpr int kFetch = kTile / (1024 * W), kRows = 1024 / RB;  // fetches of a wave, rows of each
  constexpr int PT = W == 2 ? 2 : 1;                           // tiles of q . k of a wave
  __shared__ __align__(1024) char kbuf[2][kTile];
  __shared__ __align__(1024) char qbuf[STATES ? 16 : kTile];
  __shared__ __align__(256) uint16_t vbuf[W][Q * 32];
  __shared__ __align__(16) char pbuf[STATES ? 16 : 8 * 1024];  // weighted q . k, operands 4 tt + ks; (0, 2) and (0, 3) are zero
  __shared__ __align__(16) float punit[kHalf && !STATES ? 4 * 32 : 4];  // fp16: 1 / unit of each tile's columns t, tiles 2 tt + st
  __shared__ int podd[4];                                       // fp16: whether a tile has a unit that is not 1
  __shared__ __align__(16) float tok[W][3 * Q];                 // each wave's c, weights of v, exp2(c + total) |scale|
  __shared__ __align__(16) float gbuf[W][64];                   // each wave's decays of a chunk
  __shared__ __align__(16) float vunit[kHalf && !STATES ? W : 1][32];  // fp16: scale / (unit_S read) of each wave's channels
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), hh = lane >> 5, col = lane & 31;
  // Workgroups go round the 8 XCDs in launch order; the parts of one head, which read the same q and k, and the heads of one segment, whose
  // rows lie side by side, go to one.
  const int at = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3), per = p.H * p.parts;
  int sg = uniform(at / per);
  const int h = uniform((at - sg * per) / p.parts), part = uniform(at - sg * per - h * p.parts);
  if (STATES && !p.starts) sg = uniform(sg + sg / max(p.segs / p.nseq - 1, 1));  // (as many segments to each prompt, the last ones left out)
  if (sg >= (STATES && p.starts ? p.blocks : p.segs)) return;
  Segment s = segment_of<STATES>(p, sg);
  if (s.seq < 0 || (STATES && s.last) || !s.fit) return;
  s.seq = uniform(s.seq), s.begin = uniform(s.begin), s.len = uniform(s.len), s.chunk0 = uniform(s.chunk0), s.chunks = uniform(s.chunks);
  const int64_t place = uniform(s.place);
  const int ch0 = (part * W + wave) * 32, ch = ch0 + col, chc = min(ch, p.V - 1);
  const bool live = ch0 < p.V;  // a wave without channels only helps
  const int slot = p.state || p.slots ? uniform(sv_slot(p.slots, s.seq, p.num_slots)) : kSlotPad;
  const bool keeps = p.state && slot >= 0, bad = slot == kSlotBad;
  const int64_t row0 = p.starts ? s.begin : (int64_t)s.seq * p.seqlen;  // of the dense output
  const int64_t ostride = (int64_t)p.H * p.V, first = (int64_t)s.chunk0 * Q;
  uint16_t* os = p.out + ((row0 + first) * p.H + h) * p.V + ch0;
  const int64_t b = p.starts ? 0 : s.seq, l0 = (p.starts ? s.begin : 0) + first;
  const uint16_t* qs = p.q + b * p.sq_b + l0 * p.sq_l + h * p.sq_h;
  const uint16_t* ks_ = p.k + b * p.sk_b + l0 * p.sk_l + h * p.sk_h;
  const uint16_t* vs = p.v + b * p.sv_b + l0 * p.sv_l + h * p.sv_h + (live ? ch0 : 0);
  const int64_t g0 = b * p.sg_b + l0 * p.sg_l + h * p.sg_h;

  v16f S[NT];
  const int64_t sbase = (int64_t)h * p.K * p.V + chc;
  {
    const float* src = STATES ? nullptr : (p.seg_state && !(s.first && s.last)) ? p.seg_state + place * p.H * p.K * p.V + sbase : keeps ? p.state + slot * p.ss_s + sbase : nullptr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[nt][r] = 0.0f;
    if (src) {  // (all requested together: none behind a condition of its own)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[nt][r] = src[min(channel(nt, hh, r), p.K - 1) * (int64_t)p.V];
      if (p.K < 32 * NT) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 16; ++r) S[nt][r] = channel(nt, hh, r) < p.K ? S[nt][r] : 0.0f;
      }
    }
  }

  if (!STATES) {
    const lq_v4i zero = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < 128; i += 64 * W) *(lq_v4i*)(pbuf + (2 * 64 + i) * 16) = zero;  // (read behind two barriers)
  }
  // channels behind K: zeros, left there for good (nothing is fetched over them)
  const bool whole = p.K == 32 * NT;
  if (!whole) {
    const lq_v4i zero = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < kTile / 16; i += 64 * W) {
      *(lq_v4i*)(kbuf[0] + i * 16) = zero, *(lq_v4i*)(kbuf[1] + i * 16) = zero;
      if (!STATES) *(lq_v4i*)(qbuf + i * 16) = zero;
    }
    __syncthreads();
  }
  // (addresses are made of a lane number that the compiler does not know to be the same: kept over the loop they are registers that it lacks)
  auto fresh = [&] {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };
  // rows of a chunk; behind the prompt its last one again (at weight zero)
  auto rows_of = [&](const uint16_t* base, int64_t stride, char* to, int left) {
    const int lane = fresh(), row = wave * kFetch * kRows + lane / PR, c = (lane % PR) ^ order<NT>(row);  // of the first fetch
    to += wave * kFetch * 1024;
    if (whole && left >= Q) {  // (the i-th fetch: rows i kRows on, their bits apart from the first one's, and so the order's)
      const uint32_t off = (uint32_t)row * (uint32_t)stride * 2u;
#pragma unroll
      for (int i = 0; i < kFetch; ++i) sv_fetch16(base + i * kRows * stride, (uint32_t)((c ^ order<NT>(i * kRows)) << 4) + off, to + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kFetch; ++i) {
        const int ci = c ^ order<NT>(i * kRows);
        const uint32_t off = (uint32_t)min(row + i * kRows, left - 1) * (uint32_t)stride * 2u + (uint32_t)ci * 16u;
        if (ci * 8 < p.K) sv_fetch16(base, off, to + i * 1024);
      }
    }
  };
  int qleft = s.len - (int)first, kleft = qleft, vleft = qleft;
  auto fetch_q = [&] { rows_of(qs, p.sq_l, qbuf, qleft), qs += Q * p.sq_l, qleft -= Q; };
  auto fetch_k = [&](int c) { rows_of(ks_, p.sk_l, kbuf[c & 1], kleft), ks_ += Q * p.sk_l, kleft -= Q; };
  const float* gs = p.g + g0;
  auto fetch_v = [&] {  // and the decays
    const int lane = fresh();
    if (live) {
      const uint32_t vcol = (uint32_t)min(8 * (lane & 3), p.V - 8 - ch0);
      if (vleft >= Q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv_fetch16(vs + 16 * i * p.sv_l, ((uint32_t)(lane >> 2) * (uint32_t)p.sv_l + vcol) * 2u, vbuf[wave] + 16 * 32 * i);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv_fetch16(vs, ((uint32_t)min(16 * i + (lane >> 2), vleft - 1) * (uint32_t)p.sv_l + vcol) * 2u, vbuf[wave] + 16 * 32 * i);
      }
    }
    if (!p.g_same) sv_fetch4(gs, (uint32_t)min(lane, vleft - 1) * (uint32_t)p.sg_l * 4u, gbuf[wave]);
    vs += Q * p.sv_l, gs += Q * p.sg_l, vleft -= Q;
  };
  const float same = p.g && p.g_same ? lane_of(*gs, 0) : 0.0f;  // (waited for here)
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
  auto meet = [&] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  fetch_k(0);
  if (!STATES) fetch_q();
  fetch_v();
  arrived();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) asm volatile("" : "+v"(S[nt]));  // (else the compiler waits for its loads in every chunk, and for all behind them)

  // What a chunk's products need of the wave's own: v in registers, decays in LDS, the state's unit.
  float* my = tok[wave];
  const float log_scale = p.log_scale + kLift;
  lq_v4i xp[4] = {};  // this lane's channel, tokens in the order of an operand
  auto x = [&](int ks, int i) { return T::to((uint16_t)((uint32_t)xp[ks][i >> 1] >> (16 * (i & 1)))); };
  float total = 0.0f, whole_decay = 0.0f;            // what the accumulators are over, the segment's decay so far (powers of two)
  float fold = 1.0f;                                 // what the accumulators are multiplied by in this chunk, mostly one
  // fp16: powers of two.  The accumulators hold the channel's state, and its weighted v enters them, times unit_S: `common` in all of the wave's
  // channels but those of other sizes.  What q multiplies is the accumulators times `read`.
  float unit_S = 1.0f, read = 1.0f, common = 1.0f;
  bool alike = true, calm = true, scaled = false;  // the same for the wave: unit_S is `common` in all channels; and read is one; the accumulators are multiplied
  auto begin = [&](int c) {
    const int lane = fresh(), hh = lane >> 5;
    const int rem = s.len - (s.chunk0 + c) * Q;
    float mx = 0.0f, ms = 0.0f;  // the channel's largest v and accumulator
    if (live) {
      const uint16_t* xl = vbuf[wave] + (4 * hh + ((lane & 15) >> 2)) * 32 + (lane & 16) + 4 * (lane & 3);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const lq_v2i lo = read_columns(xl + 16 * ks * 32), hi = read_columns(xl + (16 * ks + 8) * 32);
        xp[ks] = lq_v4i{lo[0], lo[1], hi[0], hi[1]};
      }
      if constexpr (kHalf) {
        // Both halves of a dword at once: magnitudes order like whole numbers.
        typedef uint16_t v2u __attribute__((ext_vector_type(2)));
        v2u top2 = {0, 0};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(v2u, (uint32_t)xp[ks][i] & 0x7fff7fffu));
        if (__ballot(max(top2[0], top2[1]) >= 0x7c00) != 0) {  // those that are no numbers must not hide the others': 2^10 above themselves they are negative
          typedef int16_t v2s __attribute__((ext_vector_type(2)));
          v2s s2 = {0x400, 0x400};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2 = __builtin_elementwise_max(s2, __builtin_bit_cast(v2s, ((uint32_t)xp[ks][i] & 0x7fff7fffu) + 0x04000400u));
          top2 = __builtin_bit_cast(v2u, s2) - (uint16_t)0x400;
        }
        float m4[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (no number where the lane has one that is none: its scale does not matter then)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 16; ++e) m4[(e >> 1) & 3] = __builtin_elementwise_maximum(m4[(e >> 1) & 3], __builtin_fabsf(S[nt][e]));
        const float m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m4[0], m4[1]), __builtin_elementwise_maximum(m4[2], m4[3]));
        mx = channel_top(T::to(max(top2[0], top2[1]))), ms = channel_top(finite_size(m));
      }
    }
    float log_read = log_scale;  // what the accumulators' products are multiplied by besides their decays, for all channels
    if (kHalf && !STATES && live) {
      const bool plain = ms == 0.0f || (ms >= 1.0f && ms < 0x1p15f);
      read = plain ? 1.0f : scale_for<13, -114, 100>(ms);
      calm = alike && __ballot(!plain) == 0;
      if (calm) {
        log_read -= (float)((int)(__float_as_uint(common) >> 23) - 127);
      } else {  // each channel by its own
        log_read = 0.0f;
        if (lane < 32) vunit[wave][lane] = exp2_fast(log_scale) * pow2_inverse(read) * pow2_inverse(unit_S);
      }
    }
    {
      // one factor of 2^-160 is zero in 32 bits, and sums of larger ones would cost the tokens behind them their last bits
      const float e = sv_decay(p.g_same ? same : gbuf[wave][lane]) * kLog2e, one = e < -160.0f ? -160.0f : e;
      float cs, behind;
      if (p.g_same) {
        cs = one * (float)min(lane + 1, rem), behind = one * (float)max(min(rem, Q) - 1 - lane, 0);
      } else {
        const float a = lane < rem ? one : 0.0f;
        cs = sums_upto(a), behind = sums_behind(a, lane);
      }
      const float last = lane_of(cs, 63), after = total + last;
      whole_decay += last;
      my[lane] = cs;
      if (!STATES) my[2 * Q + lane] = exp2_fast(cs + total + log_read);
      const bool now = after < kFloor;
      fold = now ? exp2_fast(after) : 1.0f, total = now ? 0.0f : after, scaled = now;
      const float weight = lane < rem ? exp2_fast(behind - total) : 0.0f;
      my[Q + lane] = weight;
      if (kHalf && live) {
        // A unit keeps the largest weighted v of its channel between 2 and 2^15, so that the second piece, evenly spaced by 2^-24, is off by 2^-26 of it at
        // most.  Weights rise from token to token, and for most chunks those of token 0, 56 and 63 tell that it does.
        float k = unit_S;
        if (c == 0) k = common = kUnit;
        const float least = lane_of(weight, 0) * k, most = exp2_fast(-total) * k;
        bool search = !alike || __ballot(!(mx == 0.0f || (mx * least >= 2.0f && mx * most < 0x1p15f))) != 0;
        if (search && alike) {
          float late = 0.0f;
#pragma unroll
          for (int i = 4; i < 8; ++i) late = fmaxf(late, __builtin_fabsf(x(3, i)));
          late = channel_top(finite_size(late)) * lane_of(weight, 56) * k;
          search = __ballot(!(mx == 0.0f || ((mx * least >= 2.0f || late >= 2.0f) && mx * most < 0x1p15f))) != 0;
        }
        if (search) {
          float m2[2] = {0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const lq_v4f f4 = *(const lq_v4f*)(my + Q + 16 * ks + 8 * j + 4 * hh);
#pragma unroll
              for (int e = 0; e < 4; ++e) m2[e & 1] = fmaxf(m2[e & 1], __builtin_fabsf(f4[e] * x(ks, 4 * j + e)));
            }
          const float mw = channel_top(finite_size(fmaxf(m2[0], m2[1]))), top = first_half_top(mw);
          if (top > 0.0f && !(top * common >= 2.0f && top * common < 0x1p14f)) common = scale_for<10, -30, 90>(top);
          k = mw == 0.0f || mw * common >= 2.0f ? common : mw * unit_S >= 2.0f && mw * unit_S < 0x1p14f ? unit_S : scale_for<10, -30, 90>(mw);
        }
        if (search || c == 0) {
          k = fminf(k, unit_S * scale_for<100, 0, 100>(ms));  // (a state far above its v would leave 32 bits)
          const float change = k * pow2_inverse(unit_S);
          unit_S = k, fold *= change;
          alike = __ballot(k != common) == 0, scaled |= __ballot(change != 1.0f) != 0;
        }
      }
    }
  };
  begin(0);
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
  // tiles of q . k: columns t of tile tt, rows s of tile st.  Y[0] has the columns of tile ta, Y[1] of the other
  const int ta = wave == 0 && W == 4 ? 0 : 1;
  for (int c = 0; c < s.chunks; ++c) {
    const bool more = c + 1 < s.chunks;
    meet();  // every wave's share of this chunk's q and k is there, and the chunk in front is read
    const char* kb = kbuf[c & 1];
    if (more) {
      fetch_k(c + 1);
      fetch_v();  // (v is in registers since `begin`)
    }
    v16f Y[2];
    if constexpr (!STATES) {
      const int lane = fresh(), hh = lane >> 5, col = lane & 31;
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
      const int a0 = col * RB + ((hh ^ order<NT>(col)) << 4);  // row lane & 31, pieces 2 ks + hh
      auto products = [&](auto plain) {
        constexpr int R = 2;
        lq_v4i q0[R], q1[R], k0[R];
        auto ask = [&](int ks) {
          const int o = a0 ^ (ks << 5);
          q0[ks % R] = *(const lq_v4i*)(qa + o), q1[ks % R] = *(const lq_v4i*)(qz + o), k0[ks % R] = *(const lq_v4i*)(kx + o);
        };
#pragma unroll
        for (int ks = 0; ks + 1 < R; ++ks) ask(ks);
#pragma unroll
        for (int ks = 0; ks < 2 * NT; ++ks) {
          if (ks + R - 1 < 2 * NT) ask(ks + R - 1);
          __builtin_amdgcn_sched_barrier(0);  // (operands of all steps read ahead are registers that it lacks)
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = S[ks >> 1][8 * (ks & 1) + i];
          lq_v4i sh;
          if constexpr (decltype(plain)::value) sh = round8<T>(v);
          else sh = round8<T>(v, read);
          P[0] = mfma<T>(k0[ks % R], q0[ks % R], P[0]);
          if constexpr (PT == 2) P[1] = mfma<T>(k0[ks % R], q1[ks % R], P[1]);
          Y[0] = mfma<T>(sh, q0[ks % R], Y[0]);
          Y[1] = mfma<T>(sh, q1[ks % R], Y[1]);
        }
      };
      if (!kHalf || calm) {
        products(std::true_type{});
      } else if constexpr (kHalf) {
        products(std::false_type{});
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const lq_v4f u4 = *(const lq_v4f*)(vunit[wave] + 8 * j + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) Y[0][4 * j + e] *= u4[e], Y[1][4 * j + e] *= u4[e];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      {
        const float ea = my[2 * Q + 32 * ta + col], ez = my[2 * Q + 32 * (1 - ta) + col];
#pragma unroll
        for (int e = 0; e < 16; ++e) Y[0][e] *= ea, Y[1][e] *= ez;
      }
      // weighted q . k, rounded, for all of the workgroup's waves
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        const int tt = i == 0 ? ta : 1 - ta;
        if ((W == 4 && wave == 3) || (W == 2 && i == 1 && wave == 1)) continue;
        const float ct = my[32 * tt + col] + log_scale;
        float w[16], m = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const lq_v4f c4 = *(const lq_v4f*)(my + 32 * st + 8 * j + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[4 * j + e] = P[i][4 * j + e] * exp2_fast(ct - c4[e]);
          }
        }
        if (st == tt) {  // nothing of tokens behind the column's
          const int t = col - 4 * hh;
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = 8 * (e >> 2) + (e & 3) > t ? 0.0f : w[e];
        }
        if constexpr (kHalf) {
#pragma unroll
          for (int e = 0; e < 16; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(w[e]));
          // (a column with an infinity or a NaN is none whatever its unit)
          m = channel_top(finite_size(m));
          const bool plain = m == 0.0f || (m >= 0x1p4f && m < 0x1p15f);
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
      meet();  // every wave has read the chunk's q, and the weighted q . k is there
      if (more) fetch_q();
    }
    // the state behind the chunk
    if (scaled) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 16; ++e) S[nt][e] *= fold;
    }
    __builtin_amdgcn_sched_barrier(0);
    {
      const int kl = fresh(), hh = kl >> 5;
      constexpr int N = kHalf ? 2 : 3;
      lq_v4i kt[3], w[2][N];
      lq_v4f w4[2][2];
      auto ask = [&](int i) { kt[i % 3] = k_columns(kb, kl, i % NT, i / NT); };  // operand i = NT ks + nt
      auto ask_w = [&](int ks) {
#pragma unroll
        for (int j = 0; j < 2; ++j) w4[ks & 1][j] = *(const lq_v4f*)(my + Q + 16 * ks + 8 * j + 4 * hh);
      };
      auto pair = [&](int ks, int q) {  // a quarter of step ks' weighted v
        const lq_v4f& f = w4[ks & 1][q >> 1];
        const float u = kHalf ? unit_S : 1.0f;
        int o[3];
        split2<T>(f[2 * (q & 1)] * u, x(ks, 2 * q), f[2 * (q & 1) + 1] * u, x(ks, 2 * q + 1), o);
#pragma unroll
        for (int n = 0; n < N; ++n) w[ks & 1][n][q] = o[n];
      };
      ask_w(0);
      ask(0);
      ask(1);
      ask_w(1);
      reads_stay();
#pragma unroll
      for (int q = 0; q < 4; ++q) pair(0, q);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int i = NT * ks + nt;
          if (i + 2 < 4 * NT) ask(i + 2);
          if (nt == NT - 1 && ks < 2) ask_w(ks + 2);
          __builtin_amdgcn_sched_barrier(0);
          // (the next step's weighted v is formed between these products: one issued behind another of the same tile waits for it)
#pragma unroll
          for (int n = 0; n < N; ++n) {
            S[nt] = mfma<T>(kt[i % 3], w[ks & 1][n], S[nt]);
            __builtin_amdgcn_sched_barrier(0);
            if (ks < 3) {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (q * NT * N / 4 == nt * N + n) pair(ks + 1, q);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!STATES) {
      bool four = false;  // whether this wave has stored four times
      if (live) {
        const int lane = fresh(), hh = lane >> 5, col = lane & 31;
        // A v that is no number must not reach the tokens in front of it, which the product below multiplies by zero: the state, which all of
        // the chunk's tokens reach, tells.  Then such tokens are left out and every output of the channel from them on is NaN.
        const bool odd = bad || __ballot(S[0][0] != S[0][0]) != 0;
        int from = bad ? 0 : Q;  // of this lane's channel
        if (odd) {
          asm volatile("");  // (not to be computed ahead)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!(__builtin_fabsf(x(ks, i)) < __builtin_inff())) {
                from = min(from, entry(ks, hh, i));
                xp[ks][i >> 1] &= i & 1 ? 0xffff : 0xffff0000;
              }
          from = min(from, __shfl_xor(from, 32, 64));
        }
        bool apart = false;
        if constexpr (kHalf) apart = uniform(podd[0] | podd[2] | podd[3]) != 0;
        auto weighted = [&](int tt, int ks) { return *(const lq_v4i*)(pbuf + (4 * tt + ks) * 1024 + lane * 16); };
        if (!apart) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int y = 0; y < 2; ++y) Y[y] = mfma<T>(xp[ks], weighted(y == 0 ? ta : 1 - ta, ks), Y[y]);
        } else if constexpr (kHalf) {  // units of their own for the columns of a tile
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tt = y == 0 ? ta : 1 - ta;
            for (int st = 0; st <= tt; ++st) {
              v16f d = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              d = mfma<T>(st ? xp[2] : xp[0], weighted(tt, 2 * st), d);
              d = mfma<T>(st ? xp[3] : xp[1], weighted(tt, 2 * st + 1), d);
              sv_settle(d);
              const float u = podd[2 * tt + st] ? punit[(2 * tt + st) * 32 + col] : 1.0f;
#pragma unroll
              for (int e = 0; e < 16; ++e) Y[y][e] = __builtin_fmaf(d[e], u, Y[y][e]);
            }
          }
        }
        sv_settle(Y[0]), sv_settle(Y[1]);
        if (odd) {  // (channel of register e: entry(e / 8, hh, e % 8))
          asm volatile("");
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int f = __shfl(from, entry(e >> 3, hh, e & 7), 64);
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (32 * (y == 0 ? ta : 1 - ta) + col >= f) Y[y][e] = __builtin_nanf("");
          }
        }
        // A lane has four channels of eight, the other half of the wave the other four: with every second eight exchanged it has whole eights.
        const int rem = s.len - (s.chunk0 + c) * Q;
        four = rem >= Q && ch0 + 32 <= p.V;
        char* oc = (char*)(os + (int64_t)c * Q * ostride);
        const uint32_t o0 = ((uint32_t)col * (uint32_t)ostride + 8 * hh) * 2u;  // (a chunk's rows are reached by 32-bit offsets)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int tt = y == 0 ? ta : 1 - ta;
          float a[8], z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = Y[y][e], z[e] = Y[y][8 + e];
          lq_v4i two[2];
          if constexpr (kHalf) {
            const float post = p.post * (1.0f / (1 << kLift));
            two[0] = round8<T>(a, post), two[1] = round8<T>(z, post);
          } else {
            if (p.post != 1.0f) {
              asm volatile("");  // (a branch)
#pragma unroll
              for (int e = 0; e < 8; ++e) a[e] *= p.post, z[e] *= p.post;
            }
            two[0] = round8<T>(a), two[1] = round8<T>(z);
          }
          if (p.negative) {
            const int sign = (int)0x80008000u;
#pragma unroll
            for (int q = 0; q < 4; ++q) two[0][q] ^= sign, two[1][q] ^= sign;
          }
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const auto r0 = __builtin_amdgcn_permlane32_swap((uint32_t)two[k2][0], (uint32_t)two[k2][2], false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap((uint32_t)two[k2][1], (uint32_t)two[k2][3], false, false);
            const lq_v4i o = {(int)r0[0], (int)r1[0], (int)r0[1], (int)r1[1]};
            char* to = oc + 64 * tt * ostride + 32 * k2;
            if (four) *(lq_v4i*)(to + o0) = o;
            else if (32 * tt + col < rem && ch0 + 16 * k2 + 8 * hh < p.V) *(lq_v4i*)(to + o0) = o;
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // Memory operations end in order: v and the decays, requested at the chunk's beginning, are in front of q and the stores.
      const bool counted = four && whole;
      if (counted) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kFetch + 4) : "memory");
      else arrived();
      if (more) begin(c + 1);
      if (counted) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    } else {
      arrived();
      if (more) begin(c + 1);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) sv_settle(S[nt]);
  float* dst = STATES ? p.seg_state + place * p.H * p.K * p.V + sbase : s.last && keeps ? p.state + slot * p.ss_s + sbase : nullptr;
  if (dst && ch < p.V) {
    const float ui = exp2_fast(total) * (kHalf ? pow2_inverse(unit_S) : 1.0f);
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) dst[channel(nt, hh, r) * (int64_t)p.V] = S[nt][r] * ui;
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (channel(nt, hh, r) < p.K) dst[channel(nt, hh, r) * (int64_t)p.V] = S[nt][r] * ui;
    }
  }
  if (STATES && threadIdx.x == 0 && part == 0) p.seg_decay[place * p.H + h] = exp2_fast(whole_decay);
}

// The state in front of each segment, in the place of what it adds to one.  A workgroup has 1024 entries of one head's state.
__global__ __launch_bounds__(256) void linear_attention_join_kernel(PromptParams p) {
  const int64_t per = (int64_t)p.K * p.V;
  const int h = blockIdx.y, at = (blockIdx.z * 256 + threadIdx.x) * 4;
  int seq = blockIdx.x, n, first;
  if (p.starts) {  // of the prompts that are cut the one with this number
    const uint32_t w = (uint32_t)p.seg_chunks * Q;
    int left = seq, s0 = 0, b = 0, len = 0;
    uint64_t longer = 0;
    for (; s0 < p.nseq; s0 += 64) {
      len = tokens_of(p, s0 + (threadIdx.x & 63), b);
      longer = __ballot((uint32_t)len > w);
      if (left < __builtin_popcountll(longer)) break;
      left -= __builtin_popcountll(longer);
    }
    if (s0 >= p.nseq) return;
    for (; left > 0; --left) longer &= longer - 1;
    const int l = __builtin_ctzll(longer);
    first = (int)((uint32_t)__builtin_amdgcn_readlane(b, l) / w) + seq, seq = s0 + l, n = segments_of(p, __builtin_amdgcn_readlane(len, l));
    if (first > p.places - n) return;
  } else {
    n = segments_of(p, p.seqlen), first = seq * n;
  }
  if (at >= per) return;
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
  int64_t segs, blocks, longer, places, decays, bytes;  // packed prompts: blocks of a segment's tokens, prompts that can be longer than one
  int waves, parts, seg_chunks, cut;
};
bool plan(const lq_linear_attention_prompt_args* a, Plan& r) {
  const int64_t nseq = a->nseq, most = ((int64_t)(a->seq_starts ? a->tokens : a->seqlen) + Q - 1) / Q;  // chunks of the longest prompt there can be
  const int64_t units = a->seq_starts ? (int64_t)a->tokens / Q + nseq : nseq * most;
  r.waves = a->vdim <= 64 ? 2 : 4;
  r.parts = (a->vdim + 32 * r.waves - 1) / (32 * r.waves);
  const int64_t parts = (int64_t)a->nheads * r.parts;
  // Tenths of a microsecond.  A chunk's step takes `one` where a compute unit has one workgroup and `full` where it has as many as fit
  // (`fit`), one of the states' 0.64 and 0.53 of it; every segment's state is taken to move three times at 2.6 TB/s (more where there are many;
  // those of prompts that are not cut do not), and the join and two more launches to come to 100.
  // Measured, heads of 128 by 128, by the chunks of a segment: 500 tokens of 16 heads, bf16, uncut 36 us, 2 chunks 27, one 26; 2 prompts of 8192, 32
  // heads, 32 chunks 233 us, 16 208, 8 226; 4 of 4096, 16 heads, 16 chunks 118, 12 125, 8 106; one of 16384, 8 heads, 16 chunks 108, 8 73; 10
  // packed prompts of 6949 tokens, the longest 2047, 16 heads, uncut 160, 12 chunks 116, 8 93, 6 85, 4 91, 3 94.
  struct Step { double one, full; int fit; };
  static constexpr Step steps[4][2] = {{{30, 50, 3}, {32, 42, 2}}, {{37, 59, 3}, {34, 51, 2}}, {{54, 60, 2}, {42, 72, 2}}, {{76, 76, 1}, {76, 76, 1}}};
  const Step s = steps[a->kdim <= 32 ? 0 : a->kdim <= 64 ? 1 : a->kdim <= 128 ? 2 : 3][r.waves == 4];
  auto step = [&](double wgs, double one, double full) {
    double left = std::max(wgs / 256, 1.0), t = 0;
    if (left > s.fit) t = std::floor(left / s.fit) * full, left -= std::floor(left / s.fit) * s.fit;
    if (left == 0) return t;
    if (!a->seq_starts) left = std::ceil(left);  // (prompts of many lengths: what ends early makes room)
    return t + one + (full - one) * (left <= 1 ? 0 : (left - 1) / (s.fit - 1));
  };
  // `longest`: chunks of the longest prompt, `segs` segments of which `ahead` have one behind them
  auto cost = [&](double longest, double n, double segs, double ahead) {
    if (n >= longest) return longest * step(segs * parts, s.one, s.full);
    return n * step(segs * parts, s.one, s.full) + n * step(ahead * parts, 0.64 * s.one, 0.53 * s.full) + (ahead + 2 * segs) * a->nheads * a->kdim * a->vdim * 4 / 2.6e5 + 100;
  };
  // Packed prompts' lengths are not known here.  They may be alike, or the longest two and a half times the mean, or one has nearly all the tokens;
  // taken is what loses least over the three, the second counted twice, each against what would be best for it.  us, taken, best and uncut:
  // the 10 prompts above 86, 85, 160; 10 of 695 72, 56, 56; one of 2000 among 60 single tokens 97, 87, 140; one of 4096 among 32, 32 heads, 200,
  // 150, 274; 64 of 200, 32 heads, 195, 157, 157; 4 of 30 to 700, 8 heads of 64 by 64, 20, 20, 47; 3000 and 200 tokens, 8 heads of 256 by 128, 56, 55, 300.
  const double mean = (double)units / nseq, rest = (double)nseq - 1;
  auto costs = [&](int64_t n, double (&c)[3]) {
    if (!a->seq_starts) {
      const double segs = (double)(nseq * ((most + n - 1) / n));
      c[0] = c[1] = c[2] = cost((double)most, (double)n, segs, segs - nseq);
    } else {
      const double alike = nseq * std::ceil(mean / n), some = std::max((double)units / n + 0.5 * nseq, (double)nseq), one = std::ceil((double)(units - nseq + 1) / n);
      c[0] = cost(mean, (double)n, alike, alike - nseq);
      c[1] = cost(std::min<double>((double)most, 2.5 * mean), (double)n, some, some - nseq);
      c[2] = cost((double)(units - nseq + 1), (double)n, one + rest, one - 1);
    }
  };
  double best[3] = {}, least = 0, c[3];
  r.seg_chunks = (int)most, r.cut = 0;
  for (int pass = 0; pass < 2; ++pass)
    for (int64_t n = most; n > 0; n = n > 16 ? n * 7 / 8 : n - 1) {  // (the whole first)
      costs(n, c);
      double loss = 0;
      for (int i = 0; i < 3; ++i) {
        if (pass == 0) best[i] = n == most ? c[i] : std::min(best[i], c[i]);
        else loss += (i == 1 ? 2 : 1) * c[i] / best[i];
      }
      if (pass == 1 && (n == most || loss < least)) least = loss, r.seg_chunks = (int)n, r.cut = n < most;
    }
  const int64_t per = (most + r.seg_chunks - 1) / r.seg_chunks;
  r.segs = a->seq_starts ? std::min<int64_t>(units / r.seg_chunks + nseq, units) : nseq * per;
  const int64_t w = (int64_t)Q * r.seg_chunks;
  r.blocks = a->seq_starts ? (a->tokens - 1) / w : nseq * (per - 1), r.longer = a->seq_starts ? std::min<int64_t>(nseq, a->tokens / (w + 1)) : nseq;
  r.places = a->seq_starts ? r.blocks + r.longer : r.segs;
  if (r.blocks == 0) r.cut = 0;
  if (!r.cut) r.segs = nseq;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  r.decays = r.cut ? up(r.places * a->nheads * a->kdim * a->vdim * 4) : 0;
  r.bytes = r.decays + (r.cut ? up(r.places * a->nheads * 4) : 0);
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
  if (a->state && (a->num_slots <= 0 || (a->num_slots > 1 && a->state_stride_s < (int64_t)a->nheads * a->kdim * a->vdim))) return LQ_ERR_SHAPE;  // (slots that overlap)
  for (const int64_t s : {a->q_stride_l, a->k_stride_l, a->v_stride_l, a->g_stride_l})
    if (s < 0 || s >= 1 << 24) return LQ_ERR_SHAPE;  // a chunk's rows are reached by 32-bit offsets
  for (const int64_t s : {a->q_stride_b, a->q_stride_l, a->q_stride_h, a->k_stride_b, a->k_stride_l, a->k_stride_h, a->v_stride_b, a->v_stride_l, a->v_stride_h})
    if (s % 8 != 0) return LQ_ERR_SHAPE;
  if (!sv_al(a->q, 16) || !sv_al(a->k, 16) || !sv_al(a->v, 16) || !sv_al(a->out, 16) || !sv_al(a->state, 16) || a->state_stride_s % 4 != 0 ||
      !sv_al(a->g, 4) || !sv_al(a->slots, 4) || !sv_al(a->seq_starts, 4))
    return LQ_ERR_SHAPE;
  Plan pl;
  if (!plan(a, pl) || a->workspace_bytes < pl.bytes || !sv_al(a->workspace, 256)) return LQ_ERR_SHAPE;
  if (pl.bytes && !a->workspace) return LQ_ERR_NULL;
  char* ws = (char*)a->workspace;
  // Weights and decays are exponentials of sums that the scale's logarithm is part of, and zero below 2^-126: a scale far from one is left out of them.
  const float size = std::fabs(a->scale);
  const int exponent = size > 0.0f && std::isfinite(size) ? std::ilogb(size) : 0;
  const float post = exponent < -40 || exponent > 40 ? std::ldexp(1.0f, std::max(exponent, -110)) : 1.0f;
  PromptParams p = {(const uint16_t*)a->q, a->q_stride_b, a->q_stride_l, a->q_stride_h, (const uint16_t*)a->k, a->k_stride_b, a->k_stride_l, a->k_stride_h,
                    (const uint16_t*)a->v, a->v_stride_b, a->v_stride_l, a->v_stride_h, a->g, a->g_stride_b, a->g_stride_l, a->g_stride_h,
                    !a->g || (a->g_stride_b == 0 && a->g_stride_l == 0), std::log2(size / post), post, a->scale < 0.0f, (uint16_t*)a->out, a->state, a->state_stride_s, a->slots, a->seq_starts,
                    a->num_slots, a->nseq, a->seqlen, a->tokens, a->nheads, a->kdim, a->vdim, pl.cut ? (float*)ws : nullptr,
                    pl.cut ? (float*)(ws + pl.decays) : nullptr, (int)pl.segs, pl.seg_chunks, pl.parts, (int)pl.blocks, (int)pl.places};
  auto grid_of = [&](int64_t segs) { return dim3((unsigned)((segs * a->nheads * pl.parts + 7) / 8 * 8)); };
  const dim3 grid = grid_of(pl.segs), ahead = grid_of(pl.blocks), threads(64 * pl.waves);
  const dim3 join((unsigned)pl.longer, (unsigned)a->nheads, (unsigned)(((int64_t)a->kdim * a->vdim + 1023) / 1024));
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
