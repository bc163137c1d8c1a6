// lq_copy_slots: slots of state tensors copied, exchanged or cleared in place, all tensors of all layers in one launch.
//   new[dst[i]] = old[src[i]], zeros where src[i] < 0, all bits one where it is beyond the slots
// HBM-bound: every entry's bytes read once and written once.
//
// A workgroup owns a strip of a tensor, some bytes of every slot, for all entries: it requests every entry's part of the strip into
// registers, waits until all of its waves have theirs, and stores.  So no source is overwritten before it is read, whatever the entries
// exchange, without a second buffer in memory, and no two workgroups touch the same bytes.  The more entries, the narrower a strip: 1024
// bytes up to 256 entries, 32 at 8192.
//
// 1 GiB of slots in another order (a copy of that size reaches 5.2 TB/s): 64 slots 5.1 TB/s, 256 4.9, 1024 4.8, 2048 4.5, 4096 3.9, 8192 2.7.
// One layer's state of 2 MB to 4 slots: 5.5 us (floor 3.2), most of it the launch and the list.
#include <algorithm>

#include "serve_common.h"

namespace {

constexpr int kWaves = 8, kMaxTensors = 64, kMaxEntries = 8192, kMaxU = 32;

struct Slots {
  char* base;
  int64_t stride, bytes;
  int64_t strips;  // of this tensor and the ones in front of it
};
struct CopyParams {
  Slots t[kMaxTensors];
  int num_tensors, num_slots;
  const int32_t* src;
  const int32_t* dst;
  int entries, lanes;  // lanes: of one entry's part of a strip, a power of two; a lane has one unit
  int beside;          // parts of a strip side by side, each with waves of its own: more than one where there are fewer entries than waves
  int near;            // strips that share 128 bytes on one die
  int log_table;       // of the places of the table of destinations
};

// of the unit that divides a tensor's address, stride and size: 16, 4, 2 or 1 bytes
LQ_DEV int unit_of(const Slots& t) {
  const uint64_t m = (uint64_t)(uintptr_t)t.base | (uint64_t)t.stride | (uint64_t)t.bytes;
  return m % 16 == 0 ? 16 : (m % 4 == 0 ? 4 : (m % 2 == 0 ? 2 : 1));
}
LQ_DEV lq_v4i load_unit(const char* at, int unit) {
  lq_v4i v = {0, 0, 0, 0};
  if (unit == 16) v = *(const lq_v4i*)at;
  else if (unit == 4) v[0] = *(const int*)at;
  else if (unit == 2) v[0] = *(const uint16_t*)at;
  else v[0] = *(const uint8_t*)at;
  return v;
}
LQ_DEV void store_unit(char* at, int unit, lq_v4i v) {
  if (unit == 16) *(lq_v4i*)at = v;
  else if (unit == 4) *(int*)at = v[0];
  else if (unit == 2) *(uint16_t*)at = (uint16_t)v[0];
  else *(uint8_t*)at = (uint8_t)v[0];
}

enum { kOpen = -3, kSkip = -2, kClear = -1 };  // what an entry's source says besides a slot; num_slots: filled with ones

template <int U>
__global__ __launch_bounds__(64 * kWaves) void copy_slots_kernel(CopyParams p) {
  extern __shared__ int list[];  // [entries] sources, [entries] destinations, [1 << log_table] table
  int *from = list, *to = list + p.entries, *table = to + p.entries;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = p.entries, places = 1 << p.log_table;
  if (n <= 64) {  // (the first wave by itself: 4 forks of 2 MB 6.7 us, by the table 8.1; with all waves at work 5.5)
    if (tid < n) {
      const int d = p.dst[tid], s = p.src[tid] < 0 ? (int)kClear : min(p.src[tid], p.num_slots);
      bool keep = d >= 0 && d < p.num_slots && d != s;
      for (int j = 1; j < n; ++j) keep &= tid >= j || __builtin_amdgcn_readlane(d, j) != d;
      to[tid] = d, from[tid] = keep ? s : (int)kSkip;
    }
    __syncthreads();
  } else {
    for (int i = tid; i < n; i += 64 * kWaves) {
      const int d = p.dst[i];
      to[i] = d, from[i] = d < 0 || d >= p.num_slots ? (int)kSkip : (int)kOpen;
    }
    // The last entry of a destination counts.  Each entry leaves its index at a place that its destination names, the largest stays; who finds
    // another destination's there tries again with other places.  (The last entry of those that do is always through.)
    auto place = [&](int d, int round) { return round == 0 ? d & (places - 1) : (int)(((uint32_t)d * (0x9e3779b1u + 2u * round)) >> (32 - p.log_table)); };
    for (int round = 0;; ++round) {
      for (int i = tid; i < places; i += 64 * kWaves) table[i] = -1;
      __syncthreads();
      for (int i = tid; i < n; i += 64 * kWaves)
        if (from[i] == kOpen) atomicMax(&table[place(to[i], round)], i);
      __syncthreads();
      bool open = false;
      for (int i = tid; i < n; i += 64 * kWaves) {
        if (from[i] != kOpen) continue;
        const int last = table[place(to[i], round)];
        if (last == i) {
          const int s = p.src[i] < 0 ? (int)kClear : min(p.src[i], p.num_slots);
          from[i] = s == to[i] ? (int)kSkip : s;
        } else if (to[last] == to[i]) {
          from[i] = kSkip;
        } else {
          open = true;
        }
      }
      if (!__syncthreads_or(open)) break;
    }
  }
  const int per = 64 / p.lanes, waves = kWaves / p.beside, part = wave / waves * p.lanes + lane % p.lanes;
  const int e0 = wave % waves * per + lane / p.lanes;  // entries e0, e0 + waves per, ..
  const int64_t all = p.t[p.num_tensors - 1].strips;
  const int64_t eighth = (all + 7) / 8;
  for (int64_t i = blockIdx.x; i < (p.near ? 8 * eighth : all); i += gridDim.x) {
    const int64_t strip = p.near ? i % 8 * eighth + i / 8 : i;
    if (strip >= all) continue;
    int t = 0;
    while (strip >= p.t[t].strips) ++t;
    const Slots& x = p.t[t];
    const int unit = unit_of(x);
    const int64_t at = ((strip - (t ? p.t[t - 1].strips : 0)) * (p.lanes * p.beside) + part) * unit;
    const bool in = at < x.bytes;
    lq_v4i v[U];
    int f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * waves * per;
      f[u] = in && e < n ? from[e] : (int)kSkip;
      const int fill = f[u] >= p.num_slots ? -1 : 0;
      v[u] = lq_v4i{fill, fill, fill, fill};
      if (f[u] >= 0 && f[u] < p.num_slots) v[u] = load_unit(x.base + f[u] * x.stride + at, unit);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every source of the strip is read
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (f[u] != kSkip) store_unit(x.base + to[e0 + u * waves * per] * x.stride + at, unit, v[u]);
  }
}

}  // namespace

extern "C" int lq_copy_slots(const lq_copy_slots_args* a, hipStream_t stream) {
  if (!a || !a->tensors || !a->src || !a->dst) return LQ_ERR_NULL;
  if (a->num_tensors <= 0 || a->num_slots <= 0 || a->entries <= 0 || a->entries > kMaxEntries) return LQ_ERR_SHAPE;
  if (!sv_al(a->src, 4) || !sv_al(a->dst, 4)) return LQ_ERR_SHAPE;
  for (int i = 0; i < a->num_tensors; ++i) {
    if (!a->tensors[3 * i]) return LQ_ERR_NULL;
    if (a->tensors[3 * i + 2] <= 0 || (a->num_slots > 1 && a->tensors[3 * i + 1] < a->tensors[3 * i + 2])) return LQ_ERR_SHAPE;
  }
  // as many lanes to an entry's part as leave every entry a place in the workgroup's registers
  int lanes = 64;
  while (lanes > 1 && (int64_t)kWaves * (64 / lanes) * kMaxU < a->entries) lanes /= 2;
  int beside = 1;
  while (2 * beside * a->entries <= kWaves) beside *= 2;
  const int64_t slots = (int64_t)kWaves / beside * (64 / lanes);
  const int u = (int)((a->entries + slots - 1) / slots);
  // Workgroups go to the 8 dies in turn.  Strips of 128 bytes and less are given out so that those which share a cache line, or are next to
  // each other, meet in one die's cache: 1 GiB of 8192 slots in 0.78 ms, 1.41 without; of 4096 0.55, 0.67.  Wider ones gain nothing by it.
  const bool near = lanes <= 8;
  int log_table = 6;
  while (1 << log_table < a->entries) ++log_table;
  for (int first = 0; first < a->num_tensors; first += kMaxTensors) {
    CopyParams p = {};
    p.num_tensors = std::min(kMaxTensors, a->num_tensors - first), p.num_slots = a->num_slots, p.src = a->src, p.dst = a->dst, p.entries = a->entries, p.lanes = lanes, p.beside = beside, p.log_table = log_table, p.near = near;
    int64_t strips = 0;
    for (int i = 0; i < p.num_tensors; ++i) {
      const int64_t* t = a->tensors + 3 * (first + i);
      const uint64_t m = (uint64_t)t[0] | (uint64_t)t[1] | (uint64_t)t[2];
      const int64_t width = (int64_t)lanes * beside * (m % 16 == 0 ? 16 : (m % 4 == 0 ? 4 : (m % 2 == 0 ? 2 : 1)));
      strips += (t[2] + width - 1) / width;
      p.t[i] = {(char*)t[0], t[1], t[2], strips};
    }
    const dim3 grid((unsigned)std::min<int64_t>(strips, near ? 1024 : 4096)), threads(64 * kWaves);
    const size_t lds = (size_t)a->entries * 8 + (a->entries > 64 ? (size_t)4 << log_table : 0);
    auto go = [&](auto k) {
      auto* kernel = copy_slots_kernel<decltype(k)::value>;
      hipLaunchKernelGGL(kernel, grid, threads, lds, stream, p);
      return lq_check_launch();
    };
    using std::integral_constant;
    const int rc = u <= 1 ? go(integral_constant<int, 1>{}) : u <= 2 ? go(integral_constant<int, 2>{}) : u <= 4 ? go(integral_constant<int, 4>{}) :
                   u <= 8 ? go(integral_constant<int, 8>{}) : u <= 16 ? go(integral_constant<int, 16>{}) : go(integral_constant<int, 32>{});
    if (rc != LQ_OK) return rc;
  }
  return LQ_OK;
}
