// Eviction from a paged key-value cache by accumulated attention weight.
//
// Per sequence of more than `keep` slots and per key head: the slots of the
// first `sink` positions and of the last `recent` ones stay, then those of the
// largest weight, equal ones by the lower slot, `keep` in all. The sequence then
// ends at slot E behind its keep-th slot: the i-th slot below E that goes takes
// over the i-th slot at or beyond E that stays, in slot order; slots below E
// that stay are not touched, so only the rows that move are read and written. A
// slot from which a row moves is at or beyond E and one to which it moves
// below: the copies need no order. Slots of missing pages are no slots here:
// they neither count nor move, and E is `keep` where there are none.
//
// Selection is one workgroup per sequence and head: a radix search for the
// keep-th largest key, 8 bits at a time with a histogram in LDS, then counts and
// ranks in slot order: 29 us for 64 heads of 20000-32760 slots, bound by the
// vector instructions of one CU per head (52 us a slot per lane and ranks among
// equals always; 94 us with keys in memory). Copies are a second launch over all
// moved rows, bound by memory: 87 us for 418 MB in and out, 4.8 TB/s.
#include "kv_cache.h"
#include "lanes.h"

namespace dmad {

constexpr int kSelectWaves = 16;
constexpr int kSelectThreads = 64 * kSelectWaves;
constexpr int kSelectRow = 4 * 64;  // slots a wave takes at a time, 4 neighbours per lane
// Copies of the histogram, by lane: lanes that count one digit meet in a copy
// four at a time, not 64.
constexpr int kHistCopies = 16;

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

// Order of weights as unsigned keys: 1 .. 0xfffffffe, NaN above all of them;
// 0xffffffff stays unconditionally and 0 is a slot that is not there.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 as +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// SLOTS > 0: keys stay in LDS (sequences of up to SLOTS slots); 0: in memory.
// LOADS: rows whose weights and positions a wave has on their way together.
template <int SLOTS, int LOADS>
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(KvEvictParams p) {
  static_assert(SLOTS % (kSelectRow * kSelectWaves) == 0, "whole rows for every wave");
  __shared__ __attribute__((aligned(16))) uint32_t lds_keys[SLOTS > 0 ? SLOTS : 4];
  __shared__ uint32_t hist[256 * kHistCopies];
  __shared__ uint32_t total[256];
  __shared__ uint32_t found[3];
  __shared__ int before_held[kSelectWaves], before_eq[kSelectWaves], before_hole[kSelectWaves], before_move[kSelectWaves];
  __shared__ int behind;
  const KvPages& kv = p.kv;
  const int h = (int)blockIdx.x % kv.heads, b = (int)blockIdx.x / kv.heads;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = kv.length(b);
  // nothing goes: a uniform decision of the workgroup
  auto leave_as_it_is = [&] {
    if (threadIdx.x == 0) p.counts[blockIdx.x] = 0;
    if (threadIdx.x == 0 && h == 0) p.ends[b] = n;
  };
  if (n <= p.keep) return leave_as_it_is();
  // Each wave has a range of whole rows, so that ranks in slot order need only
  // its running counts; a lane reads back only the keys it wrote. Slots of
  // missing pages and those from n on to the end of a row have key 0: with more
  // than keep other slots they are never among the ones that stay.
  const int span = (n + kSelectRow * kSelectWaves - 1) / (kSelectRow * kSelectWaves) * kSelectRow;
  const int begin = min(n, wave * span), end = min(n, begin + span);
  uint32_t* keys = SLOTS > 0 ? lds_keys : p.keys + (int64_t)blockIdx.x * kv.capacity();
  const int seen = kv.seen[b], oldest = seen < INT32_MIN + p.recent ? INT32_MIN : seen - p.recent;

  int held = 0;  // slots of this lane that a page holds
  for (int row = begin; row < end; row += kSelectRow * LOADS) {
    KvSlot at[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int s = row + kSelectRow * j + 4 * lane;
      at[j] = KvSlot{-1, 0};
      if (s < end) at[j] = kv.locate(b, s);  // 4 slots from a multiple of 4 lie on one page
    }
    f32x4_t w[LOADS];
    i32x4_t position[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      if (at[j].page < 0) continue;
      const int64_t i = kv.index(at[j], h);
      w[j] = *(const f32x4_t*)(kv.weight + i);
      position[j] = *(const i32x4_t*)(kv.position + i);
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      if (row + kSelectRow * j >= end) continue;
      const int s = row + kSelectRow * j + 4 * lane;
      u32x4_t key;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        key[e] = 0u;
        if (at[j].page >= 0 && s + e < n) {
          key[e] = position[j][e] < p.sink || position[j][e] >= oldest ? 0xffffffffu : weight_key(w[j][e]);
          ++held;
        }
      }
      if (SLOTS > 0 || s < n) *(u32x4_t*)(keys + s) = key;
    }
  }
  // f(row, the lane's first slot of it, its 4 keys) for this wave's rows in order
  auto each = [&](auto f) {
    for (int row = begin; row < end; row += 4 * kSelectRow) {
      u32x4_t key[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = row + kSelectRow * j + 4 * lane;
        key[j] = u32x4_t{0, 0, 0, 0};
        if (row + kSelectRow * j < end && (SLOTS > 0 || s < n)) key[j] = *(const u32x4_t*)(keys + s);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row + kSelectRow * j < end) f(row + kSelectRow * j, row + kSelectRow * j + 4 * lane, key[j]);
    }
  };

#pragma unroll
  for (int m = 1; m < 64; m <<= 1) held += __shfl_xor(held, m);
  if (lane == 0) before_held[wave] = held;
  __syncthreads();
  int held0 = 0, held_all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    if (w < wave) held0 += before_held[w];
    held_all += before_held[w];
  }
  if (held_all <= p.keep) return leave_as_it_is();

  // the keep-th largest key, and how many of its equals stay
  uint32_t prefix = 0, mask = 0;
  uint32_t left = (uint32_t)p.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256 * kHistCopies; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    each([&](int, int, u32x4_t k) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((k[e] & mask) == prefix) atomicAdd(&hist[((k[e] >> shift) & 255) * kHistCopies + (lane & (kHistCopies - 1))], 1u);
    });
    __syncthreads();
    if (threadIdx.x < 256) {
      uint32_t t = 0;
#pragma unroll
      for (int c = 0; c < kHistCopies; ++c) t += hist[threadIdx.x * kHistCopies + ((c + threadIdx.x) & (kHistCopies - 1))];
      total[threadIdx.x] = t;
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // lane i: digits 255 - 4 i down to 252 - 4 i
      uint32_t d[4], sum = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += d[k] = total[255 - 4 * lane - k];
      uint32_t upto = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const uint32_t y = __shfl_up(upto, m);
        if (lane >= m) upto += y;
      }
      uint32_t above = upto - sum;
      if (above < left && left <= upto) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (above < left && left <= above + d[k]) {
            found[0] = 255 - 4 * lane - k;
            found[1] = left - above;
            found[2] = d[k];
          }
          above += d[k];
        }
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= 255u << shift;
    left = found[1];
  }
  const bool ties = left != found[2];  // only some of the equals stay: the first ones

  // what a row's 4 votes per lane come to below this lane, and in all
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  struct Votes {
    int before, all;
  };
  auto vote = [&](const bool (&x)[4]) {
    Votes v{0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t m = __ballot(x[e]);
      v.before += (int)__popcll(m & below);
      v.all += (int)__popcll(m);
    }
    return v;
  };
  // where the sequence ends afterwards: behind its keep-th slot
  int cut = p.keep;
  if (held_all != n) {
    if (held0 < p.keep && p.keep <= held0 + held) {  // in one wave's range
      int rank = held0;
      each([&](int, int s, u32x4_t k) {
        const bool here[4] = {k[0] != 0, k[1] != 0, k[2] != 0, k[3] != 0};
        const Votes v = vote(here);
        int r = rank + v.before;
        rank += v.all;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r += here[e];
          if (here[e] && r == p.keep) behind = s + e + 1;
        }
      });
    }
    __syncthreads();
    cut = behind;
  }
  if (threadIdx.x == 0 && h == 0) p.ends[b] = cut;

  int eq0 = 0;  // equals before this wave
  if (ties) {
    int count = 0;
    each([&](int, int, u32x4_t k) {
      const bool equal[4] = {k[0] == prefix, k[1] == prefix, k[2] == prefix, k[3] == prefix};
      count += vote(equal).all;
    });
    if (lane == 0) before_eq[wave] = count;
    __syncthreads();
    for (int w = 0; w < wave; ++w) eq0 += before_eq[w];
  }
  // which of a lane's 4 slots stay; eq runs over the equals
  auto stays = [&](u32x4_t k, int& eq, bool (&st)[4]) {
    if (!ties) {
#pragma unroll
      for (int e = 0; e < 4; ++e) st[e] = k[e] >= prefix;
      return;
    }
    const bool equal[4] = {k[0] == prefix, k[1] == prefix, k[2] == prefix, k[3] == prefix};
    const Votes v = vote(equal);
    int rank = eq + v.before;
    eq += v.all;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      st[e] = k[e] > prefix || (equal[e] && (uint32_t)rank < left);
      rank += equal[e];
    }
  };
  // which of them change: slots below the cut that go, or beyond that stay
  auto changes = [&](int s, u32x4_t k, const bool (&st)[4], bool hole, bool (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = hole ? s + e < cut && k[e] != 0 && !st[e] : s + e >= cut && st[e];
  };
  int holes = 0, moves = 0, eq = eq0;
  each([&](int row, int s, u32x4_t k) {
    bool st[4], x[4];
    stays(k, eq, st);
    if (row < cut) {
      changes(s, k, st, true, x);
      holes += vote(x).all;
    }
    if (row + kSelectRow > cut) {
      changes(s, k, st, false, x);
      moves += vote(x).all;
    }
  });
  if (lane == 0) {
    before_hole[wave] = holes;
    before_move[wave] = moves;
  }
  __syncthreads();
  int hole0 = 0, move0 = 0;
  for (int w = 0; w < wave; ++w) {
    hole0 += before_hole[w];
    move0 += before_move[w];
  }
  int32_t* to = p.moves + (int64_t)blockIdx.x * 2 * p.max_moves;
  int32_t* from = to + p.max_moves;
  auto list = [&](int32_t* out, int& base, int s, const bool (&x)[4]) {
    const Votes v = vote(x);
    int at = base + v.before;
    base += v.all;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // as many slots move as go below the cut: at most keep, and at most those beyond it
      if (x[e] && at < p.max_moves) out[at] = s + e;
      at += x[e];
    }
  };
  eq = eq0;
  each([&](int row, int s, u32x4_t k) {
    bool st[4], x[4];
    stays(k, eq, st);
    if (row < cut) {
      changes(s, k, st, true, x);
      list(to, hole0, s, x);
    }
    if (row + kSelectRow > cut) {
      changes(s, k, st, false, x);
      list(from, move0, s, x);
    }
  });
  if (threadIdx.x == kSelectThreads - 1) p.counts[blockIdx.x] = min(move0, p.max_moves);
}

// A row per D/8 lanes, K and V together.
template <int D>
__global__ __launch_bounds__(256) void kv_move_kernel(KvEvictParams p) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const KvPages& kv = p.kv;
  const int h = (int)blockIdx.y, b = (int)blockIdx.z;
  const int64_t bh = (int64_t)b * kv.heads + h;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) kv.lengths[b] = p.ends[b];
  const int el = ((int)threadIdx.x % LANES) * 8, count = p.counts[bh];
  uint16_t *kp = (uint16_t*)kv.k + el, *vp = (uint16_t*)kv.v + el;
  for (int i = (int)blockIdx.x * ROWS + (int)threadIdx.x / LANES; i < count; i += (int)gridDim.x * ROWS) {
    const KvSlot to = kv.locate(b, p.moves[bh * 2 * p.max_moves + i]);
    const KvSlot from = kv.locate(b, p.moves[(bh * 2 + 1) * p.max_moves + i]);
    if (to.page < 0 || from.page < 0) continue;
    const i32x4_t k = *(const i32x4_t*)(kp + kv.k_offset(from, h)), v = *(const i32x4_t*)(vp + kv.v_offset(from, h));
    *(i32x4_t*)(kp + kv.k_offset(to, h)) = k;
    *(i32x4_t*)(vp + kv.v_offset(to, h)) = v;
    if (el == 0) {
      const int64_t a = kv.index(to, h), f = kv.index(from, h);
      kv.weight[a] = kv.weight[f];
      kv.position[a] = kv.position[f];
    }
  }
}

// Workgroups of all heads and sequences together: two rounds of what the chip
// holds, each going through its head's rows. How many move is known on the
// device only, and a workgroup for every row that the capacity allows costs a
// cache that is cut by little or nothing: 16 x 8 heads of 131072 slots, keep
// 65536: 121 us with none over, 183 with one, against 18 and 75. Many rows do not
// mind (evict_half 130 us against 126; 128 with 2048 and 8192 workgroups).
constexpr int kMoveGroups = 4096;

template <int D>
static hipError_t move_launch(const KvEvictParams& p, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  const int groups = max(1, min((p.max_moves + ROWS - 1) / ROWS, kMoveGroups / (p.kv.heads * p.kv.B)));
  hipLaunchKernelGGL((kv_move_kernel<D>), dim3((unsigned)groups, (unsigned)p.kv.heads, (unsigned)p.kv.B), dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_kv_evict(const KvEvictParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.kv.B * p.kv.heads)), block(kSelectThreads);
  const int slots = p.kv.M * p.kv.P;
  if (slots <= kSelectInLds / 8) hipLaunchKernelGGL((kv_select_kernel<kSelectInLds / 8, 1>), grid, block, 0, s, p);
  else if (slots <= kSelectInLds) hipLaunchKernelGGL((kv_select_kernel<kSelectInLds, 4>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv_select_kernel<0, 4>), grid, block, 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  switch (p.D) {
    case 16: return move_launch<16>(p, s);
    case 32: return move_launch<32>(p, s);
    case 64: return move_launch<64>(p, s);
    case 128: return move_launch<128>(p, s);
    case 256: return move_launch<256>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace dmad
