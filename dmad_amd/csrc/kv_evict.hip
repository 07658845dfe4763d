// Eviction from a paged key-value cache by accumulated attention weight.
//
// Per sequence of more than `keep` slots and per key head: the slots of the
// first `sink` positions and of the last `recent` ones stay, then those of the
// largest weight, equal ones by the lower slot, `keep` in all. The i-th slot
// below `keep` that goes takes over the i-th slot at or beyond `keep` that
// stays, in slot order; slots below `keep` that stay are not touched, so only
// the rows that move are read and written. A slot from which a row moves is at
// or beyond `keep` and one to which it moves below: the copies need no order.
//
// Selection is one workgroup per sequence and head: a radix search for the
// keep-th largest key, 8 bits at a time with a histogram in LDS, then counts and
// ranks in slot order. Copies are a second launch over all moved rows.
#include "kv_cache.h"
#include "lanes.h"

namespace dmad {

constexpr int kSelectWaves = 16;
constexpr int kSelectThreads = 64 * kSelectWaves;
constexpr int kSelectBatch = 4;  // keys a lane reads together

// Copies of the histogram, by lane: lanes that count one digit meet in a copy
// four at a time, not 64.
constexpr int kHistCopies = 16;

// Order of weights as unsigned keys: 1 .. 0xfffffffe, NaN above all of them;
// 0xffffffff stays unconditionally and 0 goes first.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 as +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// SLOTS > 0: keys stay in LDS (sequences of up to SLOTS slots); 0: in memory.
template <int SLOTS>
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(KvEvictParams p) {
  __shared__ uint32_t lds_keys[SLOTS > 0 ? SLOTS : 1];
  __shared__ uint32_t hist[256 * kHistCopies];
  __shared__ uint32_t total[256];
  __shared__ uint32_t found[2];
  __shared__ int before_eq[kSelectWaves], before_hole[kSelectWaves], before_move[kSelectWaves];
  const KvPages& kv = p.kv;
  const int h = (int)blockIdx.x % kv.heads, b = (int)blockIdx.x / kv.heads;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = kv.length(b);
  if (n <= p.keep) {
    if (threadIdx.x == 0) p.counts[blockIdx.x] = 0;
    return;
  }
  // each wave has a range of slots, so that ranks in slot order need only its running counts
  const int span = ((n + kSelectThreads - 1) / kSelectThreads) * 64;
  const int begin = min(n, wave * span), end = min(n, begin + span);
  uint32_t* keys = SLOTS > 0 ? lds_keys : p.keys + (int64_t)blockIdx.x * kv.capacity();
  const int oldest = kv.seen[b] - p.recent;

  // Keys from weights and positions, LOADS slots of a lane under way together
  // (the page ids, then what is there); a lane reads back only its own.
  constexpr int LOADS = SLOTS == kSelectInLds / 8 ? 4 : 16;
  for (int s0 = begin; s0 < end; s0 += 64 * LOADS) {
    KvSlot at[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int s = s0 + 64 * j + lane;
      at[j] = KvSlot{-1, 0};
      if (s < end) at[j] = kv.locate(b, s);
    }
    float w[LOADS];
    int position[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      if (at[j].page < 0) continue;
      w[j] = kv.weight[kv.index(at[j], h)];
      position[j] = kv.position[kv.index(at[j], h)];
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int s = s0 + 64 * j + lane;
      // slots of a missing page: none moves, none is moved to
      uint32_t key = s < p.keep ? 0xffffffffu : 0u;
      if (at[j].page >= 0) key = position[j] < p.sink || position[j] >= oldest ? 0xffffffffu : weight_key(w[j]);
      if (s < end) keys[s] = key;
    }
  }
  // f(slot, its key, whether there is one) for this wave's slots, 64 at a time in order
  auto each = [&](auto f) {
    for (int s0 = begin; s0 < end; s0 += 64 * kSelectBatch) {
      uint32_t key[kSelectBatch];
#pragma unroll
      for (int j = 0; j < kSelectBatch; ++j) {
        const int s = s0 + 64 * j + lane;
        key[j] = s < end ? keys[s] : 0u;
      }
#pragma unroll
      for (int j = 0; j < kSelectBatch; ++j)
        if (s0 + 64 * j < end) f(s0 + 64 * j + lane, key[j], s0 + 64 * j + lane < end);  // the test is the wave's
    }
  };

  // the keep-th largest key, and how many of its equals stay
  uint32_t prefix = 0, mask = 0;
  uint32_t left = (uint32_t)p.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256 * kHistCopies; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    each([&](int, uint32_t k, bool there) {
      if (there && (k & mask) == prefix) atomicAdd(&hist[((k >> shift) & 255) * kHistCopies + (lane & (kHistCopies - 1))], 1u);
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

  // equals before each wave
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  int count = 0;
  each([&](int, uint32_t k, bool there) { count += (int)__popcll(__ballot(there && k == prefix)); });
  if (lane == 0) before_eq[wave] = count;
  __syncthreads();
  int eq0 = 0;
  for (int w = 0; w < wave; ++w) eq0 += before_eq[w];

  // whether a slot stays; eq runs over the equals
  auto stays = [&](uint32_t k, bool there, int& eq) {
    const bool equal = there && k == prefix;
    const uint64_t votes = __ballot(equal);
    const int rank = eq + (int)__popcll(votes & below);
    eq += (int)__popcll(votes);
    return there && (k > prefix || (equal && (uint32_t)rank < left));
  };
  int holes = 0, moves = 0, eq = eq0;
  each([&](int s, uint32_t k, bool there) {
    const bool st = stays(k, there, eq);
    holes += (int)__popcll(__ballot(s < p.keep && there && !st));
    moves += (int)__popcll(__ballot(s >= p.keep && st));
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
  eq = eq0;
  each([&](int s, uint32_t k, bool there) {
    const bool st = stays(k, there, eq);
    const bool hole = s < p.keep && there && !st, move = s >= p.keep && st;
    const uint64_t hv = __ballot(hole), mv = __ballot(move);
    // as many slots move as go below keep: min(keep, n - keep) at most
    const int hi = hole0 + (int)__popcll(hv & below), mi = move0 + (int)__popcll(mv & below);
    if (hole && hi < p.max_moves) to[hi] = s;
    if (move && mi < p.max_moves) from[mi] = s;
    hole0 += (int)__popcll(hv);
    move0 += (int)__popcll(mv);
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
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) kv.lengths[b] = min(kv.length(b), p.keep);
  const int i = (int)blockIdx.x * ROWS + (int)threadIdx.x / LANES, el = ((int)threadIdx.x % LANES) * 8;
  if (i >= p.counts[bh]) return;
  const KvSlot to = kv.locate(b, p.moves[bh * 2 * p.max_moves + i]);
  const KvSlot from = kv.locate(b, p.moves[(bh * 2 + 1) * p.max_moves + i]);
  if (to.page < 0 || from.page < 0) return;
  uint16_t *kp = (uint16_t*)kv.k + el, *vp = (uint16_t*)kv.v + el;
  const i32x4_t k = *(const i32x4_t*)(kp + kv.k_offset(from, h)), v = *(const i32x4_t*)(vp + kv.v_offset(from, h));
  *(i32x4_t*)(kp + kv.k_offset(to, h)) = k;
  *(i32x4_t*)(vp + kv.v_offset(to, h)) = v;
  if (el == 0) {
    const int64_t a = kv.index(to, h), f = kv.index(from, h);
    kv.weight[a] = kv.weight[f];
    kv.position[a] = kv.position[f];
  }
}

template <int D>
static hipError_t move_launch(const KvEvictParams& p, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  hipLaunchKernelGGL((kv_move_kernel<D>), dim3((unsigned)((p.max_moves + ROWS - 1) / ROWS), (unsigned)p.kv.heads, (unsigned)p.kv.B),
                     dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_kv_evict(const KvEvictParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.kv.B * p.kv.heads)), block(kSelectThreads);
  const int slots = p.kv.M * p.kv.P;
  if (slots <= kSelectInLds / 8) hipLaunchKernelGGL((kv_select_kernel<kSelectInLds / 8>), grid, block, 0, s, p);
  else if (slots <= kSelectInLds) hipLaunchKernelGGL((kv_select_kernel<kSelectInLds>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv_select_kernel<0>), grid, block, 0, s, p);
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
