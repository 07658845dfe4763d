// Rotations of queries and keys by their positions, and of their tangents or
// gradients. With angle = position * frequency_i, c = m cos, s = m sin:
//   (a, b) -> (a c - b s, b c + a s)
// over pairs (a, b) of elements 2i, 2i + 1 (interleaved) or i, i + R/2 (halves) of
// the first R of a head's D elements; the others are copied. m is one factor for
// all (stretched frequencies come with one). Backwards the same by -angle.
//
// Far positions have angles of many turns: position times frequency is taken in
// 64 bits, reduced to a part of a turn there, and only that part is rounded to
// float32 (position 131072 in float32 would be off by 0.008 radians).
//
// Bound by its bytes: 4 D per row of 16 bits, in and out; 40 + 40 heads of 128 over 32760
// tokens with tangents take 455 us (2.7 GB, 5.9 TB/s). A workgroup takes a tile of
// tokens: its threads first compute the tile's sines and cosines into LDS, each
// once for all heads and both operands, then walk over units of two 16-byte
// accesses: both halves of 8 pairs, 8 pairs of neighbours, or 16 elements to
// copy. Smaller accesses where sizes or strides ask for them.
#include "block_ops.h"
#include "lanes.h"

namespace dmad {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryLdsPairs = 4096;  // sines and cosines of a tile: 32 KiB
constexpr int kRotaryMaxTile = 64;

// A float32 result to its element. The compiler makes one instruction with one rounding of
// some of the products and conversions to fp16 and two of others, which ones by the kernel's
// form: about one element in 4000 then depended on whether there are tangents and on the
// alignment. The empty asm keeps the two apart: float32, then fp16, for every element.
template <typename T>
__device__ __forceinline__ T rotary_round(float x) {
  if constexpr (__is_same(T, _Float16)) asm("" : "+v"(x));
  return (T)x;
}

// V consecutive elements, in one access of up to 16 bytes.
template <typename T, int V>
struct Piece {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  vec_t v;
  template <bool NT>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (NT) v = __builtin_nontemporal_load((const vec_t*)p);
    else v = *(const vec_t*)p;
  }
  template <bool NT>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (NT) __builtin_nontemporal_store(v, (vec_t*)p);
    else *(vec_t*)p = v;
  }
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
  __device__ __forceinline__ void set(int i, float x) { v[i] = rotary_round<T>(x); }
};
template <typename T>
struct Piece<T, 1> {
  T v;
  template <bool>
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  template <bool>
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ float get(int) const { return (float)v; }
  __device__ __forceinline__ void set(int, float x) { v = rotary_round<T>(x); }
};

// x / d by d's multiplier, of which 1 has none.
__device__ __forceinline__ int rotary_div(int x, uint32_t mul) { return mul == 0 ? x : (int)__umulhi((uint32_t)x, mul); }

// One unit of a row: its two pieces turned. Halves: one is the other's partner, with the
// V angles at c and s. Neighbours: V / 2 pairs in each, with the angles at c, s and half
// the table further on (V = 1: the pieces are one pair).
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void rotary_turn(Piece<T, V>& u, Piece<T, V>& w, const float* c, const float* s, int far) {
  if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float a = u.get(2 * i), b = u.get(2 * i + 1), d = w.get(2 * i), e = w.get(2 * i + 1);
      u.set(2 * i, fmaf(a, c[i], -(b * s[i])));
      u.set(2 * i + 1, fmaf(b, c[i], a * s[i]));
      w.set(2 * i, fmaf(d, c[far + i], -(e * s[far + i])));
      w.set(2 * i + 1, fmaf(e, c[far + i], d * s[far + i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = u.get(i), b = w.get(i);
      u.set(i, fmaf(a, c[i], -(b * s[i])));
      w.set(i, fmaf(b, c[i], a * s[i]));
    }
  }
}

template <typename T, int V, bool INTERLEAVED, bool JVP, bool NT>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryParams p) {
  __shared__ __attribute__((aligned(16))) float cs[kRotaryLdsPairs], sn[kRotaryLdsPairs];
  __shared__ int tok_b[kRotaryMaxTile], tok_s[kRotaryMaxTile];
  const int64_t token0 = (int64_t)blockIdx.x * p.tile;
  const int tokens = (int)min((int64_t)p.tile, p.tokens - token0), pairs = p.R >> 1;
  if ((int)threadIdx.x < tokens) {
    const int64_t t = token0 + threadIdx.x;
    tok_b[threadIdx.x] = (int)(t / p.S);
    tok_s[threadIdx.x] = (int)(t % p.S);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * pairs; i += kRotaryThreads) {
    const int k = i / pairs, f = i - k * pairs;
    const int64_t at = tok_b[k] * p.pos_b + tok_s[k] * p.pos_s;
    const int64_t pos = p.pos64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
    double turns = (double)pos * p.frequencies[f] * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[i] = c * p.factor;
    sn[i] = s * p.factor * (float)p.sign;
  }
  __syncthreads();
  const int units = tokens * p.per_token, turned = pairs / V;
  for (int i = threadIdx.x; i < units; i += kRotaryThreads) {
    const int k = rotary_div(i, p.token_mul), in_token = i - k * p.per_token;
    int h = rotary_div(in_token, p.head_mul);
    const int unit = in_token - h * p.per_head;
    const RotaryOperand& o = p.op[h >= p.op[0].H];
    if (h >= p.op[0].H) h -= p.op[0].H;
    const int b = tok_b[k], s = tok_s[k];
    const int64_t in = b * o.xb + s * o.xs + h * o.xh;
    const int64_t tin = b * o.tb + s * o.ts + h * o.th;
    const int64_t out = (((int64_t)b * p.S + s) * o.H + h) * p.D;
    const bool turns = unit < turned;
    int first, second;  // elements of the two pieces
    if (turns) {
      // neighbours too in pieces half the turned part apart: the lanes' accesses are contiguous
      constexpr bool PAIR = INTERLEAVED && V == 1;
      first = PAIR ? 2 * unit : V * unit;
      second = PAIR ? first + 1 : first + pairs;
    } else {
      first = p.R + 2 * V * (unit - turned);
      second = first + V;
    }
    const bool two = second < p.D;
    Piece<T, V> u, w, tu, tw;
    u.template load<NT>((const T*)o.x + in + first);
    if (two) w.template load<NT>((const T*)o.x + in + second);
    if constexpr (JVP) {
      tu.template load<NT>((const T*)o.t + tin + first);
      if (two) tw.template load<NT>((const T*)o.t + tin + second);
    }
    if (turns) {
      const int at = k * pairs + (INTERLEAVED && V > 1 ? V / 2 : V) * unit;
      rotary_turn<T, V, INTERLEAVED>(u, w, cs + at, sn + at, pairs / 2);
      if constexpr (JVP) rotary_turn<T, V, INTERLEAVED>(tu, tw, cs + at, sn + at, pairs / 2);
    }
    u.template store<NT>((T*)o.out + out + first);
    if (two) w.template store<NT>((T*)o.out + out + second);
    if constexpr (JVP) {
      tu.template store<NT>((T*)o.tout + out + first);
      if (two) tw.template store<NT>((T*)o.tout + out + second);
    }
  }
}

// Units that a workgroup aims at, and workgroups that fill the chip. A tile's angles are
// shared by its threads alone, and its loads start only behind them: at [1, 32760, 40, 128]
// with tangents 256 and 512 units take 455 us, 1024 489.
constexpr int kRotaryUnits = 512, kRotaryFill = 1024;

bool rotary_plan(RotaryParams& p, int elem_size, int align) {
  const int heads = p.op[0].H + p.op[1].H, pairs = p.R / 2, rest = p.D - p.R;
  int v = 16 / elem_size;
  while (v > 1 && (pairs % v != 0 || rest % v != 0 || p.D % v != 0 || align % v != 0)) v >>= 1;
  p.vec = v;
  p.per_head = pairs / v + (rest + 2 * v - 1) / (2 * v);
  const int64_t per_token = (int64_t)heads * p.per_head;
  int64_t tile = (kRotaryUnits + per_token - 1) / per_token;
  const int64_t fill = (p.tokens + kRotaryFill - 1) / kRotaryFill;
  if (tile > fill) tile = fill;
  if (tile > kRotaryMaxTile) tile = kRotaryMaxTile;
  if (pairs > 0 && tile > kRotaryLdsPairs / pairs) tile = kRotaryLdsPairs / pairs;
  if (tile < 1) tile = 1;
  if (pairs > kRotaryLdsPairs || per_token >= (1 << 20)) return false;
  p.per_token = (int)per_token;
  p.tile = (int)tile;
  // m = ceil(2^32 / d) is off by e = m d - 2^32 < d parts of d: x m >> 32 = x / d while x e < 2^32
  auto mul = [&](int64_t d, uint32_t& m) {
    const int64_t q = (((int64_t)1 << 32) + d - 1) / d, e = q * d - ((int64_t)1 << 32);
    m = d == 1 ? 0u : (uint32_t)q;
    return per_token * tile * e < ((int64_t)1 << 32);
  };
  if (!mul(p.per_head, p.head_mul) || !mul(per_token, p.token_mul)) return false;
  return (p.tokens + tile - 1) / tile < ((int64_t)1 << 24);
}

// Past the caches a call's 16-byte accesses are marked as used once: 456 us instead of 494
// at [1, 32760, 40, 128] bf16 with tangents, 5.9 TB/s. Narrower ones share their lines with the
// next unit's and stay ordinary.
template <typename T, int V, bool INTERLEAVED, bool JVP>
static void rotary_launch_j(const RotaryParams& p, dim3 grid, hipStream_t s) {
  if constexpr (V * sizeof(T) == 16) {
    if (p.past_caches) {
      hipLaunchKernelGGL((rotary_kernel<T, V, INTERLEAVED, JVP, true>), grid, dim3(kRotaryThreads), 0, s, p);
      return;
    }
  }
  hipLaunchKernelGGL((rotary_kernel<T, V, INTERLEAVED, JVP, false>), grid, dim3(kRotaryThreads), 0, s, p);
}

template <typename T, int V>
static hipError_t rotary_launch_v(const RotaryParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.tokens + p.tile - 1) / p.tile));
  const bool jvp = p.op[0].t != nullptr || p.op[1].t != nullptr;
  if (p.interleaved) jvp ? rotary_launch_j<T, V, true, true>(p, grid, s) : rotary_launch_j<T, V, true, false>(p, grid, s);
  else jvp ? rotary_launch_j<T, V, false, true>(p, grid, s) : rotary_launch_j<T, V, false, false>(p, grid, s);
  return hipGetLastError();
}

template <typename T>
static hipError_t rotary_launch_t(const RotaryParams& p, hipStream_t s) {
  switch (p.vec) {
    case 8:
      if constexpr (sizeof(T) == 2) return rotary_launch_v<T, 8>(p, s);
      return hipErrorInvalidValue;
    case 4: return rotary_launch_v<T, 4>(p, s);
    case 2: return rotary_launch_v<T, 2>(p, s);
    default: return rotary_launch_v<T, 1>(p, s);
  }
}

hipError_t launch_rotary(const RotaryParams& p, int dtype, hipStream_t s) {
  if (dtype == 0) return rotary_launch_t<__bf16>(p, s);
  if (dtype == 1) return rotary_launch_t<_Float16>(p, s);
  return rotary_launch_t<float>(p, s);
}

}  // namespace dmad
