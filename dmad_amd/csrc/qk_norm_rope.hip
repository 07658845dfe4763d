// RMSNorm of queries and keys for each head, with the rotation of their pairs
// in the same pass; tangents; the backward pass; and the form that puts new
// keys and values straight into the pages of a cache.
//
// Per head row x of D values, weight w, tangent t, angles theta (one per pair):
//   r = (mean(x^2) + eps)^(-1/2),  n = x r,  y = R(theta)(n w)
//   t' = r (t - n mean(n t)),      ty = R(theta)(t' w)
// and backwards, with g the gradient of y:
//   u = R(-theta) g,  dw = sum over rows of u n,  a = u w,  dx = r (a - n mean(a n))
// R turns each pair (x[2i], x[2i+1]) by theta[i]. Everything is in float32 and
// rounded once, on the store.
//
// A row is D/8 lanes of 8 elements, so one wave pass covers 512/D heads of a
// token with 16-byte loads and the means are sums over D/8 neighbouring lanes.
// A token's rows share their angles: a wave takes up to `per_wave` passes of
// one token (q's heads, then k's, then v's), and its lanes share the sines and
// cosines (D <= 128: one each). HBM-bound: 2 D bytes in and out per row and
// tensor for about 60 vector instructions per 8 elements. 14B with tangents,
// 2.7 GB: 500 us, 5.4 TB/s; gradients of 1.3B, 604 MB: 104 us, 5.8 TB/s.
#include "kv_cache.h"
#include "lanes.h"

namespace dmad {

constexpr int kQkWaves = 4;   // waves per workgroup
constexpr int kQkUnroll = 2;  // passes whose loads are in flight together
constexpr int kQkAppendWaves = 16;  // waves of a workgroup that takes a sequence's new tokens

// Sines and cosines of the 4 pairs of a lane's 8 elements. The 64 / LPH lanes
// at one position of a row share them: each computes 4 LPH / 64 (at least one)
// and takes the others by cross-lane reads.
template <int D>
__device__ __forceinline__ void row_angles(const float* f, int lane, float (&cs)[4], float (&sn)[4]) {
  constexpr int LPH = D / 8, SHARE = 64 / LPH, OWN = SHARE >= 4 ? 1 : 4 / SHARE;
  const int pos = lane % LPH, rank = lane / LPH;
  float s[OWN], c[OWN];
#pragma unroll
  for (int k = 0; k < OWN; ++k) sincosf(f[4 * pos + (rank * OWN + k) % 4], &s[k], &c[k]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int from = pos + LPH * (k / OWN);
    cs[k] = __shfl(c[k % OWN], from);
    sn[k] = __shfl(s[k % OWN], from);
  }
}

// (even, odd) turned by the angle, or back
__device__ __forceinline__ void turn(float (&x)[8], const float (&cs)[4], const float (&sn)[4], float sign) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float e = x[2 * k], o = x[2 * k + 1], s = sign * sn[k];
    x[2 * k] = fmaf(e, cs[k], -(o * s));
    x[2 * k + 1] = fmaf(o, cs[k], e * s);
  }
}

// What a wave works on: a token and a range of its passes.
struct QkUnit {
  int b, i, first, last;
};
__device__ __forceinline__ QkUnit qk_unit(const QkNormRopeParams& p, int64_t unit) {
  const uint32_t per_token = (uint32_t)((p.passes + p.per_wave - 1) / p.per_wave);
  const uint32_t token = (uint32_t)unit / per_token, u = (uint32_t)unit % per_token;
  QkUnit r;
  r.b = (int)(token / (uint32_t)p.S);
  r.i = (int)(token % (uint32_t)p.S);
  r.first = (int)u * p.per_wave;
  r.last = min(r.first + p.per_wave, p.passes);
  return r;
}

// The operand and its pass that pass number `pass` of a token is.
__device__ __forceinline__ int qk_operand(const QkNormRopeParams& p, int& pass) {
  if (pass < p.op[0].passes) return 0;
  pass -= p.op[0].passes;
  if (pass < p.op[1].passes) return 1;
  pass -= p.op[1].passes;
  return 2;
}

// One wave's rows. NT: operands and results past the caches.
template <typename T, typename W, int D, QkMode MODE, bool NT = false>
__device__ __forceinline__ void qk_norm_rope_rows(const QkNormRopeParams& p, const QkUnit u) {
  constexpr int LPH = D / 8, HPP = 64 / LPH;
  constexpr bool JVP = MODE == QkMode::kTangent, APPEND = MODE == QkMode::kAppend;
  const int lane = lane_id();
  const int el = (lane % LPH) * 8, hl = lane / LPH;

  // where the token goes: its slot's page, or none
  KvSlot at{-1, 0};
  int seen = 0;
  if constexpr (APPEND) {
    seen = p.kv.seen[u.b] + u.i;
    at = p.kv.locate(u.b, kv_append_slot(p.kv.length(u.b), u.i, p.kv.capacity()));
  }

  float cs[4], sn[4];
  const bool rope = p.freqs != nullptr;
  if (rope) {
    if constexpr (APPEND) {
      // a position the table has no row for gives NaN
      const bool in = (unsigned)seen < (unsigned)p.freqs_rows;
      row_angles<D>(p.freqs + (int64_t)(in ? seen : 0) * (D / 2), lane, cs, sn);
      if (!in) {
#pragma unroll
        for (int k = 0; k < 4; ++k) cs[k] = sn[k] = __builtin_nanf("");
      }
    } else {
      row_angles<D>(p.freqs + (int64_t)u.b * p.freqs_b + (int64_t)u.i * (D / 2), lane, cs, sn);
    }
  }

  for (int first = u.first; first < u.last; first += kQkUnroll) {
    Row8<T> x[kQkUnroll], t[kQkUnroll];
    Row8<W> w[kQkUnroll];
#pragma unroll
    for (int j = 0; j < kQkUnroll; ++j) {
      int pass = first + j;
      if (pass >= u.last) continue;
      const QkOperand& o = p.op[qk_operand(p, pass)];
      const int h = pass * HPP + hl;
      x[j].zero();
      if constexpr (JVP) t[j].zero();
      if (h < o.H) {
        x[j].template load<NT>((const T*)o.x + u.b * o.xb + u.i * o.xs + h * o.xh + el);
        if constexpr (JVP) t[j].template load<NT>((const T*)o.t + u.b * o.tb + u.i * o.ts + h * o.th + el);
      }
      if (o.w != nullptr) w[j].load((const W*)o.w + el);
    }
#pragma unroll
    for (int j = 0; j < kQkUnroll; ++j) {
      int pass = first + j;
      if (pass >= u.last) continue;
      const int which = qk_operand(p, pass);
      const QkOperand& o = p.op[which];
      const int h = pass * HPP + hl;
      float y[8], ty[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = x[j].get(e);
        if constexpr (JVP) ty[e] = t[j].get(e);
      }
      if (o.w != nullptr) {
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sq = fmaf(y[e], y[e], sq);
          if constexpr (JVP) dot = fmaf(y[e], ty[e], dot);
        }
        const float r = rsqrtf(group_sum<LPH>(sq) * (1.f / D) + p.eps);
        float m = 0.f;
        if constexpr (JVP) m = group_sum<LPH>(dot) * (1.f / D) * r;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = y[e] * r, we = w[j].get(e);
          y[e] = n * we;
          if constexpr (JVP) ty[e] = fmaf(-n, m, ty[e]) * r * we;
        }
      }
      if (rope && which < 2) {
        turn(y, cs, sn, 1.f);
        if constexpr (JVP) turn(ty, cs, sn, 1.f);
      }
      if (h >= o.H) continue;
      if (!APPEND || which == 0) {
        const int64_t out = (((int64_t)u.b * p.S + u.i) * o.H + h) * D + el;
        Row8<T>::template store<NT>((T*)o.out + out, y);
        if constexpr (JVP) Row8<T>::template store<NT>((T*)o.tout + out, ty);
      } else if constexpr (APPEND) {
        if (at.page < 0) continue;
        if (which == 1) {
          Row8<T>::store((T*)p.kv.k + p.kv.k_offset(at, h) + el, y);
          if (el == 0 && p.kv.weight != nullptr) {
            p.kv.weight[p.kv.index(at, h)] = 0.f;
            p.kv.position[p.kv.index(at, h)] = seen;
          }
        } else {
          *(i32x4_t*)((T*)p.kv.v + p.kv.v_offset(at, h) + el) = x[j].v;
        }
      }
    }
  }
}

template <typename T, typename W, int D, QkMode MODE, bool NT>
__global__ __launch_bounds__(64 * kQkWaves) void qk_norm_rope_kernel(QkNormRopeParams p) {
  const int64_t unit = (int64_t)blockIdx.x * kQkWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit < p.units) qk_norm_rope_rows<T, W, D, MODE, NT>(p, qk_unit(p, unit));  // the whole wave
}

__device__ __forceinline__ void kv_advance(const KvPages& kv, int b, int S) {
  kv.lengths[b] = kv_append_length(kv.length(b), S, kv.capacity());
  kv.seen[b] += S;
}

// An append of few rows per sequence: one workgroup takes them all and, when
// every wave has read the length, sets it.
template <typename T, typename W, int D>
__global__ __launch_bounds__(64 * kQkAppendWaves) void kv_append_kernel(QkNormRopeParams p) {
  const int b = (int)blockIdx.x, per_token = (p.passes + p.per_wave - 1) / p.per_wave;
  for (int unit = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < p.S * per_token; unit += (int)(blockDim.x >> 6))
    qk_norm_rope_rows<T, W, D, QkMode::kAppend>(p, qk_unit(p, (int64_t)b * p.S * per_token + unit));
  __syncthreads();
  if (threadIdx.x == 0) kv_advance(p.kv, b, p.S);
}

// Lengths and counts after any other append, in a launch of its own: every wave
// of the append reads them.
__global__ void kv_advance_kernel(KvPages kv, int S) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < kv.B) kv_advance(kv, b, S);
}

// Backward: persistent waves take units in turn and keep the sums of the
// weights' gradients in registers; a workgroup's sums go to its row of
// `partial`, and a second kernel adds the rows in order, so the result does
// not change from call to call.
constexpr int kQkBwdBlocks = 1024;

template <typename T, typename W, int D, bool NT>
__global__ __launch_bounds__(64 * kQkWaves) void qk_norm_rope_bwd_kernel(QkNormRopeParams p) {
  constexpr int LPH = D / 8, HPP = 64 / LPH;
  __shared__ float sums[kQkWaves][2][D];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int el = (lane % LPH) * 8, hl = lane / LPH;
  float dw[2][8] = {};
  for (int64_t unit = (int64_t)blockIdx.x * kQkWaves + wave; unit < p.units; unit += (int64_t)gridDim.x * kQkWaves) {
    const QkUnit u = qk_unit(p, unit);
    float cs[4], sn[4];
    const bool rope = p.freqs != nullptr;
    if (rope) row_angles<D>(p.freqs + (int64_t)u.b * p.freqs_b + (int64_t)u.i * (D / 2), lane, cs, sn);
    for (int first = u.first; first < u.last; first += kQkUnroll) {
      Row8<T> x[kQkUnroll], g[kQkUnroll];
      Row8<W> w[kQkUnroll];
#pragma unroll
      for (int j = 0; j < kQkUnroll; ++j) {
        int pass = first + j;
        if (pass >= u.last) continue;
        const QkOperand& o = p.op[qk_operand(p, pass)];
        const int h = pass * HPP + hl;
        x[j].zero();
        g[j].zero();
        if (h < o.H) {
          x[j].template load<NT>((const T*)o.x + u.b * o.xb + u.i * o.xs + h * o.xh + el);
          g[j].template load<NT>((const T*)o.t + u.b * o.tb + u.i * o.ts + h * o.th + el);
        }
        if (o.w != nullptr) w[j].load((const W*)o.w + el);
      }
#pragma unroll
      for (int j = 0; j < kQkUnroll; ++j) {
        int pass = first + j;
        if (pass >= u.last) continue;
        const int which = qk_operand(p, pass);
        const QkOperand& o = p.op[which];
        const int h = pass * HPP + hl;
        float a[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = g[j].get(e);
        if (rope) turn(a, cs, sn, -1.f);
        if (o.w != nullptr) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sq = fmaf(x[j].get(e), x[j].get(e), sq);
          const float r = rsqrtf(group_sum<LPH>(sq) * (1.f / D) + p.eps);
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float n = x[j].get(e) * r;
            // a row beyond the last head reads as zero: with eps = 0 its r is
            // infinite and n not a number, and it may not reach the sums
            if (h < o.H) {
              if (which == 0) dw[0][e] = fmaf(a[e], n, dw[0][e]);
              else dw[1][e] = fmaf(a[e], n, dw[1][e]);
            }
            a[e] *= w[j].get(e);
            dot = fmaf(a[e], n, dot);
          }
          const float m = group_sum<LPH>(dot) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = r * fmaf(-(x[j].get(e) * r), m, a[e]);
        }
        if (h < o.H) Row8<T>::template store<NT>((T*)o.out + (((int64_t)u.b * p.S + u.i) * o.H + h) * D + el, a);
      }
    }
  }
  if (p.partial == nullptr) return;
  // the heads of a wave, then the waves
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s = dw[c][e];
#pragma unroll
      for (int m = LPH; m < 64; m <<= 1) s += __shfl_xor(s, m);
      if (hl == 0) sums[wave][c][el + e] = s;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += 64 * kQkWaves) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kQkWaves; ++v) s += (&sums[v][0][0])[i];
    p.partial[(int64_t)blockIdx.x * 2 * D + i] = s;
  }
}

// dw[c] = sum of column c of partial [blocks][2 D]: 16 columns and 64 strands
// of rows per workgroup, at most kQkBwdBlocks / 64 rows each.
template <typename W>
__global__ __launch_bounds__(1024) void qk_weight_grad_kernel(const float* partial, int blocks, int D, W* dwq, W* dwk) {
  __shared__ float sums[64][17];
  const int col = threadIdx.x & 15, strand = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float x[kQkBwdBlocks / 64];
#pragma unroll
  for (int j = 0; j < kQkBwdBlocks / 64; ++j) {
    const int i = strand + 64 * j;
    x[j] = i < blocks ? partial[(int64_t)i * 2 * D + c] : 0.f;
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < kQkBwdBlocks / 64; ++j) s += x[j];
  sums[strand][col] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // strands 16 apart in each of four lane groups, then the groups
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += sums[4 * i + strand][col];
  s = across32<LaneAdd>(across16<LaneAdd>(s));
  W* out = c < D ? dwq : dwk;
  if (strand == 0 && out != nullptr) out[c < D ? c : c - D] = (W)s;
}

// A backward pass or a forward with tangents that moves more than the 256 MB
// memory-side cache holds goes past it (non-temporal loads and stores). A plain
// forward does not: its results are read next by the attention, and its
// operands again by the backward pass. Forward and backward together, none past
// the cache -> backward only -> both: 201 MB of 1.3B queries and keys 194 ->
// 187 -> 184 us, 671 MB of 14B 652 -> 627 -> 614 us, 168 MB of 256-wide heads
// 170 -> 143 -> 155 us; with tangents 518 -> 499 us for 14B.
bool qk_past_caches(int64_t bytes) { return bytes > (int64_t)256 << 20; }

// A workgroup per sequence saves the launch that advances the lengths and is
// slower where a wave takes more than two passes. 32 sequences, one launch
// against two, per replayed append: 4.0 against 5.2 us for 4 passes, 4.5 - 5.3 for
// 12, 5.3 - 5.3 for 24, 5.6 to 5.9 - 5.5 for 32, 6.8 - 5.7 to 6.0 for 48. An eager call
// also saves the second launch's host time.
constexpr int kQkAppendPasses = 32;
void qk_append_split(QkNormRopeParams& p) {
  const int64_t passes = (int64_t)p.S * p.passes;
  p.by_sequence = passes <= kQkAppendPasses;
  if (!p.by_sequence) return;
  p.per_wave = (int)((passes + kQkAppendWaves - 1) / kQkAppendWaves);
  if (p.per_wave > p.passes) p.per_wave = p.passes;
  p.units = (int64_t)p.B * p.S * ((p.passes + p.per_wave - 1) / p.per_wave);
}

int64_t qk_norm_rope_bwd_blocks(int64_t units) {
  const int64_t blocks = (units + kQkWaves - 1) / kQkWaves;
  return blocks < kQkBwdBlocks ? blocks : kQkBwdBlocks;
}

template <typename T, typename W, int D>
static hipError_t qk_launch_d(const QkNormRopeParams& p, QkMode mode, hipStream_t s) {
  const dim3 grid((unsigned)((p.units + kQkWaves - 1) / kQkWaves)), block(64 * kQkWaves);
  if (mode == QkMode::kPrimal) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<T, W, D, QkMode::kPrimal, false>), grid, block, 0, s, p);
  } else if (mode == QkMode::kTangent) {
    if (p.past_caches) hipLaunchKernelGGL((qk_norm_rope_kernel<T, W, D, QkMode::kTangent, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<T, W, D, QkMode::kTangent, false>), grid, block, 0, s, p);
  } else if constexpr (sizeof(T) == 2) {
    if (p.by_sequence) {
      const int64_t units = p.units / p.B;
      const unsigned waves = (unsigned)(units < kQkAppendWaves ? units : kQkAppendWaves);
      hipLaunchKernelGGL((kv_append_kernel<T, W, D>), dim3((unsigned)p.B), dim3(64 * waves), 0, s, p);
      return hipGetLastError();
    }
    hipLaunchKernelGGL((qk_norm_rope_kernel<T, W, D, QkMode::kAppend, false>), grid, block, 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kv_advance_kernel, dim3((unsigned)((p.B + 255) / 256)), dim3(256), 0, s, p.kv, p.S);
  }
  return hipGetLastError();
}

template <typename T, typename W, int D>
static hipError_t qk_launch_bwd_d(const QkNormRopeParams& p, void* dwq, void* dwk, hipStream_t s) {
  const int blocks = (int)qk_norm_rope_bwd_blocks(p.units);
  if (p.past_caches) hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, W, D, true>), dim3(blocks), dim3(64 * kQkWaves), 0, s, p);
  else hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, W, D, false>), dim3(blocks), dim3(64 * kQkWaves), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.partial == nullptr) return e;
  hipLaunchKernelGGL((qk_weight_grad_kernel<W>), dim3(2 * D / 16), dim3(1024), 0, s, p.partial, blocks, D, (W*)dwq, (W*)dwk);
  return hipGetLastError();
}

// The instantiation for a type, a weight type (the same or fp32) and a head dim.
template <typename T, typename W, typename F>
static hipError_t qk_by_dim(int D, F f) {
  switch (D) {
    case 16: return f(T{}, W{}, IC<16>{});
    case 32: return f(T{}, W{}, IC<32>{});
    case 64: return f(T{}, W{}, IC<64>{});
    case 128: return f(T{}, W{}, IC<128>{});
    case 256: return f(T{}, W{}, IC<256>{});
  }
  return hipErrorInvalidValue;
}
template <typename F>
static hipError_t qk_by_type(int dtype, int wdtype, int D, F f) {
  const bool wide = wdtype == 2;
  if (dtype == 0) return wide ? qk_by_dim<__bf16, float>(D, f) : qk_by_dim<__bf16, __bf16>(D, f);
  if (dtype == 1) return wide ? qk_by_dim<_Float16, float>(D, f) : qk_by_dim<_Float16, _Float16>(D, f);
  return qk_by_dim<float, float>(D, f);
}

hipError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dtype, int wdtype, QkMode mode, hipStream_t s) {
  return qk_by_type(dtype, wdtype, p.D, [&](auto t, auto w, auto d) {
    return qk_launch_d<decltype(t), decltype(w), decltype(d)::value>(p, mode, s);
  });
}

hipError_t launch_qk_norm_rope_bwd(const QkNormRopeParams& p, int dtype, int wdtype, void* dwq, void* dwk, hipStream_t s) {
  return qk_by_type(dtype, wdtype, p.D, [&](auto t, auto w, auto d) {
    return qk_launch_bwd_d<decltype(t), decltype(w), decltype(d)::value>(p, dwq, dwk, s);
  });
}

}  // namespace dmad
