// Gate, residual and norm in one pass, between the two halves of a block:
//   y'  = y, or y * (mean(y^2) + eps)^(-1/2) * wp  (the norm after the branch)
//   x'  = x + rs g y'
//   c   = x' - mean(x') (layer) or x' (rms),  r = (mean(c^2) + eps)^(-1/2),  N = c r
//   n   = N A + O,   A = w (1 + s),  O = b (1 + s) + h
// with g, s, h one row per group of T tokens and w, b, wp one for all. Tangents:
//   N.  = r (t - mean(t) - N mean(N t)),  t = x'.   (without mean(t) for rms)
//   n.  = N. A + (N w + b) s. + h.
// and backwards, with gx and gn the gradients of x' and n, a = gn A:
//   dx  = gx + r (a - mean(a) - N mean(a N)),  dy' = rs g dx  (dy through the
//   norm after the branch by the same formula), and per group and channel
//   P = sum gn N,  Q = sum gn,  R = sum dx y/|y| :
//   ds = w P + b Q,  dh = Q,  dg = rs wp R,
//   dw = sum (1 + s) P,  db = sum (1 + s) Q,  dwp = sum rs g R.
// x' is normed as computed, not as rounded for its store; everything is in
// float32 and rounded once. The backward pass computes x' again from x and y.
//
// A row of up to 2048 channels is one wave's, a wider one a workgroup's; a
// thread holds 8 neighbouring channels of every 8 TPR, so that the whole row is
// in registers and each operand is read once with 16-byte loads.
#include "block_ops.h"
#include "lanes.h"

namespace dmad {

constexpr int kNormThreads = 256;

// Sums over the threads of a row. W waves: each leaves its part in LDS. `slot`
// numbers the reductions between two uses of the same memory, of which there
// is a barrier in between as long as a row makes two.
template <int W, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = group_sum<64>(x[i]);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[wave * N + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += slot[w * N + i];
      x[i] = s;
    }
  }
}

// What a thread holds of a row: 8 channels at col0 + j STEP.
template <int TPR_, int NCH_>
struct NormShape {
  static constexpr int TPR = TPR_, NCH = NCH_, W = TPR / 64, STEP = 8 * TPR, RPB = kNormThreads / TPR;
};

template <typename T, typename S>
struct NormRow {
  Row8<T> v[S::NCH];
  template <bool NT>
  __device__ __forceinline__ void load(const NormRows& o, int b, int s, int col0, int C, bool there) {
    const T* p = (const T*)o.p + b * o.b + s * o.s;
#pragma unroll
    for (int j = 0; j < S::NCH; ++j) {
      v[j].zero();
      if (there && col0 + j * S::STEP < C) v[j].template load<NT>(p + col0 + j * S::STEP);
    }
  }
};

// 8 channels of a vector, widened; `none` where it is absent.
template <typename W>
__device__ __forceinline__ void vec8(const W* p, int col, float none, float (&x)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = none;
    return;
  }
  Row8<W> r;
  r.load(p + col);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = r.get(e);
}
template <typename W>
__device__ __forceinline__ const W* vec_row(const NormVec& v, int b, int f) {
  return v.p == nullptr ? nullptr : (const W*)v.p + b * v.b + f * v.f;
}

enum class Branch { kNone, kPlain, kNormed };

// Mean and sum of squares about it of a row in one exchange: each wave's about
// its own mean, put together by the parallel form. With a tangent t also
// sum t and sum (x - mean) t.
template <typename S, bool JVP>
__device__ __forceinline__ void row_moments(const float (&x)[S::NCH][8], const float (&t)[S::NCH][8], bool layer, int col0, int C,
                                            float* slot, float& mean, float& m2, float& st, float& xt) {
  float own = 0.f;
  if (layer) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < S::NCH; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[j][e];  // zero beyond the row
    sum = group_sum<64>(sum);
    // channels of this wave
    int n = 0;
    const int first = col0 - 8 * lane_id();
#pragma unroll
    for (int j = 0; j < S::NCH; ++j) n += min(max(C - first - j * S::STEP, 0), 512);
    own = n > 0 ? sum / (float)n : 0.f;
    mean = own;
    if constexpr (S::W > 1) {
      // (sum, count are exact enough to be exchanged as they are)
      if (lane_id() == 0) {
        slot[16 + 2 * (threadIdx.x >> 6)] = sum;
        slot[17 + 2 * (threadIdx.x >> 6)] = (float)n;
      }
    }
  } else {
    mean = 0.f;
  }
  float sums[JVP ? 3 : 1] = {};
#pragma unroll
  for (int j = 0; j < S::NCH; ++j) {
    const bool in = col0 + j * S::STEP < C;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = in ? x[j][e] - own : 0.f;
      sums[0] = fmaf(d, d, sums[0]);
      if constexpr (JVP) {
        sums[1] += t[j][e];
        sums[2] = fmaf(d, t[j][e], sums[2]);
      }
    }
  }
  constexpr int N = JVP ? 3 : 1;
  if constexpr (S::W == 1) {
    row_sums<1, N>(sums, slot);
    m2 = sums[0];
    if constexpr (JVP) {
      st = sums[1];
      xt = sums[2];
    }
  } else {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i] = group_sum<64>(sums[i]);
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[wave * N + i] = sums[i];
    }
    __syncthreads();
    if (layer) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < S::W; ++w) total += slot[16 + 2 * w];
      mean = total / (float)C;
    }
    m2 = st = xt = 0.f;
#pragma unroll
    for (int w = 0; w < S::W; ++w) {
      const float n = layer ? slot[17 + 2 * w] : 0.f, off = n > 0.f ? slot[16 + 2 * w] / n - mean : 0.f;
      m2 += fmaf(n * off, off, slot[w * N]);
      if constexpr (JVP) {
        st += slot[w * N + 1];
        xt += fmaf(off, slot[w * N + 1], slot[w * N + 2]);
      }
    }
  }
}
constexpr int kMomentSlot = 24;  // floats of LDS that row_moments takes

template <typename T, typename W, typename S, bool JVP, Branch BR, bool NT>
__global__ __launch_bounds__(kNormThreads) void gated_norm_kernel(GatedNormParams p) {
  __shared__ float slots[2][kMomentSlot];
  const int64_t row = (int64_t)blockIdx.x * S::RPB + threadIdx.x / S::TPR;
  const bool there = row < p.rows;
  if (S::W == 1 && !there) return;  // a whole wave, and no barriers
  const int b = (int)(row / p.S), s = (int)(row % p.S), f = s / p.T;
  const int col0 = (threadIdx.x % S::TPR) * 8;
  const float inv_c = 1.f / (float)p.C;

  float x[S::NCH][8], t[S::NCH][8];
  NormRow<T, S> rx, ry, rtx, rty;
  rx.template load<NT>(p.x, b, s, col0, p.C, there);
  if constexpr (BR != Branch::kNone) ry.template load<NT>(p.y, b, s, col0, p.C, there);
  if constexpr (JVP) rtx.template load<NT>(p.tx, b, s, col0, p.C, there);
  if constexpr (JVP && BR != Branch::kNone) rty.template load<NT>(p.ty, b, s, col0, p.C, there);

  const W* gate = vec_row<W>(p.gate, b, f);
  const W* tgate = vec_row<W>(p.tgate, b, f);
  float yr = 1.f, ym = 0.f;
  if constexpr (BR == Branch::kNormed) {
    float sums[JVP ? 2 : 1] = {};
#pragma unroll
    for (int j = 0; j < S::NCH; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = ry.v[j].get(e);
        sums[0] = fmaf(y, y, sums[0]);
        if constexpr (JVP) sums[1] = fmaf(y, rty.v[j].get(e), sums[1]);
      }
    row_sums<S::W>(sums, slots[0]);
    yr = rsqrtf(sums[0] * inv_c + p.eps);
    if constexpr (JVP) ym = sums[1] * inv_c * yr;
  }
#pragma unroll
  for (int j = 0; j < S::NCH; ++j) {
    const int col = col0 + j * S::STEP;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[j][e] = rx.v[j].get(e);
      t[j][e] = JVP ? rtx.v[j].get(e) : 0.f;
    }
    if (col >= p.C) continue;
    if constexpr (BR != Branch::kNone) {
      float g[8], tg[8], wp[8];
      vec8(gate, col, 1.f, g);
      if constexpr (JVP) vec8(tgate, col, 0.f, tg);
      if constexpr (BR == Branch::kNormed) vec8((const W*)p.post, col, 1.f, wp);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float y = ry.v[j].get(e), ty = JVP ? rty.v[j].get(e) : 0.f;
        if constexpr (BR == Branch::kNormed) {
          y *= yr;
          if constexpr (JVP) ty = fmaf(-y, ym, ty) * yr * wp[e];
          y *= wp[e];
        }
        x[j][e] = fmaf(p.rs * g[e], y, x[j][e]);
        if constexpr (JVP) t[j][e] += p.rs * fmaf(tg[e], y, g[e] * ty);
      }
      if (there) {
        const int64_t at = row * p.C + col;
        Row8<T>::template store<NT>((T*)p.xo + at, x[j]);
        if constexpr (JVP) Row8<T>::template store<NT>((T*)p.txo + at, t[j]);
      }
    }
  }

  float mean, m2, st, xt;
  row_moments<S, JVP>(x, t, p.layer, col0, p.C, slots[1], mean, m2, st, xt);
  const float r = rsqrtf(m2 * inv_c + p.eps);
  const float tm = p.layer ? st * inv_c : 0.f, nt = xt * inv_c * r;

  const W* scale = vec_row<W>(p.scale, b, f);
  const W* shift = vec_row<W>(p.shift, b, f);
  const W* tscale = vec_row<W>(p.tscale, b, f);
  const W* tshift = vec_row<W>(p.tshift, b, f);
#pragma unroll
  for (int j = 0; j < S::NCH; ++j) {
    const int col = col0 + j * S::STEP;
    if (col >= p.C || !there) continue;
    float w[8], o[8], sc[8], sh[8], tsc[8], tsh[8], n[8], tn[8];
    vec8((const W*)p.weight, col, 1.f, w);
    vec8((const W*)p.bias, col, 0.f, o);
    vec8(scale, col, 0.f, sc);
    vec8(shift, col, 0.f, sh);
    if constexpr (JVP) {
      vec8(tscale, col, 0.f, tsc);
      vec8(tshift, col, 0.f, tsh);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = (x[j][e] - mean) * r, v = fmaf(u, w[e], o[e]);  // normed, and with weight and bias
      n[e] = fmaf(v, sc[e], v) + sh[e];
      if constexpr (JVP) {
        const float tv = (t[j][e] - tm - u * nt) * r * w[e];
        tn[e] = fmaf(tv, sc[e], tv) + fmaf(v, tsc[e], tsh[e]);
      }
    }
    const int64_t at = row * p.C + col;
    Row8<T>::template store<NT>((T*)p.no + at, n);
    if constexpr (JVP) Row8<T>::template store<NT>((T*)p.tno + at, tn);
  }
}

// Backward: a workgroup takes a run of a group's tokens, one after the other
// (a token per wave, or all four waves on one), and keeps the group's sums P, Q,
// R in registers.
template <typename T, typename W, typename S, Branch BR, bool NT>
__global__ __launch_bounds__(kNormThreads) void gated_norm_bwd_kernel(GatedNormParams p) {
  __shared__ float slots[3][kMomentSlot];
  __shared__ float strip[S::W == 1 ? S::RPB : 1][S::W == 1 ? 512 : 1];
  const int group = (int)blockIdx.x / p.split, piece = (int)blockIdx.x % p.split;
  const int b = group / p.F, f = group % p.F;
  const int first = (int)((int64_t)p.T * piece / p.split), last = (int)((int64_t)p.T * (piece + 1) / p.split);
  const int col0 = (threadIdx.x % S::TPR) * 8;
  const float inv_c = 1.f / (float)p.C;
  const W* gate = vec_row<W>(p.gate, b, f);
  const W* scale = vec_row<W>(p.scale, b, f);
  float P[S::NCH][8] = {}, Q[S::NCH][8] = {}, R[S::NCH][8] = {};

  for (int i = first + (int)threadIdx.x / S::TPR; i < last; i += S::RPB) {
    const int s = f * p.T + i;
    const int64_t row = (int64_t)b * p.S + s;
    NormRow<T, S> rx, ry, rgx, rgn;
    rx.template load<NT>(p.x, b, s, col0, p.C, true);
    if constexpr (BR != Branch::kNone) ry.template load<NT>(p.y, b, s, col0, p.C, true);
    rgx.template load<NT>(p.tx, b, s, col0, p.C, p.tx.p != nullptr);
    rgn.template load<NT>(p.ty, b, s, col0, p.C, p.ty.p != nullptr);

    float yr = 1.f;
    if constexpr (BR == Branch::kNormed) {
      float sums[1] = {0.f};
#pragma unroll
      for (int j = 0; j < S::NCH; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[0] = fmaf(ry.v[j].get(e), ry.v[j].get(e), sums[0]);
      row_sums<S::W>(sums, slots[2]);
      yr = rsqrtf(sums[0] * inv_c + p.eps);
    }
    float x[S::NCH][8];
#pragma unroll
    for (int j = 0; j < S::NCH; ++j) {
      const int col = col0 + j * S::STEP;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = rx.v[j].get(e);
      if (col >= p.C) continue;
      if constexpr (BR != Branch::kNone) {
        float g[8], wp[8];
        vec8(gate, col, 1.f, g);
        if constexpr (BR == Branch::kNormed) vec8((const W*)p.post, col, 1.f, wp);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float y = ry.v[j].get(e);
          if constexpr (BR == Branch::kNormed) y = y * yr * wp[e];
          x[j][e] = fmaf(p.rs * g[e], y, x[j][e]);
        }
      }
    }
    float mean, m2, st, xt;
    row_moments<S, false>(x, x, p.layer, col0, p.C, slots[0], mean, m2, st, xt);
    const float r = rsqrtf(m2 * inv_c + p.eps);

    // a = gn A, its mean and its mean with N
    float sums[2] = {0.f, 0.f};
    float a[S::NCH][8];
#pragma unroll
    for (int j = 0; j < S::NCH; ++j) {
      const int col = col0 + j * S::STEP;
      if (col >= p.C) continue;
      float w[8], sc[8];
      vec8((const W*)p.weight, col, 1.f, w);
      vec8(scale, col, 0.f, sc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = rgn.v[j].get(e), n = (x[j][e] - mean) * r, gw = g * w[e];
        x[j][e] = n;
        P[j][e] = fmaf(g, n, P[j][e]);
        Q[j][e] += g;
        a[j][e] = fmaf(gw, sc[e], gw);
        sums[0] += a[j][e];
        sums[1] = fmaf(a[j][e], n, sums[1]);
      }
    }
    row_sums<S::W>(sums, slots[1]);
    const float am = p.layer ? sums[0] * inv_c : 0.f, an = sums[1] * inv_c;
    float yu[1] = {0.f};
#pragma unroll
    for (int j = 0; j < S::NCH; ++j) {
      const int col = col0 + j * S::STEP;
      if (col >= p.C) continue;
      const int64_t at = row * p.C + col;
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf(r, a[j][e] - am - x[j][e] * an, rgx.v[j].get(e));
      Row8<T>::template store<NT>((T*)p.xo + at, d);
      if constexpr (BR != Branch::kNone) {
        float g[8];
        vec8(gate, col, 1.f, g);
        if constexpr (BR == Branch::kPlain) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            R[j][e] = fmaf(d[e], ry.v[j].get(e), R[j][e]);
            d[e] *= p.rs * g[e];
          }
          if (p.txo != nullptr) Row8<T>::template store<NT>((T*)p.txo + at, d);
        } else {
          float wp[8];
          vec8((const W*)p.post, col, 1.f, wp);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = ry.v[j].get(e) * yr;
            R[j][e] = fmaf(d[e], y, R[j][e]);
            a[j][e] = d[e] * p.rs * g[e] * wp[e];
            yu[0] = fmaf(a[j][e], y, yu[0]);
          }
        }
      }
    }
    if constexpr (BR == Branch::kNormed) {
      row_sums<S::W>(yu, slots[2] + 8);
      const float m = yu[0] * inv_c;
#pragma unroll
      for (int j = 0; j < S::NCH; ++j) {
        const int col = col0 + j * S::STEP;
        if (col >= p.C || p.txo == nullptr) continue;
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = yr * fmaf(-(ry.v[j].get(e) * yr), m, a[j][e]);
        Row8<T>::template store<NT>((T*)p.txo + row * p.C + col, d);
      }
    }
  }

  // the tokens of the waves put together, 512 channels at a time
  if constexpr (S::W == 1) {
    const int wave = threadIdx.x >> 6, lane = lane_id();
#pragma unroll
    for (int j = 0; j < S::NCH; ++j)
#pragma unroll
      for (int q = 0; q < kNormSums; ++q) {
        if (q == 2 && BR == Branch::kNone) continue;
        float(&acc)[8] = q == 0 ? P[j] : q == 1 ? Q[j] : R[j];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) strip[wave][lane * 8 + e] = acc[e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float sum = strip[0][lane * 8 + e];
#pragma unroll
            for (int w = 1; w < S::RPB; ++w) sum += strip[w][lane * 8 + e];
            acc[e] = sum;
          }
        }
      }
    if (wave != 0) return;
  }
#pragma unroll
  for (int j = 0; j < S::NCH; ++j) {
    const int col = col0 + j * S::STEP;
    if (col >= p.C) continue;
    if (p.partial != nullptr) {
      float* out = p.partial + (int64_t)blockIdx.x * kNormSums * p.C + col;
      Row8<float>::store(out, P[j]);
      Row8<float>::store(out + p.C, Q[j]);
      if constexpr (BR != Branch::kNone) Row8<float>::store(out + 2 * p.C, R[j]);
      continue;
    }
    const int64_t at = (int64_t)group * p.C + col;
    if (p.dscale != nullptr) {
      float w[8], o[8], d[8];
      vec8((const W*)p.weight, col, 1.f, w);
      vec8((const W*)p.bias, col, 0.f, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf(w[e], P[j][e], o[e] * Q[j][e]);
      Row8<W>::store((W*)p.dscale + at, d);
    }
    if (p.dshift != nullptr) Row8<W>::store((W*)p.dshift + at, Q[j]);
    if (BR != Branch::kNone && p.dgate != nullptr) {
      float wp[8], d[8];
      vec8((const W*)p.post, col, 1.f, wp);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = p.rs * wp[e] * R[j][e];
      Row8<W>::store((W*)p.dgate + at, d);
    }
  }
}

// The small operands' gradients from the workgroups' sums, in a fixed order:
// 32 channels and 32 strands of the workgroups per workgroup of this one;
// blockIdx.y is a group, or behind the groups the weights', over all of them.
constexpr int kNormGradCols = 32, kNormGradStrands = 32;

template <typename W>
__global__ __launch_bounds__(1024) void gated_norm_grad_kernel(GatedNormParams p, int group0, int groups) {
  __shared__ float sums[kNormSums][kNormGradStrands][kNormGradCols + 1];
  const int lane = threadIdx.x % kNormGradCols, strand = threadIdx.x / kNormGradCols;
  const int col = (int)blockIdx.x * kNormGradCols + lane;
  const int group = group0 + (int)blockIdx.y;
  const bool all = group >= groups;
  const int64_t first = all ? 0 : (int64_t)group * p.split, last = all ? (int64_t)groups * p.split : first + p.split;
  const bool branch = p.y.p != nullptr;
  float s[kNormSums] = {};
  if (col < p.C) {
#pragma unroll 4
    for (int64_t i = first + strand; i < last; i += kNormGradStrands) {
      const float* x = p.partial + i * kNormSums * p.C + col;
      float by = 1.f, g = 1.f;
      if (all) {
        const int gr = (int)(i / p.split), b = gr / p.F, f = gr % p.F;
        if (p.scale.p != nullptr) by += (float)vec_row<W>(p.scale, b, f)[col];
        if (p.gate.p != nullptr) g = (float)vec_row<W>(p.gate, b, f)[col];
      }
      s[0] = fmaf(by, x[0], s[0]);
      s[1] = fmaf(by, x[p.C], s[1]);
      if (branch) s[2] = fmaf(g, x[2 * (int64_t)p.C], s[2]);
    }
  }
#pragma unroll
  for (int q = 0; q < kNormSums; ++q) sums[q][strand][lane] = s[q];
  __syncthreads();
  if (strand >= kNormSums || col >= p.C) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kNormGradStrands; ++i) sum += sums[strand][i][lane];
  if (all) {
    W* out = (W*)(strand == 0 ? p.dweight : strand == 1 ? p.dbias : p.dpost);
    if (out != nullptr) out[col] = (W)(strand == 2 ? p.rs * sum : sum);
    return;
  }
  const int64_t at = (int64_t)group * p.C + col;
  const float w = p.weight != nullptr ? (float)((const W*)p.weight)[col] : 1.f;
  const float o = p.bias != nullptr ? (float)((const W*)p.bias)[col] : 0.f;
  if (strand == 0 && p.dscale != nullptr) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < kNormGradStrands; ++i) q += sums[1][i][lane];
    ((W*)p.dscale)[at] = (W)fmaf(w, sum, o * q);
  }
  if (strand == 1 && p.dshift != nullptr) ((W*)p.dshift)[at] = (W)sum;
  if (strand == 2 && p.dgate != nullptr)
    ((W*)p.dgate)[at] = (W)(p.rs * (p.post != nullptr ? (float)((const W*)p.post)[col] : 1.f) * sum);
}

#if DMAD_T == 0 && DMAD_W == 0
// Workgroups that a backward pass aims at, and the fewest tokens that one takes.
constexpr int kNormBwdBlocks = 768;
int gated_norm_split(int64_t groups, int T, int C) {
  const int least = C <= kNormWaveC ? 4 : 1;
  int64_t split = (kNormBwdBlocks + groups - 1) / groups;
  const int64_t most = (T + least - 1) / least;
  if (split > most) split = most;
  return split < 1 ? 1 : (int)split;
}
#endif

template <typename T, typename W, typename S>
static hipError_t norm_launch_s(const GatedNormParams& p, bool backward, hipStream_t s) {
  const bool branch = p.y.p != nullptr, normed = p.post != nullptr;
  const dim3 block(kNormThreads);
  if (backward) {
    const dim3 grid((unsigned)(p.B * p.F * p.split));
    if (normed) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, S, Branch::kNormed, false>), grid, block, 0, s, p);
    else if (branch) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, S, Branch::kPlain, false>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, S, Branch::kNone, false>), grid, block, 0, s, p);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((p.rows + S::RPB - 1) / S::RPB));
  auto go = [&](auto jvp) {
    constexpr bool JVP = decltype(jvp)::value != 0;
    if (normed) hipLaunchKernelGGL((gated_norm_kernel<T, W, S, JVP, Branch::kNormed, false>), grid, block, 0, s, p);
    else if (branch) hipLaunchKernelGGL((gated_norm_kernel<T, W, S, JVP, Branch::kPlain, false>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_norm_kernel<T, W, S, JVP, Branch::kNone, false>), grid, block, 0, s, p);
  };
  if (p.tx.p != nullptr) go(IC<1>{});
  else go(IC<0>{});
  return hipGetLastError();
}

template <typename T, typename W>
static hipError_t norm_launch_t(const GatedNormParams& p, bool backward, hipStream_t s) {
  if (p.C <= 512) return norm_launch_s<T, W, NormShape<64, 1>>(p, backward, s);
  if (p.C <= 1536) return norm_launch_s<T, W, NormShape<64, 3>>(p, backward, s);
  if (p.C <= kNormWaveC) return norm_launch_s<T, W, NormShape<64, 4>>(p, backward, s);
  if (p.C <= 6144) return norm_launch_s<T, W, NormShape<256, 3>>(p, backward, s);
  return norm_launch_s<T, W, NormShape<256, 4>>(p, backward, s);
}

// One unit per operand type and type of the small operands (DMAD_T, DMAD_W).
#if DMAD_T == 0
typedef __bf16 NormT;
#elif DMAD_T == 1
typedef _Float16 NormT;
#else
typedef float NormT;
#endif
#if DMAD_W == 0
typedef NormT NormW;
#else
typedef float NormW;
#endif

template <int DTYPE, int WIDE>
hipError_t gated_norm_unit(const GatedNormParams& p, bool backward, hipStream_t s);

template <>
hipError_t gated_norm_unit<DMAD_T, DMAD_W>(const GatedNormParams& p, bool backward, hipStream_t s) {
  hipError_t e = norm_launch_t<NormT, NormW>(p, backward, s);
  if (e != hipSuccess || !backward || p.partial == nullptr) return e;
  const int groups = p.B * p.F;
  const bool per_group = p.dgate != nullptr || p.dscale != nullptr || p.dshift != nullptr;
  const bool weights = p.dweight != nullptr || p.dbias != nullptr || p.dpost != nullptr;
  const int group0 = per_group ? 0 : groups, end = groups + (weights ? 1 : 0);
  const unsigned cols = (unsigned)((p.C + kNormGradCols - 1) / kNormGradCols);
  constexpr int kRows = 32768;  // of a grid
  for (int g = group0; g < end; g += kRows) {
    const int n = end - g < kRows ? end - g : kRows;
    hipLaunchKernelGGL((gated_norm_grad_kernel<NormW>), dim3(cols, (unsigned)n), dim3(1024), 0, s, p, g, groups);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return e;
}

#if DMAD_T == 0 && DMAD_W == 0
template <> hipError_t gated_norm_unit<0, 1>(const GatedNormParams&, bool, hipStream_t);
template <> hipError_t gated_norm_unit<1, 0>(const GatedNormParams&, bool, hipStream_t);
template <> hipError_t gated_norm_unit<1, 1>(const GatedNormParams&, bool, hipStream_t);
template <> hipError_t gated_norm_unit<2, 0>(const GatedNormParams&, bool, hipStream_t);

static hipError_t norm_dispatch(const GatedNormParams& p, int dtype, int wdtype, bool backward, hipStream_t s) {
  const bool wide = wdtype == 2 && dtype != 2;
  if (dtype == 0) return wide ? gated_norm_unit<0, 1>(p, backward, s) : gated_norm_unit<0, 0>(p, backward, s);
  if (dtype == 1) return wide ? gated_norm_unit<1, 1>(p, backward, s) : gated_norm_unit<1, 0>(p, backward, s);
  return gated_norm_unit<2, 0>(p, backward, s);
}
hipError_t launch_gated_norm(const GatedNormParams& p, int dtype, int wdtype, hipStream_t s) {
  return norm_dispatch(p, dtype, wdtype, false, s);
}
hipError_t launch_gated_norm_bwd(const GatedNormParams& p, int dtype, int wdtype, hipStream_t s) {
  return norm_dispatch(p, dtype, wdtype, true, s);
}
#endif

}  // namespace dmad
