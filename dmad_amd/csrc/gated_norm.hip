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
// Bound by its bytes: 32760 tokens of 1536 channels in bf16 take 77 us forward (403 MB, 5.2
// TB/s) and 108 + 8 us backward (604 MB and 23 MB of sums, 5.8 TB/s), of 5120 264, 428 + 18
// and, forward with tangents, 508 us (5.1, 4.7 and 5.3 TB/s); a 4 GiB copy reaches 4.7. A
// lane holds 8 neighbouring channels (one 16-byte access per
// operand), so a row is ceil(C / 512) waves, which make one workgroup and exchange
// their sums through LDS: behind one barrier per row forwards, two backwards, and with
// a norm after the branch two and four; a row of one wave needs none, and
// four of them share a workgroup. A workgroup takes a run of a group's tokens: gate,
// scale, shift and the weights stay in its registers, and the next token's rows are
// requested before this one's are worked on.
#include "block_ops.h"
#include "lanes.h"

namespace dmad {

constexpr int kNormRowsPerGroup = 4;  // waves of a workgroup whose rows are one wave's

// One token's operands as loaded: up to four rows, 8 channels each.
template <typename T, int N>
struct NormToken {
  Row8<T> v[N];
  template <bool NT>
  __device__ __forceinline__ void load(const NormRows* const (&o)[N], int b, int s, int col, bool there) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k].zero();
      if (there && o[k]->p != nullptr) v[k].template load<NT>((const T*)o[k]->p + b * o[k]->b + s * o[k]->s + col);
    }
  }
};

// 8 channels of a vector, widened; `none` where it is absent.
template <typename W>
__device__ __forceinline__ void vec8(const W* p, int col, bool there, float none, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = none;
  if (p == nullptr || !there) return;
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

constexpr int kNormMaxWaves = kNormMaxC / 512;
typedef float NormSlot[kNormMaxWaves][4];  // what the waves of a row exchange at once

// Sums over a row. Each wave leaves its own in `slot`, then a lane takes a wave's
// and 16 lanes add them up. The same slot may be used again behind another barrier.
template <bool ONE, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], NormSlot& slot, int waves) {
  static_assert(N <= 4);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = group_sum<64>(x[i]);
  if constexpr (!ONE) {
    const int lane = lane_id(), w = lane & 15;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[threadIdx.x >> 6][i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = group_sum<16>(w < waves ? slot[w < waves ? w : 0][i] : 0.f);
  }
}

// Mean (layer) and sum of squares about it of a row in one exchange: each wave's
// about its own mean, put together by the parallel form. With a tangent t also
// sum t and sum (x - mean) t.
template <bool ONE, bool JVP>
__device__ __forceinline__ void row_moments(const float (&x)[8], const float (&t)[8], bool layer, bool there, int C, int waves,
                                            NormSlot& slot, float& mean, float& m2, float& st, float& xt) {
  const int lane = lane_id();
  float sum = 0.f, own = 0.f;
  if (layer) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e];  // zero beyond the row
    sum = group_sum<64>(sum);
    const int n = min(C - (int)(ONE ? 0 : threadIdx.x >> 6) * 512, 512);
    own = sum / (float)n;
  }
  constexpr int N = JVP ? 3 : 1;
  float s[N] = {};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = there ? x[e] - own : 0.f;
    s[0] = fmaf(d, d, s[0]);
    if constexpr (JVP) {
      s[1] += t[e];
      s[2] = fmaf(d, t[e], s[2]);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = group_sum<64>(s[i]);
  mean = own;
  m2 = s[0];
  if constexpr (JVP) {
    st = s[1];
    xt = s[2];
  }
  if constexpr (!ONE) {
    const int w = lane & 15;
    if (lane == 0) {
      slot[threadIdx.x >> 6][0] = sum;
#pragma unroll
      for (int i = 0; i < N; ++i) slot[threadIdx.x >> 6][1 + i] = s[i];
    }
    __syncthreads();
    const bool in = w < waves;
    const NormSlot& r = slot;
    const int at = in ? w : 0;
    const float n = in ? (float)min(C - 512 * w, 512) : 0.f, ws = in ? r[at][0] : 0.f;
    float off = 0.f;
    if (layer) {
      mean = group_sum<16>(ws) / (float)C;
      off = in ? ws / n - mean : 0.f;
    }
    m2 = group_sum<16>(in ? fmaf(n * off, off, r[at][1]) : 0.f);
    if constexpr (JVP) {
      st = group_sum<16>(in ? r[at][2] : 0.f);
      xt = group_sum<16>(in ? fmaf(off, r[at][2], r[at][3]) : 0.f);
    }
  }
}

// The tokens of a workgroup (ONE: of a wave in turn): [first, last) of group
// blockIdx.x / split, every `step`-th from `i` on.
struct NormRun {
  int group, b, f, i, last, step;
};
template <bool ONE>
__device__ __forceinline__ NormRun norm_run(const GatedNormParams& p) {
  NormRun r;
  const int piece = (int)blockIdx.x % p.split;
  r.group = (int)blockIdx.x / p.split;
  r.b = r.group / p.F;
  r.f = r.group % p.F;
  r.i = (int)((int64_t)p.T * piece / p.split) + (ONE ? (int)(threadIdx.x >> 6) : 0);
  r.last = (int)((int64_t)p.T * (piece + 1) / p.split);
  r.step = ONE ? kNormRowsPerGroup : 1;
  return r;
}

template <typename T, typename W, bool ONE, bool JVP, Branch BR, bool NT>
__global__ __launch_bounds__(ONE ? 64 * kNormRowsPerGroup : 64 * kNormMaxWaves) void gated_norm_kernel(GatedNormParams p) {
  __shared__ NormSlot slots[2][2];
  const NormRun run = norm_run<ONE>(p);
  const int col = (ONE ? lane_id() : (int)threadIdx.x) * 8, waves = (int)blockDim.x >> 6;
  const bool there = col < p.C;
  const float inv_c = 1.f / (float)p.C;
  constexpr bool BRANCH = BR != Branch::kNone;
  constexpr int N = (BRANCH ? 2 : 1) * (JVP ? 2 : 1), TX = BRANCH ? 2 : 1;
  const NormRows* ops[N];
  ops[0] = &p.x;
  if constexpr (BRANCH) ops[1] = &p.y;
  if constexpr (JVP) ops[TX] = &p.tx;
  if constexpr (JVP && BRANCH) ops[3] = &p.ty;

  // n = u A + O and its tangent u. A + u B + Q
  float g[8], tg[8], wp[8], A[8], O[8], tB[8], tQ[8];
  {
    float w[8], o[8], sc[8];
    vec8((const W*)p.weight, col, there, 1.f, w);
    vec8((const W*)p.bias, col, there, 0.f, o);
    vec8(vec_row<W>(p.scale, run.b, run.f), col, there, 0.f, sc);
    vec8(vec_row<W>(p.shift, run.b, run.f), col, there, 0.f, O);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      A[e] = fmaf(w[e], sc[e], w[e]);
      O[e] += fmaf(o[e], sc[e], o[e]);
    }
    if constexpr (JVP) {
      vec8(vec_row<W>(p.tscale, run.b, run.f), col, there, 0.f, sc);
      vec8(vec_row<W>(p.tshift, run.b, run.f), col, there, 0.f, tQ);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        tB[e] = w[e] * sc[e];
        tQ[e] = fmaf(o[e], sc[e], tQ[e]);
      }
    }
    if constexpr (BRANCH) {
      vec8(vec_row<W>(p.gate, run.b, run.f), col, there, 1.f, g);
      if constexpr (JVP) vec8(vec_row<W>(p.tgate, run.b, run.f), col, there, 0.f, tg);
      if constexpr (BR == Branch::kNormed) vec8((const W*)p.post, col, there, 1.f, wp);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] *= p.rs;
        if constexpr (JVP) tg[e] *= p.rs;
      }
    }
  }

  // (with tangents the registers for a second token cost a workgroup per CU: 541 us
  // against 510 for 14B)
  constexpr bool AHEAD = !JVP;
  NormToken<T, N> now, next;
  if constexpr (AHEAD) next.template load<NT>(ops, run.b, run.f * p.T + run.i, col, there && run.i < run.last);
  int odd = 0;
  for (int i = run.i; i < run.last; i += run.step, odd ^= 1) {
    if constexpr (AHEAD) {
      now = next;
      next.template load<NT>(ops, run.b, run.f * p.T + i + run.step, col, there && i + run.step < run.last);
    } else {
      now.template load<NT>(ops, run.b, run.f * p.T + i, col, there);
    }
    const int64_t at = ((int64_t)run.b * p.S + run.f * p.T + i) * p.C + col;
    float x[8], t[8];
    float yr = 1.f, ym = 0.f;
    if constexpr (BR == Branch::kNormed) {
      float sums[JVP ? 2 : 1] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = now.v[1].get(e);
        sums[0] = fmaf(y, y, sums[0]);
        if constexpr (JVP) sums[1] = fmaf(y, now.v[3].get(e), sums[1]);
      }
      row_sums<ONE>(sums, slots[odd][0], waves);
      yr = rsqrtf(sums[0] * inv_c + p.eps);
      if constexpr (JVP) ym = sums[1] * inv_c * yr;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = now.v[0].get(e);
      t[e] = JVP ? now.v[JVP ? TX : 0].get(e) : 0.f;
      if constexpr (BRANCH) {
        float y = now.v[1].get(e), ty = JVP ? now.v[JVP ? 3 : 0].get(e) : 0.f;
        if constexpr (BR == Branch::kNormed) {
          y *= yr;
          if constexpr (JVP) ty = fmaf(-y, ym, ty) * yr * wp[e];
          y *= wp[e];
        }
        x[e] = fmaf(g[e], y, x[e]);
        if constexpr (JVP) t[e] += fmaf(tg[e], y, g[e] * ty);
      }
    }
    if (BRANCH && there) {
      Row8<T>::template store<NT>((T*)p.xo + at, x);
      if constexpr (JVP) Row8<T>::template store<NT>((T*)p.txo + at, t);
    }
    float mean, m2, st, xt;
    row_moments<ONE, JVP>(x, t, p.layer, there, p.C, waves, slots[odd][1], mean, m2, st, xt);
    if (!there) continue;
    const float r = rsqrtf(m2 * inv_c + p.eps);
    float n[8], tn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = (x[e] - mean) * r;
      n[e] = fmaf(u, A[e], O[e]);
      if constexpr (JVP) {
        const float tm = p.layer ? st * inv_c : 0.f, nt = xt * inv_c * r;
        tn[e] = fmaf((t[e] - tm - u * nt) * r, A[e], fmaf(u, tB[e], tQ[e]));
      }
    }
    Row8<T>::template store<NT>((T*)p.no + at, n);
    if constexpr (JVP) Row8<T>::template store<NT>((T*)p.tno + at, tn);
  }
}

// Backward: the run's sums P, Q, R stay in registers.
template <typename T, typename W, bool ONE, Branch BR, bool NT>
__global__ __launch_bounds__(ONE ? 64 * kNormRowsPerGroup : 64 * kNormMaxWaves) void gated_norm_bwd_kernel(GatedNormParams p) {
  __shared__ NormSlot slots[4];
  __shared__ float strip[ONE ? kNormRowsPerGroup : 1][ONE ? 512 : 1];
  const NormRun run = norm_run<ONE>(p);
  const int col = (ONE ? lane_id() : (int)threadIdx.x) * 8, waves = (int)blockDim.x >> 6;
  const bool there = col < p.C;
  const float inv_c = 1.f / (float)p.C;
  constexpr bool BRANCH = BR != Branch::kNone;
  constexpr int N = BRANCH ? 4 : 3;
  const NormRows* ops[N];
  ops[0] = &p.x;
  ops[1] = &p.tx;  // the gradient of x'
  ops[2] = &p.ty;  // and of n
  if constexpr (BRANCH) ops[3] = &p.y;

  float g[8], wp[8], A[8];
  {
    float sc[8];
    vec8((const W*)p.weight, col, there, 1.f, A);
    vec8(vec_row<W>(p.scale, run.b, run.f), col, there, 0.f, sc);
#pragma unroll
    for (int e = 0; e < 8; ++e) A[e] = fmaf(A[e], sc[e], A[e]);
    if constexpr (BRANCH) {
      vec8(vec_row<W>(p.gate, run.b, run.f), col, there, 1.f, g);
      if constexpr (BR == Branch::kNormed) vec8((const W*)p.post, col, there, 1.f, wp);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] *= p.rs;
    }
  }
  float P[8] = {}, Q[8] = {}, R[8] = {};

  // (in float32 a second token's registers spill: 469 us against 454 for 12480 tokens of 5120)
  constexpr bool AHEAD = sizeof(T) == 2;
  NormToken<T, N> next;
  if constexpr (AHEAD) next.template load<NT>(ops, run.b, run.f * p.T + run.i, col, there && run.i < run.last);
  for (int i = run.i; i < run.last; i += run.step) {
    NormToken<T, N> now;
    if constexpr (AHEAD) {
      now = next;
      next.template load<NT>(ops, run.b, run.f * p.T + i + run.step, col, there && i + run.step < run.last);
    } else {
      now.template load<NT>(ops, run.b, run.f * p.T + i, col, there);
    }
    const int64_t at = ((int64_t)run.b * p.S + run.f * p.T + i) * p.C + col;
    float yr = 1.f;
    if constexpr (BR == Branch::kNormed) {
      float sums[1] = {0.f};
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[0] = fmaf(now.v[3].get(e), now.v[3].get(e), sums[0]);
      row_sums<ONE>(sums, slots[2], waves);
      yr = rsqrtf(sums[0] * inv_c + p.eps);
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = now.v[0].get(e);
      if constexpr (BRANCH) {
        float y = now.v[3].get(e);
        if constexpr (BR == Branch::kNormed) y = y * yr * wp[e];
        x[e] = fmaf(g[e], y, x[e]);
      }
    }
    float mean, m2, st, xt;
    row_moments<ONE, false>(x, x, p.layer, there, p.C, waves, slots[0], mean, m2, st, xt);
    const float r = rsqrtf(m2 * inv_c + p.eps);
    // a = gn A, its mean and its mean with N
    float sums[2] = {0.f, 0.f}, a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float gn = now.v[2].get(e), n = there ? (x[e] - mean) * r : 0.f;
      x[e] = n;
      P[e] = fmaf(gn, n, P[e]);
      Q[e] += gn;
      a[e] = gn * A[e];
      sums[0] += a[e];
      sums[1] = fmaf(a[e], n, sums[1]);
    }
    row_sums<ONE>(sums, slots[1], waves);
    const float am = p.layer ? sums[0] * inv_c : 0.f, an = sums[1] * inv_c;
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = fmaf(r, a[e] - am - x[e] * an, now.v[1].get(e));
    if (there) Row8<T>::template store<NT>((T*)p.xo + at, d);
    if constexpr (BR == Branch::kPlain) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        R[e] = fmaf(d[e], now.v[3].get(e), R[e]);
        d[e] *= g[e];
      }
      if (there && p.txo != nullptr) Row8<T>::template store<NT>((T*)p.txo + at, d);
    }
    if constexpr (BR == Branch::kNormed) {
      float yu[1] = {0.f};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = now.v[3].get(e) * yr;
        // (beyond the row y is zero, and d is not: it may not be a number there)
        if (there) R[e] = fmaf(d[e], y, R[e]);
        d[e] = there ? d[e] * g[e] * wp[e] : 0.f;
        yu[0] = fmaf(d[e], y, yu[0]);
      }
      row_sums<ONE>(yu, slots[3], waves);
      const float m = yu[0] * inv_c;
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = yr * fmaf(-(now.v[3].get(e) * yr), m, d[e]);
      if (there && p.txo != nullptr) Row8<T>::template store<NT>((T*)p.txo + at, d);
    }
  }

  // the tokens of the waves put together
  if constexpr (ONE) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < (BRANCH ? 3 : 2); ++q) {
      float(&acc)[8] = q == 0 ? P : q == 1 ? Q : R;
      if (q > 0) __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) strip[wave][col + e] = acc[e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc[e] = strip[0][col + e];
#pragma unroll
        for (int w = 1; w < kNormRowsPerGroup; ++w) acc[e] += strip[ONE ? w : 0][col + e];
      }
    }
    if (wave != 0) return;
  }
  if (!there) return;
  if (p.partial != nullptr) {
    float* out = p.partial + (int64_t)blockIdx.x * kNormSums * p.C + col;
    Row8<float>::store(out, P);
    Row8<float>::store(out + p.C, Q);
    if constexpr (BRANCH) Row8<float>::store(out + 2 * p.C, R);
    return;
  }
  const int64_t at = (int64_t)run.group * p.C + col;
  if (p.dscale != nullptr) {
    float w[8], o[8], d[8];
    vec8((const W*)p.weight, col, true, 1.f, w);
    vec8((const W*)p.bias, col, true, 0.f, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = fmaf(w[e], P[e], o[e] * Q[e]);
    Row8<W>::store((W*)p.dscale + at, d);
  }
  if (p.dshift != nullptr) Row8<W>::store((W*)p.dshift + at, Q);
  if (BRANCH && p.dgate != nullptr) {
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = p.rs * (BR == Branch::kNormed ? wp[e] : 1.f) * R[e];
    Row8<W>::store((W*)p.dgate + at, d);
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
    if (all && (p.scale.p != nullptr || p.gate.p != nullptr)) {
#pragma unroll 2
      for (int64_t i = first + strand; i < last; i += kNormGradStrands) {
        const float* x = p.partial + i * kNormSums * p.C + col;
        const int gr = (int)(i / p.split), b = gr / p.F, f = gr % p.F;
        const float by = p.scale.p != nullptr ? 1.f + (float)vec_row<W>(p.scale, b, f)[col] : 1.f;
        const float g = p.gate.p != nullptr ? (float)vec_row<W>(p.gate, b, f)[col] : 1.f;
        s[0] = fmaf(by, x[0], s[0]);
        s[1] = fmaf(by, x[p.C], s[1]);
        if (branch) s[2] = fmaf(g, x[2 * (int64_t)p.C], s[2]);
      }
    } else if (all) {
      // many workgroups, few gradients: 27 us in the loop below for two weights' over 2997
      // tokens of 1536, 9 with only their sums read and eight loads in flight
      const bool take[kNormSums] = {p.dweight != nullptr, p.dbias != nullptr, p.dpost != nullptr};
#pragma unroll
      for (int q = 0; q < kNormSums; ++q) {
        if (!take[q]) continue;
        const float* x = p.partial + q * (int64_t)p.C + col;
#pragma unroll 8
        for (int64_t i = first + strand; i < last; i += kNormGradStrands) s[q] += x[i * kNormSums * p.C];
      }
    } else {
#pragma unroll 4
      for (int64_t i = first + strand; i < last; i += kNormGradStrands) {
        const float* x = p.partial + i * kNormSums * p.C + col;
        s[0] += x[0];
        s[1] += x[p.C];
        if (branch) s[2] += x[2 * (int64_t)p.C];
      }
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
int norm_waves(int C) { return C <= 512 ? kNormRowsPerGroup : (C + 511) / 512; }
// Workgroups per group of tokens. A forward pass takes short runs, eight rounds of 20 waves
// per CU, and a call too small for runs of two tokens one such round: 32760 tokens of
// 5120 264 us with 4096 workgroups, 293 with 1638, 288 with 512; 6000 tokens 55, 50 and 42. A
// backward pass leaves sums behind for each, and of rows of ten waves a CU
// holds one (16 waves of 128 registers): it has as few as fill a round of those, or a few
// rounds, best. 32760 tokens of 5120 with the weights' gradients alone take 553 us with 410
// workgroups, 371 with 256; of 1536 in 21 modulated groups 116 us with 1029, 110 with 1260. The rule
// does not weigh the sums' bytes, which count where groups are many: 32256 tokens of 1536 in 672
// groups get 7392 workgroups, whose 272 MB of sums take 123 + 118 us with the data's 595 MB.
int gated_norm_split(int64_t groups, int T, int C, NormPass pass) {
  const int waves = norm_waves(C);
  int64_t split;
  if (pass == NormPass::kTangent) {
    split = (kNormTangentWaves / waves + groups - 1) / groups;
  } else if (pass == NormPass::kForward) {
    int64_t aim = kNormFwdWaves / waves;
    if (groups * T < 2 * aim * (C <= 512 ? kNormRowsPerGroup : 1)) aim = 256 * (waves < kNormFwdHeld ? kNormFwdHeld / waves : 1);
    split = aim / groups;
  } else {
    const int64_t slots = 256 * (waves < kNormBwdHeld ? kNormBwdHeld / waves : 1);
    split = slots / groups;
    if (groups > slots / 16) {
      double fullest = 0;
      for (int64_t n = 1; n <= 16 && fullest < 0.95; ++n) {
        const int64_t rounds = (n * groups + slots - 1) / slots;
        const double full = (double)(n * groups) / (double)(rounds * slots);
        if (full > fullest) fullest = full, split = n;
      }
    }
  }
  const int64_t least = C <= 512 ? kNormRowsPerGroup : 1, most = (T + least - 1) / least;
  if (split > most) split = most;
  return split < 1 ? 1 : (int)split;
}
#endif

template <typename T, typename W, bool ONE, bool NT>
static hipError_t norm_launch_s(const GatedNormParams& p, bool backward, hipStream_t s) {
  const bool branch = p.y.p != nullptr, normed = p.post != nullptr;
  const dim3 grid((unsigned)(p.B * p.F * p.split)), block(64 * norm_waves(p.C));
  if (backward) {
    if (normed) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, ONE, Branch::kNormed, NT>), grid, block, 0, s, p);
    else if (branch) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, ONE, Branch::kPlain, NT>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, W, ONE, Branch::kNone, NT>), grid, block, 0, s, p);
    return hipGetLastError();
  }
  auto go = [&](auto jvp, auto nt) {
    constexpr bool JVP = decltype(jvp)::value != 0, PAST = decltype(nt)::value != 0;
    if (normed) hipLaunchKernelGGL((gated_norm_kernel<T, W, ONE, JVP, Branch::kNormed, PAST>), grid, block, 0, s, p);
    else if (branch) hipLaunchKernelGGL((gated_norm_kernel<T, W, ONE, JVP, Branch::kPlain, PAST>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_norm_kernel<T, W, ONE, JVP, Branch::kNone, PAST>), grid, block, 0, s, p);
  };
  if (p.tx.p != nullptr) go(IC<1>{}, IC<NT>{});
  else go(IC<0>{}, IC<0>{});
  return hipGetLastError();
}

template <typename T, typename W>
static hipError_t norm_launch_t(const GatedNormParams& p, bool backward, hipStream_t s) {
  if (p.past_caches) return p.C <= 512 ? norm_launch_s<T, W, true, true>(p, backward, s) : norm_launch_s<T, W, false, true>(p, backward, s);
  return p.C <= 512 ? norm_launch_s<T, W, true, false>(p, backward, s) : norm_launch_s<T, W, false, false>(p, backward, s);
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
