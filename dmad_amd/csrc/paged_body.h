// One workgroup of attention over a paged cache (its description stands with
// paged_attn_kernel), for that kernel and for launches that run it beside other work.
#pragma once

#include "paged_pieces.h"

namespace dmad {

constexpr int kPagedWaves = 4;
constexpr int kStep = 32;  // slots per wave step

// Elements of O, or of a partial: 4 floats to 4 elements.
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4_t x) {
  *(u32x2_t*)p = u32x2_t{Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3])};
}

// Whether one of two packed elements is infinite or not a number.
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
  constexpr uint32_t EXP = sizeof(T) == 2 && __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  return (w & EXP) == EXP || ((w >> 16) & EXP) == EXP;
}

// P = exp2(score - running maximum) <= 1 is rounded to the operand type for its
// product with V alone (off by at most 2^-8 of each in bf16, 2^-11 in fp16; the sums of P stay
// float32). In fp16 it goes in as 2^15 P and O is scaled back with its last
// store: P itself would be subnormal from 14 binary orders below the maximum on
// and zero from 25, and a long tail of equally light slots, whose P all round the
// same way, can be what the output is made of when the heavy slot's V is small.
// The float32 accumulators have room for 2^15 times anything fp16 holds.
template <typename T>
struct PagedP {
  static constexpr float UP = __is_same(T, _Float16) ? 32768.f : 1.f;
};

template <int D>
struct PagedCfg {
  static constexpr int KC = D >= 32 ? D / 32 : 1;   // 32-wide slices of a K row
  static constexpr int VE = D / 16;                 // elements of a V row per lane
  static constexpr int VD = VE >= 2 ? VE / 2 : 1;   // dwords of them
  static constexpr int OP = D + 4;                  // floats per row of O in LDS
};

// A lane's part of one V row.
template <int D>
__device__ __forceinline__ void load_v(const char* base, uint32_t off, uint32_t (&v)[PagedCfg<D>::VD]) {
  const char* p = base + off;
  if constexpr (D == 16) {
    v[0] = *(const uint16_t*)p;
  } else if constexpr (D == 32) {
    v[0] = *(const uint32_t*)p;
  } else if constexpr (D == 64) {
    const u32x2_t x = *(const u32x2_t*)p;
    v[0] = x[0];
    v[1] = x[1];
  } else {
#pragma unroll
    for (int c = 0; c < D / 128; ++c) {
      const i32x4_t x = *(const i32x4_t*)(p + 16 * c);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * c + k] = (uint32_t)x[k];
    }
  }
}

// CAUSAL: rows of different tokens see different slots. `block` of the launch's.
// What the waves leave one another lies in LDS: o(wave), [16][OP], m(wave) and l(wave), [16 NT].
template <typename T, int D, int NT, bool ACC, bool CAUSAL, typename Lds>
__device__ __forceinline__ void paged_attn_body(const PagedAttnParams& p, int block, const Lds& lds) {
  // no contraction but the written ones: a call that accumulates has the outputs
  // of one that does not, bit for bit
#pragma clang fp contract(off)
  using C = PagedCfg<D>;
  const KvPages& kv = p.kv;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  // Blocks are dealt to the 8 XCDs in turn: the row groups of one piece and head
  // are 8 blocks apart, on one XCD, whose L2 then reads K and V once for them.
  const int work = block / (8 * p.row_groups) * 8 + (block & 7), rg = block / 8 % p.row_groups;
  const int hk = work % kv.heads, x = work / kv.heads;
  if (x >= p.splits) return;
  PagedPiece piece(kv, p.splits, x, lane);
  for (; !piece.done(); piece.next()) {  // the same segments in every wave
  const int b = piece.run.b, n = piece.run.n;
  const int first = piece.first_slot(), last = piece.end_slot();
  const int steps = (last - first + kStep - 1) / kStep;
  const int mine = steps > wave ? (steps - wave + kPagedWaves - 1) / kPagedWaves : 0;  // this wave's: wave, wave + 4, ...

  // Q^T, and how many slots each row sees
  i32x4_t qf[NT][C::KC];
  int sees[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (rg * NT + t) * 16 + row;
    const int i = r / p.G, h = hk * p.G + r % p.G;
    sees[t] = r < p.R ? (CAUSAL ? n - (p.S - 1 - i) : n) : 0;
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      qf[t][c] = i32x4_t{0, 0, 0, 0};
      if (r < p.R && c * 32 + g * 8 < D)
        qf[t][c] = *(const i32x4_t*)((const T*)p.q + b * p.qb + i * p.qs + h * p.qh + c * 32 + g * 8);
    }
  }
  // slots below this are seen by every row
  const int all_see = CAUSAL ? n - (p.S - 1) : n;

  const uint32_t koff = (uint32_t)(row * kv.k_sl + g * 8) * 2;
  uint32_t voff[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) voff[v] = (uint32_t)((g * 4 + v) * kv.v_sl + row * C::VE) * 2;

  // Pages of the next 32 steps' halves, one per lane: step lane/2, half lane%2.
  int pages = 0, slots = 0;
  auto look_up = [&](int step) {
    const int j = step + (lane >> 1);
    const int key = first + (wave + kPagedWaves * j) * kStep + (lane & 1) * 16;
    pages = -1;
    slots = 0;
    if (j < mine && key < last) {
      const KvSlot at = kv.locate(b, key);
      pages = at.page;
      slots = at.slot;
    }
  };

  i32x4_t kf[2][C::KC];
  uint32_t vf[8][C::VD];
  auto half = [&](int step, int hh) {
    return KvSlot{__builtin_amdgcn_readlane(pages, 2 * (step & 31) + hh), __builtin_amdgcn_readlane(slots, 2 * (step & 31) + hh)};
  };
  // A half without a page reads page 0, whose 16 first slots exist, and is masked.
  auto readable = [](KvSlot at) { return KvSlot{max(at.page, 0), at.slot}; };
  auto request_k = [&](int step) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const char* base = (const char*)kv.k + 2 * kv.k_offset(readable(half(step, hh)), hk);
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        if constexpr (D == 16) {
          kf[hh][c] = i32x4_t{0, 0, 0, 0};
          if (g < 2) kf[hh][c] = *(const i32x4_t*)(base + koff);
        } else {
          kf[hh][c] = *(const i32x4_t*)(base + koff + c * 64);
        }
      }
    }
  };
  auto request_v = [&](int step) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const char* base = (const char*)kv.v + 2 * kv.v_offset(readable(half(step, hh)), hk);
#pragma unroll
      for (int v = 0; v < 4; ++v) load_v<D>(base, voff[v], vf[hh * 4 + v]);
    }
  };

  float* score_row[NT];  // this lane's row, from its 4 slots of a half on
#pragma unroll
  for (int t = 0; t < NT && ACC; ++t)
    score_row[t] = p.scores + (((int64_t)b * kv.heads + hk) * p.R + (rg * NT + t) * 16 + row) * kv.capacity() + g * 4;

  f32x4_t acc[NT][C::VE];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < C::VE; ++j) acc[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // Q and the page ids have to be here before the loop, on every path to it:
  // with them still on their way the compiler waits, in every step, for all
  // loads in flight
  look_up(0);
  wait_vmem();
  if (mine > 0) {
    request_k(0);
    request_v(0);
  }
  // Whether every row sees every slot of a step, and another step follows.
  auto plain_step = [&](int step) {
    return step + 1 < mine && first + (wave + kPagedWaves * step + 1) * kStep <= min(all_see, last) &&
           half(step, 0).page >= 0 && half(step, 1).page >= 0;  // uniform
  };
  // One step. Those that need no mask, nearly all, request the next one's K and V
  // without a branch around them, so that each product waits for its own
  // operand alone; the others (EDGE) mask what is not there or not seen.
  auto run_step = [&](int step, auto edge) {
    constexpr bool EDGE = edge.value != 0;
    const int key0 = first + (wave + kPagedWaves * step) * kStep;
    const int page[2] = {half(step, 0).page, half(step, 1).page};
    const bool more = !EDGE || step + 1 < mine;

    f32x4_t s[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        s[t][hh] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C::KC; ++c) s[t][hh] = mfma16(kf[hh][c], qf[t][c], s[t][hh], T{});
      }
    if (more) {
      if ((step & 31) == 31) look_up(step + 1);
      request_k(step + 1);
    }

    bool hidden = false;  // an infinity or NaN in V that some row must not see
    if constexpr (EDGE) {
      // slots beyond the sequence, this piece or the row's view, and of missing pages
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int key = key0 + hh * 16 + g * 4 + v;
          const bool there = page[hh] >= 0 && key < last;
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (!(there && key < sees[t])) s[t][hh][v] = -__builtin_inff();
          // V of such slots may hold anything: zero times it must be zero
          if (!there) {
#pragma unroll
            for (int k = 0; k < C::VD; ++k) vf[hh * 4 + v][k] = 0;
          } else if (CAUSAL && key >= all_see) {
#pragma unroll
            for (int k = 0; k < C::VD; ++k) hidden |= any_nonfinite<T>(vf[hh * 4 + v][k]);
          }
        }
      if constexpr (CAUSAL) hidden = __ballot(hidden) != 0;
    }

    i32x4_t pf[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -__builtin_inff();
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          s[t][hh][v] *= p.scale_log2;
          top = fmaxf(top, s[t][hh][v]);
        }
      if constexpr (ACC) {
        if ((rg * NT + t) * 16 + row < p.R) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            if (!EDGE || key0 + hh * 16 < last) *(f32x4_t*)(score_row[t] + key0 + hh * 16) = s[t][hh];
        }
      }
      top = across32<LaneMax>(across16<LaneMax>(top));
      const float up = fmaxf(m[t], top);
      const float base = up == -__builtin_inff() ? 0.f : up;  // nothing seen yet: every p is exp2(-inf)
      if (__ballot(up > m[t]) != 0) {
        const float f = fast_exp2(m[t] - base);
        l[t] *= f;
#pragma unroll
        for (int j = 0; j < C::VE; ++j) acc[t][j] *= f;
        m[t] = up;
      }
      float e[8];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          e[hh * 4 + v] = fast_exp2(s[t][hh][v] - base);
          l[t] += e[hh * 4 + v];
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) pf[t][k] = (int)Elem<T>::pack2(e[2 * k] * PagedP<T>::UP, e[2 * k + 1] * PagedP<T>::UP);
    }

    if (EDGE && CAUSAL && hidden) {
      // Zero times such a value is NaN: token by token, with the slots it does
      // not see zeroed in V, and only its own rows taking the result.
      for (int i = 0; i < p.S; ++i) {
        const int see = all_see + i;
        bool any = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) any |= sees[t] == see;
        if (__ballot(any) == 0) continue;
#pragma unroll
        for (int j = 0; j < C::VE; ++j) {
          auto seen = [&](int e) { return key0 + (e >> 2) * 16 + g * 4 + (e & 3) < see ? vf[e][j >> 1] : 0u; };
          i32x4_t a;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            a[k] = (int)__builtin_amdgcn_perm(seen(2 * k + 1), seen(2 * k), (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const f32x4_t o = mfma16(a, pf[t], acc[t][j], T{});
            if (sees[t] == see) acc[t][j] = o;
          }
          __builtin_amdgcn_sched_barrier(0);  // one column of V at a time: few registers
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < C::VE; ++j) {
        i32x4_t a;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          a[k] = (int)__builtin_amdgcn_perm(vf[2 * k + 1][j >> 1], vf[2 * k][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][j] = mfma16(a, pf[t], acc[t][j], T{});
      }
    }
    if (more) request_v(step + 1);
  };
  for (int step = 0; step < mine; ++step) {
    for (; plain_step(step); ++step) run_step(step, IC<0>{});
    run_step(step, IC<1>{});
  }

  // The waves' results joined through LDS, 16 rows at a time.
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] = across32<LaneAdd>(across16<LaneAdd>(l[t]));
    if (g == 0) {
      lds.m(wave)[t * 16 + row] = m[t];
      lds.l(wave)[t * 16 + row] = l[t];
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t > 0) __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int j = 0; j < C::VE; ++j) lds.o(wave)[row * C::OP + (g * 4 + v) * C::VE + j] = acc[t][j][v] * (1.f / PagedP<T>::UP);
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 64 * kPagedWaves) {
      const int rr = i / (D / 4), d = (i % (D / 4)) * 4;
      const int r = (rg * NT + t) * 16 + rr;
      if (r >= p.R) continue;
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) top = fmaxf(top, lds.m(w)[t * 16 + rr]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      float sum = 0.f;
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) {
        const float f = fast_exp2(lds.m(w)[t * 16 + rr] - base);
        sum = fmaf(f, lds.l(w)[t * 16 + rr], sum);
        const f32x4_t y = *(const f32x4_t*)&lds.o(w)[rr * C::OP + d];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(f, y[k], o[k]);
      }
      if (piece.whole() && !p.keep_parts) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int hq = hk * p.G + r % p.G, tok = r / p.G, Hq = kv.heads * p.G;
        store4<T>((T*)p.o + (((int64_t)b * p.S + tok) * Hq + hq) * D + d, o * inv);
        if (d == 0) {
          const float l2 = base + __builtin_amdgcn_logf(sum);  // log2
          p.lse[((int64_t)b * Hq + hq) * p.S + tok] = sum == 0.f ? -__builtin_inff() : l2 * 0.6931471805599453f;
          if constexpr (ACC) p.lse2[((int64_t)b * kv.heads + hk) * p.R + r] = sum == 0.f ? __builtin_inff() : l2;
        }
      } else {
        const int64_t at = ((int64_t)(x + b) * kv.heads + hk) * p.R + r;
        *(f32x4_t*)(p.part_o + at * D + d) = o;
        if (d == 0) {
          p.part_ml[2 * at] = top;
          p.part_ml[2 * at + 1] = sum;
        }
      }
    }
  }
  if (!piece.last()) __syncthreads();  // the next segment writes the same LDS
  }
}

}  // namespace dmad
