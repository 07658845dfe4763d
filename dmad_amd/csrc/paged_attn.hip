// Attention of one or a few new tokens per sequence over a paged key-value
// cache, split over the cache's length and joined.
//
// Row r of key head h (S new tokens times the G query heads that share it):
//   s_j = scale q_r . k_j,  p_j = exp(s_j - lse_r),  o_r = sum_j p_j v_j
// over the slots j the row sees, in one pass with the running maximum and sum.
// Optionally weight_j += sum_r p_j for every slot.
//
// Bound by reading K and V once: 5.9-6.2 TB/s (a 4 GiB copy reaches 4.7, reads
// and writes together): 112 us for one token over 40 heads of 32760 slots,
// 1.33 ms for 4 tokens of 64 query heads over 16 sequences of about 125000
// slots (8.2 GB). A wave takes 32 slots at a time and needs no LDS and no
// barrier for them:
//   * S^T = K Q^T on 16x16x32 MFMAs. K's rows go from memory straight into the
//     A operand (lane = slot, 16 bytes of its row), Q^T stays in registers.
//   * In the C layout a lane holds slots 4 g + v (g = lane / 16) of both 16-slot
//     halves for one row: exactly the B operand of O^T = V^T P^T when its 8
//     k-values are numbered half, v. P goes from VALU to MFMA in registers.
//   * V's rows are loaded for those same 8 slots, D/16 elements per lane, so a
//     row is one contiguous access of 16 lanes; the lane then holds an
//     8 x D/16 block, and pairing its 16-bit halves (one v_perm per two
//     elements) gives V^T's A operands. Column m of MFMA j is element
//     m D/16 + j of the row, so a lane's results are D/16 neighbours.
// The next step's K is requested when this step's scores are done, and V when
// its products are. The arithmetic hides behind the bytes: 16 rows per key head
// take 76 us where 4 take 66 (355 MB). K and V are read once per 16 or 32 rows, by
// workgroups that meet in one L2: up to 32 rows cost what one does (118-121 us for
// 40 heads of 32760 slots), from about 64 on the arithmetic bounds (143 us for 64,
// 243 for 128, 2.34 ms for 1560: 450 TFLOP/s).
//
// Split: the launch has `splits` pieces of equal work for all sequences
// together; the device finds from the lengths which tiles are whose, so ragged
// batches load the chip evenly and a captured graph follows the lengths (48
// sequences of 1 to 16000 slots: 66 us against 74 with pieces that end where a
// sequence does, 60 for equal lengths; the 16 sequences above 1.33 ms against
// 1.59). A sequence that lies in several pieces leaves (maximum, sum, O) of each
// in float32 and a second kernel joins them in order; one that lies in a single
// piece is finished by the first kernel.
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

// CAUSAL: rows of different tokens see different slots.
template <typename T, int D, int NT, bool ACC, bool CAUSAL>
__global__ __launch_bounds__(64 * kPagedWaves, D * NT <= 128 ? 2 : 1) void paged_attn_kernel(PagedAttnParams p) {
  // no contraction but the written ones: a call that accumulates has the outputs
  // of one that does not, bit for bit
#pragma clang fp contract(off)
  using C = PagedCfg<D>;
  __shared__ float sm_o[kPagedWaves][16][C::OP];
  __shared__ float sm_m[kPagedWaves][NT * 16], sm_l[kPagedWaves][NT * 16];
  const KvPages& kv = p.kv;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  // Blocks are dealt to the 8 XCDs in turn: the row groups of one piece and head
  // are 8 blocks apart, on one XCD, whose L2 then reads K and V once for them.
  const int work = (int)blockIdx.x / (8 * p.row_groups) * 8 + ((int)blockIdx.x & 7), rg = (int)blockIdx.x / 8 % p.row_groups;
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
      sm_m[wave][t * 16 + row] = m[t];
      sm_l[wave][t * 16 + row] = l[t];
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t > 0) __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int j = 0; j < C::VE; ++j) sm_o[wave][row][(g * 4 + v) * C::VE + j] = acc[t][j][v] * (1.f / PagedP<T>::UP);
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 64 * kPagedWaves) {
      const int rr = i / (D / 4), d = (i % (D / 4)) * 4;
      const int r = (rg * NT + t) * 16 + rr;
      if (r >= p.R) continue;
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) top = fmaxf(top, sm_m[w][t * 16 + rr]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      float sum = 0.f;
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) {
        const float f = fast_exp2(sm_m[w][t * 16 + rr] - base);
        sum = fmaf(f, sm_l[w][t * 16 + rr], sum);
        const f32x4_t y = *(const f32x4_t*)&sm_o[w][rr][d];
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

// Joins the pieces of one row: D/4 lanes per piece, the pieces over the rest.
template <typename T, int D, bool ACC>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p) {
#pragma clang fp contract(off)  // as in paged_attn_kernel
  constexpr int LANES = D / 4, STRANDS = 256 / LANES;
  __shared__ float sm_o[STRANDS][D], sm_m[STRANDS], sm_l[STRANDS];
  const KvPages& kv = p.kv;
  const int r = (int)blockIdx.x % p.R, hk = ((int)blockIdx.x / p.R) % kv.heads, b = (int)blockIdx.x / (p.R * kv.heads);
  const PagedLengths len(kv, lane_id());
  const int chunk = max(1, (len.total() + p.splits - 1) / p.splits);
  const PagedRun run = run_of_sequence(len, b);
  const int first = run.base / chunk, last = min((run.base + paged_tiles(run.n) - 1) / chunk, p.splits - 1);  // pieces
  if (first == last) return;  // finished
  const int strand = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  float m = -__builtin_inff(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i = first + strand; i <= last; i += STRANDS) {
    const int64_t at = ((int64_t)(i + b) * kv.heads + hk) * p.R + r;
    const float mi = p.part_ml[2 * at], li = p.part_ml[2 * at + 1];
    const f32x4_t oi = *(const f32x4_t*)(p.part_o + at * D + d);
    const float up = fmaxf(m, mi), base = up == -__builtin_inff() ? 0.f : up;
    const float f = fast_exp2(m - base), fi = fast_exp2(mi - base);
    l = l * f + li * fi;
    o = o * f + oi * fi;
    m = up;
  }
  *(f32x4_t*)&sm_o[strand][d] = o;
  if (d == 0) {
    sm_m[strand] = m;
    sm_l[strand] = l;
  }
  __syncthreads();
  if (strand != 0) return;
  float top = -__builtin_inff();
  for (int i = 0; i < STRANDS; ++i) top = fmaxf(top, sm_m[i]);
  const float base = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  o = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < STRANDS; ++i) {
    const float f = fast_exp2(sm_m[i] - base);
    sum = fmaf(f, sm_l[i], sum);
    o = o + *(const f32x4_t*)&sm_o[i][d] * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int hq = hk * p.G + r % p.G, tok = r / p.G, Hq = kv.heads * p.G;
  store4<T>((T*)p.o + (((int64_t)b * p.S + tok) * Hq + hq) * D + d, o * inv);
  if (d == 0) {
    const float l2 = base + __builtin_amdgcn_logf(sum);
    p.lse[((int64_t)b * Hq + hq) * p.S + tok] = sum == 0.f ? -__builtin_inff() : l2 * 0.6931471805599453f;
    if constexpr (ACC) p.lse2[((int64_t)b * kv.heads + hk) * p.R + r] = sum == 0.f ? __builtin_inff() : l2;
  }
}

// Joins a row's pieces over a prefix that sequences share with those over its own
// slots: `shared` has a run of n = B / P sequences' rows per prefix, and row r of
// sequence b is row (b % n) R + r of prefix b / n. D/4 lanes hold a row, WAYS such
// strands share its pieces, and a workgroup has 256 / (D/4 WAYS) rows of one
// sequence; each strand requests four pieces at a time.
template <typename T, int D, int WAYS>
__global__ __launch_bounds__(256) void prefix_join_kernel(PagedAttnParams shared, PagedAttnParams p) {
  constexpr int LANES = D / 4, ROWS = 256 / (LANES * WAYS), AHEAD = 4;
  __shared__ float sm_o[WAYS > 1 ? WAYS : 1][ROWS][D], sm_m[WAYS][ROWS], sm_l[WAYS][ROWS];
  const int rows = p.kv.heads * p.R, groups = (rows + ROWS - 1) / ROWS;  // of a sequence
  const int b = (int)blockIdx.x / groups;
  const int strand = threadIdx.x / LANES, way = strand / ROWS, slot = strand % ROWS, d = (threadIdx.x % LANES) * 4;
  const int at_row = ((int)blockIdx.x % groups) * ROWS + slot;
  const bool there = at_row < rows;
  const int hk = min(at_row, rows - 1) / p.R, r = min(at_row, rows - 1) % p.R;
  const int n = p.kv.B / shared.kv.B;
  float m = -__builtin_inff(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  auto gather = [&](const PagedAttnParams& a, int seq, int row, int turn) {
    const PagedLengths len(a.kv, lane_id());
    const int chunk = max(1, (len.total() + a.splits - 1) / a.splits);
    const PagedRun run = run_of_sequence(len, seq);
    const int first = run.base / chunk, last = min((run.base + paged_tiles(run.n) - 1) / chunk, a.splits - 1);
    for (int i = first + (way + turn) % WAYS; i <= last; i += AHEAD * WAYS) {
      float mi[AHEAD], li[AHEAD];
      f32x4_t oi[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int64_t at = ((int64_t)(min(i + j * WAYS, last) + seq) * a.kv.heads + hk) * a.R + row;
        mi[j] = a.part_ml[2 * at];
        li[j] = a.part_ml[2 * at + 1];
        oi[j] = *(const f32x4_t*)(a.part_o + at * D + d);
      }
      float up = m;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i + j * WAYS > last) mi[j] = -__builtin_inff(), li[j] = 0.f, oi[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        up = fmaxf(up, mi[j]);
      }
      const float base = up == -__builtin_inff() ? 0.f : up, f = fast_exp2(m - base);
      l *= f;
      o *= f;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float fi = fast_exp2(mi[j] - base);
        l = l + li[j] * fi;
        o = o + oi[j] * fi;
      }
      m = up;
    }
  };
  gather(shared, b / n, (b % n) * p.R + r, 0);
  gather(p, b, r, WAYS / 2);  // from the other end of the strands, which few pieces leave idle
  if constexpr (WAYS > 1) {
    *(f32x4_t*)&sm_o[way][slot][d] = o;
    if (d == 0) {
      sm_m[way][slot] = m;
      sm_l[way][slot] = l;
    }
    __syncthreads();
    if (way != 0) return;
    for (int i = 0; i < WAYS; ++i) m = fmaxf(m, sm_m[i][slot]);
    const float base = m == -__builtin_inff() ? 0.f : m;
    l = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < WAYS; ++i) {
      const float f = fast_exp2(sm_m[i][slot] - base);
      l = fmaf(f, sm_l[i][slot], l);
      o = o + *(const f32x4_t*)&sm_o[i][slot][d] * f;
    }
  }
  if (!there) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int hq = hk * p.G + r % p.G, tok = r / p.G, Hq = p.kv.heads * p.G;
  store4<T>((T*)p.o + (((int64_t)b * p.S + tok) * Hq + hq) * D + d, o * inv);
  if (d == 0) {
    const float l2 = (m == -__builtin_inff() ? 0.f : m) + __builtin_amdgcn_logf(l);
    p.lse[((int64_t)b * Hq + hq) * p.S + tok] = l == 0.f ? -__builtin_inff() : l2 * 0.6931471805599453f;
  }
}

// weight_j += sum over the rows of exp2(score - lse2), a tile of slots at a time
// and a slot per thread. The line of tiles is cut finer than for the attention:
// short sequences follow one another through the same wait for every one (17
// -> 10 us for 48 of them). In one launch with the joins, each row's lse found
// again from the pieces, both took what they take one after the other.
__global__ __launch_bounds__(kPagedTile) void paged_weight_kernel(PagedAttnParams p, int splits) {
  const KvPages& kv = p.kv;
  const int hk = (int)blockIdx.x % kv.heads;
  for (PagedPiece piece(kv, splits, (int)blockIdx.x / kv.heads, lane_id()); !piece.done(); piece.next()) {
    const int b = piece.run.b, last = piece.end_slot();
    const int64_t bh = (int64_t)b * kv.heads + hk;
    for (int key = piece.first_slot() + (int)threadIdx.x; key < last; key += kPagedTile) {
      const KvSlot at = kv.locate(b, key);
      const float* s = p.scores + bh * p.R * kv.capacity() + key;
      float sum = 0.f;
      for (int r0 = 0; r0 < p.R; r0 += 8) {
        float x[8], lse[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = min(r0 + j, p.R - 1);
          lse[j] = r0 + j < p.R ? p.lse2[bh * p.R + r] : __builtin_inff();
          x[j] = s[(int64_t)r * kv.capacity()];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += fast_exp2(x[j] - lse[j]);
      }
      if (at.page >= 0) kv.weight[kv.index(at, hk)] += sum;
    }
  }
}
// Its workgroups: up to 32 per CU.
constexpr int kPagedWeightGroups = 8192;

// Two row tiles share one reading of K and V where their registers allow, which
// those of 256-wide heads do not: 119 us against 136 with one tile each for 32 rows
// of 40 heads of 32760 slots, 140 against 233 for 64 rows; 50 against 55 us for 32
// rows of 64-wide heads (8 sequences of 16000 slots). 256-wide heads pay: 158 us for
// 40 rows where 16 take 103 (526 MB).
static int paged_row_tiles(int D, int R) { return R <= 16 || D == 256 ? 1 : 2; }
int paged_attn_rows(int D, int R) { return 16 * paged_row_tiles(D, R); }
// Workgroups per CU that the cut aims at. Four waves with 16 KiB of K and V on
// their way each (128-wide heads) keep a CU's share of the memory busy: one, two
// and three took 115, 116, 119 us for 40 heads of 32760 slots, 634, 643, 642 for 8
// sequences of 120000 and 80, 84, 81 for 48 ragged ones; 51, 52, 57 at 256-wide heads.
// Narrower rows gain by two where they are many: 96, 89, 89 us for 32-wide heads, 96,
// 98, 94 for 64-wide ones.
int paged_attn_resident(int D) { return D >= 128 ? 1 : 2; }

template <typename T, int D, bool ACC, bool CAUSAL>
static void paged_launch_rows(const PagedAttnParams& p, hipStream_t s) {
  const int work = (p.splits * p.kv.heads + 7) / 8 * 8;
  const dim3 grid((unsigned)(work * p.row_groups)), block(64 * kPagedWaves);
  if constexpr (D < 256) {
    if (paged_row_tiles(D, p.R) == 2) {
      hipLaunchKernelGGL((paged_attn_kernel<T, D, 2, ACC, CAUSAL>), grid, block, 0, s, p);
      return;
    }
  }
  hipLaunchKernelGGL((paged_attn_kernel<T, D, 1, ACC, CAUSAL>), grid, block, 0, s, p);
}

template <typename T, int D, bool ACC>
static hipError_t paged_launch(const PagedAttnParams& p, hipStream_t s) {
  if (p.causal && p.S > 1) paged_launch_rows<T, D, ACC, true>(p, s);
  else paged_launch_rows<T, D, ACC, false>(p, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.part_o != nullptr && !p.keep_parts) {
    hipLaunchKernelGGL((paged_join_kernel<T, D, ACC>), dim3((unsigned)(p.kv.B * p.kv.heads * p.R)), dim3(256), 0, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if constexpr (ACC) {
    const int splits = max(p.splits, kPagedWeightGroups / p.kv.heads);
    hipLaunchKernelGGL(paged_weight_kernel, dim3((unsigned)(splits * p.kv.heads)), dim3(kPagedTile), 0, s, p, splits);
    e = hipGetLastError();
  }
  return e;
}

template <typename T, int D>
static hipError_t paged_launch_d(const PagedAttnParams& p, hipStream_t s) {
  return p.scores != nullptr ? paged_launch<T, D, true>(p, s) : paged_launch<T, D, false>(p, s);
}

template <typename T>
static hipError_t paged_launch_t(const PagedAttnParams& p, int D, hipStream_t s) {
  switch (D) {
    case 16: return paged_launch_d<T, 16>(p, s);
    case 32: return paged_launch_d<T, 32>(p, s);
    case 64: return paged_launch_d<T, 64>(p, s);
    case 128: return paged_launch_d<T, 128>(p, s);
    case 256: return paged_launch_d<T, 256>(p, s);
  }
  return hipErrorInvalidValue;
}

constexpr int kJoinRowsFrom = 2048, kJoinWays = 1;

template <typename T, int D>
static hipError_t prefix_launch_d(const PagedAttnParams& shared, const PagedAttnParams& p, hipStream_t s) {
  hipError_t e = prefix_rows_takes(D, shared.R) ? launch_prefix_rows(shared, __is_same(T, _Float16) ? 1 : 0, D, s)
                                                : paged_launch<T, D, false>(shared, s);
  if (e != hipSuccess || (e = paged_launch<T, D, false>(p, s)) != hipSuccess) return e;
  constexpr int LANES = D / 4, ALL = 256 / LANES;
  const int rows = p.kv.heads * p.R;
  if (rows * p.kv.B >= kJoinRowsFrom) {
    constexpr int WAYS = kJoinWays;
    hipLaunchKernelGGL((prefix_join_kernel<T, D, WAYS>), dim3((unsigned)(p.kv.B * ((rows * WAYS + ALL - 1) / ALL))), dim3(256), 0, s, shared, p);
  } else {
    hipLaunchKernelGGL((prefix_join_kernel<T, D, ALL>), dim3((unsigned)(p.kv.B * rows)), dim3(256), 0, s, shared, p);
  }
  return hipGetLastError();
}

template <typename T>
static hipError_t prefix_launch_t(const PagedAttnParams& shared, const PagedAttnParams& p, int D, hipStream_t s) {
  switch (D) {
    case 16: return prefix_launch_d<T, 16>(shared, p, s);
    case 32: return prefix_launch_d<T, 32>(shared, p, s);
    case 64: return prefix_launch_d<T, 64>(shared, p, s);
    case 128: return prefix_launch_d<T, 128>(shared, p, s);
    case 256: return prefix_launch_d<T, 256>(shared, p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_prefix_attn(const PagedAttnParams& shared, const PagedAttnParams& p, int dtype, int D, hipStream_t s) {
  return dtype == 0 ? prefix_launch_t<__bf16>(shared, p, D, s) : prefix_launch_t<_Float16>(shared, p, D, s);
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, int D, hipStream_t s) {
  return dtype == 0 ? paged_launch_t<__bf16>(p, D, s) : paged_launch_t<_Float16>(p, D, s);
}

}  // namespace dmad
