// Attention of one or a few new tokens per sequence over a paged key-value
// cache, split over the cache's length and joined.
//
// Row r of key head h (S new tokens times the G query heads that share it):
//   s_j = scale q_r . k_j,  p_j = exp(s_j - lse_r),  o_r = sum_j p_j v_j
// over the slots j the row sees, in one pass with the running maximum and sum.
// Optionally weight_j += sum_r p_j for every slot.
//
// Bound by reading K and V once. A wave takes 32 slots at a time and needs no
// LDS and no barrier for them:
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
// The next step's K is requested when this step's scores are done, and V
// when its products are.
//
// Split: the launch aims at `splits` pieces for all sequences together; the
// device turns that into a number of 128-slot tiles per piece from the lengths
// it finds, so ragged batches load the chip evenly and a captured graph
// follows the lengths. Each piece leaves (maximum, sum, O) in float32 and a
// second kernel joins them in order. A sequence of one piece is finished by
// the first kernel.
#include "kv_cache.h"
#include "lanes.h"

namespace dmad {

constexpr int kPagedWaves = 4;
constexpr int kStep = 32;  // slots per wave step

__device__ __forceinline__ int wave_sum_int(int x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ int wave_scan_int(int x, int lane) {  // inclusive
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  return x;
}

// How the sequences are cut: tiles per piece, from all lengths.
__device__ __forceinline__ int paged_tiles(int n) { return max(1, (n + kPagedTile - 1) / kPagedTile); }
__device__ __forceinline__ int paged_chunk(const KvPages& kv, int splits, int lane) {
  int tiles = 0;
  for (int b = lane; b < kv.B; b += 64) tiles += paged_tiles(kv.length(b));
  tiles = wave_sum_int(tiles);
  return max(1, (tiles + splits - 1) / splits);
}

struct PagedPiece {
  int b, n;          // sequence and its length; b < 0: no such piece
  int index, count;  // this piece among the sequence's, and how many it has
  int first;         // number of its first piece among all
  int chunk;         // tiles per piece
};

// Piece `x` of all sequences in order (every wave finds it for itself).
__device__ __forceinline__ PagedPiece find_piece(const KvPages& kv, int splits, int x, int lane) {
  PagedPiece r{-1, 0, 0, 0, 0, 0};
  r.chunk = paged_chunk(kv, splits, lane);
  int before = 0;
  for (int b0 = 0; b0 < kv.B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < kv.B ? kv.length(b) : 0;
    const int mine = b < kv.B ? (paged_tiles(n) + r.chunk - 1) / r.chunk : 0;
    const int end = before + wave_scan_int(mine, lane);
    const uint64_t past = __ballot(end > x);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      r.b = b0 + at;
      r.n = __builtin_amdgcn_readlane(n, at);
      r.count = __builtin_amdgcn_readlane(mine, at);
      r.first = __builtin_amdgcn_readlane(end, at) - r.count;
      r.index = x - r.first;
      return r;
    }
    before = __builtin_amdgcn_readlane(end, 63);
  }
  return r;
}

// The pieces of sequence b.
__device__ __forceinline__ PagedPiece pieces_of(const KvPages& kv, int splits, int b, int lane) {
  PagedPiece r{b, kv.length(b), 0, 0, 0, 0};
  r.chunk = paged_chunk(kv, splits, lane);
  int first = 0;
  for (int i = lane; i < b; i += 64) first += (paged_tiles(kv.length(i)) + r.chunk - 1) / r.chunk;
  r.first = wave_sum_int(first);
  r.count = (paged_tiles(r.n) + r.chunk - 1) / r.chunk;
  return r;
}

// Elements of O, or of a partial: 4 floats to 4 elements.
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4_t x) {
  *(u32x2_t*)p = u32x2_t{Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3])};
}

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

template <typename T, int D, int NT, bool ACC>
__global__ __launch_bounds__(64 * kPagedWaves, 2) void paged_attn_kernel(PagedAttnParams p) {
  using C = PagedCfg<D>;
  __shared__ float sm_o[kPagedWaves][16][C::OP];
  __shared__ float sm_m[kPagedWaves][NT * 16], sm_l[kPagedWaves][NT * 16];
  const KvPages& kv = p.kv;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int rg = (int)blockIdx.x % p.row_groups, hk = ((int)blockIdx.x / p.row_groups) % kv.heads;
  const int x = (int)blockIdx.x / (p.row_groups * kv.heads);
  const PagedPiece piece = find_piece(kv, p.splits, x, lane);
  if (piece.b < 0) return;  // the whole workgroup
  const int b = piece.b, n = piece.n;
  const int first = piece.index * piece.chunk * kPagedTile;
  // a sequence of several pieces has fewer tiles than int holds
  const int last = piece.index + 1 == piece.count ? n : first + piece.chunk * kPagedTile;
  const int steps = (last - first + kStep - 1) / kStep;
  const int mine = steps > wave ? (steps - wave + kPagedWaves - 1) / kPagedWaves : 0;  // this wave's: wave, wave + 4, ...

  // Q^T, and how many slots each row sees
  i32x4_t qf[NT][C::KC];
  int sees[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (rg * NT + t) * 16 + row;
    const int i = r / p.G, h = hk * p.G + r % p.G;
    sees[t] = r < p.R ? (p.causal ? n - (p.S - 1 - i) : n) : 0;
#pragma unroll
    for (int c = 0; c < C::KC; ++c) {
      qf[t][c] = i32x4_t{0, 0, 0, 0};
      if (r < p.R && c * 32 + g * 8 < D)
        qf[t][c] = *(const i32x4_t*)((const T*)p.q + b * p.qb + i * p.qs + h * p.qh + c * 32 + g * 8);
    }
  }
  // slots below this are seen by every row
  const int all_see = p.causal ? n - (p.S - 1) : n;

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

  f32x4_t acc[NT][C::VE];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < C::VE; ++j) acc[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  if (mine > 0) {
    look_up(0);
    request_k(0);
    request_v(0);
  }
  for (int step = 0; step < mine; ++step) {
    const int key0 = first + (wave + kPagedWaves * step) * kStep;
    const int page[2] = {half(step, 0).page, half(step, 1).page};
    const bool whole = key0 + kStep <= min(all_see, last) && page[0] >= 0 && page[1] >= 0;  // uniform

    f32x4_t s[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        s[t][hh] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C::KC; ++c) s[t][hh] = mfma16(kf[hh][c], qf[t][c], s[t][hh], T{});
      }
    const bool more = step + 1 < mine;
    if (more) {
      if ((step & 31) == 31) look_up(step + 1);
      request_k(step + 1);
    }

    if (!whole) {
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
          }
        }
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
        const int r = (rg * NT + t) * 16 + row;
        if (r < p.R) {
          float* out = p.scores + (((int64_t)b * kv.heads + hk) * p.R + r) * kv.capacity();
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            if (key0 + hh * 16 < last) *(f32x4_t*)(out + key0 + hh * 16 + g * 4) = s[t][hh];
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
      // rounded to the operand type for the product alone: the sum keeps float32
#pragma unroll
      for (int k = 0; k < 4; ++k) pf[t][k] = (int)Elem<T>::pack2(e[2 * k], e[2 * k + 1]);
    }

#pragma unroll
    for (int j = 0; j < C::VE; ++j) {
      i32x4_t a;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        a[k] = (int)__builtin_amdgcn_perm(vf[2 * k + 1][j >> 1], vf[2 * k][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][j] = mfma16(a, pf[t], acc[t][j], T{});
    }
    if (more) request_v(step + 1);
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
      for (int j = 0; j < C::VE; ++j) sm_o[wave][row][(g * 4 + v) * C::VE + j] = acc[t][j][v];
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
      if (piece.count == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int hq = hk * p.G + r % p.G, tok = r / p.G, Hq = kv.heads * p.G;
        store4<T>((T*)p.o + (((int64_t)b * p.S + tok) * Hq + hq) * D + d, o * inv);
        if (d == 0) {
          const float l2 = base + __builtin_amdgcn_logf(sum);  // log2
          p.lse[((int64_t)b * Hq + hq) * p.S + tok] = sum == 0.f ? -__builtin_inff() : l2 * 0.6931471805599453f;
          if constexpr (ACC) p.lse2[((int64_t)b * kv.heads + hk) * p.R + r] = sum == 0.f ? __builtin_inff() : l2;
        }
      } else {
        const int64_t at = ((int64_t)x * kv.heads + hk) * p.R + r;
        *(f32x4_t*)(p.part_o + at * D + d) = o;
        if (d == 0) {
          p.part_ml[2 * at] = top;
          p.part_ml[2 * at + 1] = sum;
        }
      }
    }
  }
}

// Joins the pieces of one row: D/4 lanes per piece, the pieces over the rest.
template <typename T, int D, bool ACC>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p) {
  constexpr int LANES = D / 4, STRANDS = 256 / LANES;
  __shared__ float sm_o[STRANDS][D], sm_m[STRANDS], sm_l[STRANDS];
  const KvPages& kv = p.kv;
  const int r = (int)blockIdx.x % p.R, hk = ((int)blockIdx.x / p.R) % kv.heads, b = (int)blockIdx.x / (p.R * kv.heads);
  const PagedPiece piece = pieces_of(kv, p.splits, b, lane_id());
  if (piece.count == 1) return;  // finished
  const int strand = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  float m = -__builtin_inff(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i = strand; i < piece.count; i += STRANDS) {
    const int64_t at = ((int64_t)(piece.first + i) * kv.heads + hk) * p.R + r;
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

// weight_j += sum over the rows of exp2(score - lse2), 4 slots per thread.
__global__ __launch_bounds__(256) void paged_weight_kernel(PagedAttnParams p) {
  const KvPages& kv = p.kv;
  const int hk = (int)blockIdx.y % kv.heads, b = (int)blockIdx.y / kv.heads;
  const int key = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
  if (key >= kv.length(b)) return;  // a group of 4 slots never leaves its page
  const KvSlot at = kv.locate(b, key);
  if (at.page < 0) return;
  const int64_t bh = (int64_t)b * kv.heads + hk;
  const float* s = p.scores + bh * p.R * kv.capacity() + key;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int r = 0; r < p.R; ++r) {
    const float lse = p.lse2[bh * p.R + r];
    const f32x4_t x = *(const f32x4_t*)(s + (int64_t)r * kv.capacity());
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] += fast_exp2(x[k] - lse);
  }
  float* w = kv.weight + kv.index(at, hk);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (key + k < kv.length(b)) w[k] += sum[k];
}

// Two row tiles share one reading of K and V where their registers leave two
// waves per SIMD (not for 256-wide heads).
static int paged_row_tiles(int D, int R) { return R > 16 && D <= 128 ? 2 : 1; }
int paged_attn_rows(int D, int R) { return 16 * paged_row_tiles(D, R); }

template <typename T, int D, bool ACC>
static hipError_t paged_launch(const PagedAttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.max_splits * p.kv.heads * p.row_groups)), block(64 * kPagedWaves);
  if (paged_row_tiles(D, p.R) == 1) {
    hipLaunchKernelGGL((paged_attn_kernel<T, D, 1, ACC>), grid, block, 0, s, p);
  } else if constexpr (D <= 128) {
    hipLaunchKernelGGL((paged_attn_kernel<T, D, 2, ACC>), grid, block, 0, s, p);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.part_o != nullptr) {
    hipLaunchKernelGGL((paged_join_kernel<T, D, ACC>), dim3((unsigned)(p.kv.B * p.kv.heads * p.R)), dim3(256), 0, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if constexpr (ACC) {
    const dim3 wgrid((unsigned)((p.kv.M * p.kv.P + 1023) / 1024), (unsigned)(p.kv.B * p.kv.heads));
    hipLaunchKernelGGL(paged_weight_kernel, wgrid, dim3(256), 0, s, p);
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

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, int D, hipStream_t s) {
  return dtype == 0 ? paged_launch_t<__bf16>(p, D, s) : paged_launch_t<_Float16>(p, D, s);
}

}  // namespace dmad
