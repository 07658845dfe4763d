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
#include "paged_body.h"

namespace dmad {

template <int D, int NT>
struct PagedOwnLds {
  float sm_o[kPagedWaves][16][PagedCfg<D>::OP];
  float sm_m[kPagedWaves][NT * 16], sm_l[kPagedWaves][NT * 16];
  __device__ __forceinline__ float* o(int w) const { return (float*)&sm_o[w][0][0]; }
  __device__ __forceinline__ float* m(int w) const { return (float*)sm_m[w]; }
  __device__ __forceinline__ float* l(int w) const { return (float*)sm_l[w]; }
};

template <typename T, int D, int NT, bool ACC, bool CAUSAL>
__global__ __launch_bounds__(64 * kPagedWaves, D * NT <= 128 ? 2 : 1) void paged_attn_kernel(PagedAttnParams p) {
  __shared__ PagedOwnLds<D, NT> lds;
  paged_attn_body<T, D, NT, ACC, CAUSAL>(p, (int)blockIdx.x, lds);
}

// Two caches in one launch: a prefix and, with the last blocks, the sequences' own
// slots behind it, of up to 16 rows per key head. (Four sequences of 1 to 64 slots
// behind 257: 18 us per call, of which the host's share is all, against 21.)
template <typename T, int D, bool CAUSAL>
__global__ __launch_bounds__(64 * kPagedWaves, D <= 128 ? 2 : 1) void prefix_pair_kernel(PagedAttnParams shared, PagedAttnParams p,
                                                                                        int shared_blocks) {
  __shared__ PagedOwnLds<D, 1> lds;
  const int own = (int)blockIdx.x - shared_blocks;
  if (own < 0) paged_attn_body<T, D, 1, false, false>(shared, (int)blockIdx.x, lds);
  else paged_attn_body<T, D, 1, false, CAUSAL>(p, own, lds);
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
  __shared__ float sm_o[WAYS][ROWS][D], sm_m[WAYS][ROWS], sm_l[WAYS][ROWS];
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

static int paged_blocks(const PagedAttnParams& p) { return (p.splits * p.kv.heads + 7) / 8 * 8 * p.row_groups; }

template <typename T, int D, bool ACC, bool CAUSAL>
static void paged_launch_rows(const PagedAttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)paged_blocks(p)), block(64 * kPagedWaves);
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

// Rows of all sequences from which one strand joins a row's pieces: enough to fill the
// chip. 14 us against 31 for 12288 rows of six pieces, 8 against 13 for 96 sequences of 32 with seventeen each;
// fewer rows need the strands where their pieces are many.
constexpr int kJoinRowsFrom = 2048;

template <typename T, int D>
static hipError_t prefix_launch_d(const PagedAttnParams& shared, const PagedAttnParams& p, hipStream_t s) {
  hipError_t e;
  if (prefix_rows_takes(D, shared.R)) {
    e = launch_prefix_rows(shared, p, __is_same(T, _Float16) ? 1 : 0, D, s);
  } else if (paged_row_tiles(D, shared.R) == 1) {
    const int first = paged_blocks(shared);
    const dim3 grid((unsigned)(first + paged_blocks(p))), block(64 * kPagedWaves);
    if (p.causal && p.S > 1) hipLaunchKernelGGL((prefix_pair_kernel<T, D, true>), grid, block, 0, s, shared, p, first);
    else hipLaunchKernelGGL((prefix_pair_kernel<T, D, false>), grid, block, 0, s, shared, p, first);
    e = hipGetLastError();
  } else if ((e = paged_launch<T, D, false>(shared, s)) == hipSuccess) {
    e = paged_launch<T, D, false>(p, s);
  }
  if (e != hipSuccess) return e;
  constexpr int LANES = D / 4, ALL = 256 / LANES;
  const int rows = p.kv.heads * p.R;
  if (rows * p.kv.B >= kJoinRowsFrom) {
    hipLaunchKernelGGL((prefix_join_kernel<T, D, 1>), dim3((unsigned)(p.kv.B * ((rows + ALL - 1) / ALL))), dim3(256), 0, s, shared, p);
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
