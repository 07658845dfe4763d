// Attention of many query rows over a paged prefix that their sequences share.
//
// The rows of all sequences behind one prefix (their tokens times the query
// heads of a key head) meet K and V as one product, so that the arithmetic
// bounds it: 4 D flops per row and slot for 4 D bytes per slot. paged_attn_kernel
// keeps 16 or 32 rows per workgroup and streams K and V through registers; here a
// workgroup takes 128 rows, 32 per wave, and K and V go through LDS once for all
// four waves:
//   * S^T = K Q^T and O^T += V^T P^T on 32x32x16 MFMAs. Lane l of a wave owns row
//     l % 32; its Q row stays in registers. K's rows are read in perm32 order, so
//     P leaves the score tile as the B operand of the second product.
//   * 32 slots per step in a four-stage ring filled three steps ahead by
//     buffer->LDS requests. A page holds whole runs of 16 slots, so each half of a
//     step has one base: its resource starts there and ends behind the last slot
//     in use, and everything beyond (a missing page: everything) reads as zeros.
//   * V^T is read from the row-major tile by transposing LDS reads.
//   * The softmax of one step runs between the MFMAs of the next one's scores.
// A row's maximum follows lazily (it moves once a score exceeds it by 2^8 in bf16; at
// once in fp16, where P enters as 2^15 P so that light slots keep their precision).
// Scores of slots that are not there are -inf. P is rounded to the operand type for its
// product with V alone (off by at most 2^-8 of each in bf16, 2^-11 in fp16, as in
// paged_attn_kernel); maxima, sums of P and O are float32.
//
// 48 sequences of 4 tokens, 64 query heads over 8 key heads, behind 131072 slots: 0.82
// ms for 8.3e11 flops, 1.0 PFLOP/s (a large matrix product reaches 1.23, plain attention
// of this package 1.04 on the same heads): what is left lies between the MFMAs, the
// softmax's VALU work (about 3 instructions per score and row) foremost.
//
// The line of slots is cut into `splits` pieces (paged_pieces.h); each leaves
// (maximum, sum, O) per row in float32 for prefix_join_kernel.
#include "attn_fwd.h"
#include "paged_body.h"

namespace dmad {

template <int D_>
struct PrefixCfg {
  static constexpr int D = D_;
  static constexpr int NW = 4, BM = kPrefixRows, BN = 32;
  static constexpr int KS = D / 16, DB = D / 32;  // slices of a score, blocks of O^T
  static constexpr int CR = D / 8, ROWB = D * 2;  // 16-byte chunks and bytes of a row
  static constexpr int TILE = BN * ROWB, STAGE = 2 * TILE;
  static constexpr int RPW = BN * CR / 64 / NW;  // 1 KiB requests per tile and wave
  static constexpr int LOADS = 2 * RPW;
  static constexpr int RPR = 64 / CR;  // rows per request
  static constexpr int NOP = KS + 2 * DB;
  static_assert(4 * STAGE <= 160 * 1024 && BM == 32 * NW);
};

template <typename T>
struct PrefixP {
  static constexpr bool HALF = __is_same(T, _Float16);
  static constexpr float SLACK = HALF ? 0.f : 8.f, UP = HALF ? 15.f : 0.f;  // log2
  static constexpr float DOWN = HALF ? 1.f / 32768.f : 1.f;
};

// The ring's stages.
struct PrefixRing {
  lds_char_t *s0, *s1, *s2, *s3;
};

template <typename T, int D>
__device__ __forceinline__ void prefix_rows_body(const PagedAttnParams& p, int block, const PrefixRing& ring) {
  using C = PrefixCfg<D>;
  using PP = PrefixP<T>;
  constexpr int KS = C::KS, DB = C::DB, CR = C::CR, ROWB = C::ROWB, NOP = C::NOP, PF = 4;
  const KvPages& kv = p.kv;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  // the row groups of one piece and head on one XCD, as in paged_attn_kernel
  const int work = block / (8 * p.row_groups) * 8 + (block & 7), rg = block / 8 % p.row_groups;
  const int hk = work % kv.heads, x = work / kv.heads;
  if (x >= p.splits) return;

  // request offsets of a lane inside 16 slots, and LDS read offsets
  uint32_t roff_k[C::RPW], roff_v[C::RPW];
#pragma unroll
  for (int j = 0; j < C::RPW; ++j) {
    const int pch = (wave + j * C::NW) * 64 + lane, row = pch / CR, logical = (pch % CR) ^ trswz<CR>(row & 15);
    roff_k[j] = (uint32_t)((row & 15) * (int64_t)kv.k_sl * 2) + logical * 16;
    roff_v[j] = (uint32_t)((row & 15) * (int64_t)kv.v_sl * 2) + logical * 16;
  }
  // (256-wide heads keep the first ones: slice s lies at kx ^ 32 s, block db at tx ^ 64 db)
  constexpr int NKX = D == 256 ? 1 : KS, NTX = D == 256 ? 1 : DB;
  int kx[NKX], tx[NTX][2];
  {
    const int r = perm32(col), g = lane >> 4, rr = (lane & 15) >> 2, c = lane & 3;
#pragma unroll
    for (int s = 0; s < NKX; ++s) kx[s] = r * ROWB + (((2 * s + half) ^ trswz<CR>(r & 15)) << 4);
#pragma unroll
    for (int db = 0; db < NTX; ++db)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = 8 * (g >> 1) + 4 * hh + rr, chunk = 4 * db + 2 * (g & 1) + (c >> 1);
        tx[db][hh] = row * ROWB + ((chunk ^ trswz<CR>(row & 15)) << 4) + 8 * (c & 1);
      }
  }
  auto k_off = [&](int s) { return NKX == 1 ? kx[0] ^ (32 * s) : kx[s % NKX]; };
  auto v_off = [&](int db, int hh) { return NTX == 1 ? tx[0][hh] ^ (64 * db) : tx[db % NTX][hh]; };
  // re-defined at each step: stage and offset fold into the LDS instructions
  auto pin = [&]() {
#pragma unroll
    for (int s = 0; s < NKX; ++s) asm volatile("" : "+v"(kx[s]));
#pragma unroll
    for (int db = 0; db < NTX; ++db) asm volatile("" : "+v"(tx[db][0]), "+v"(tx[db][1]));
  };
  auto stage = [&](auto kk) -> lds_char_t* {
    constexpr int k = decltype(kk)::value % 4;
    if constexpr (k == 0) return ring.s0;
    else if constexpr (k == 1) return ring.s1;
    else if constexpr (k == 2) return ring.s2;
    else return ring.s3;
  };

  PagedPiece piece(kv, p.splits, x, lane);
  for (; !piece.done(); piece.next()) {  // the same segments in every wave
    const int b = piece.run.b, first = piece.first_slot(), last = piece.end_slot();
    const int ntiles = (last - first + C::BN - 1) / C::BN;
    const int r = rg * C::BM + wave * 32 + col;  // this lane's row
    i32x4_t qreg[KS];
    {
      const int i = r / p.G, h = hk * p.G + r % p.G;
      const T* q = (const T*)p.q + b * p.qb + i * p.qs + h * p.qh + half * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qreg[s] = i32x4_t{0, 0, 0, 0};
        if (r < p.R) qreg[s] = *(const i32x4_t*)(q + s * 16);
      }
    }
    // Where 32 steps' halves begin and what of them is there, one half per lane (step
    // lane/2, half lane%2): addresses of K's and V's 16 rows, bytes up to the last row
    // in use (none for a missing page). And whether all 16 slots of each are there, of
    // these steps and of the 32 before.
    uint64_t k_at = 0, v_at = 0;
    uint32_t k_bytes = 0, v_bytes = 0;
    uint64_t whole = 0, whole_before = 0;
    int window = -1;
    auto look_up = [&](int j0) {
      const int j = j0 + (lane >> 1), key = first + j * C::BN + (lane & 1) * 16;
      KvSlot at{-1, 0};
      if (j < ntiles && key < last) at = kv.locate(b, key);
      const int there = at.page < 0 ? 0 : min(last - key, 16);
      const KvSlot from{max(at.page, 0), at.slot};
      k_at = (uint64_t)kv.k + 2 * kv.k_offset(from, hk);
      v_at = (uint64_t)kv.v + 2 * kv.v_offset(from, hk);
      k_bytes = there ? (uint32_t)(((there - 1) * kv.k_sl + D) * 2) : 0;
      v_bytes = there ? (uint32_t)(((there - 1) * kv.v_sl + D) * 2) : 0;
      whole_before = whole;
      whole = __ballot(there == 16);
      window = j0 >> 5;
    };
    auto lane_of = [](uint32_t v, int at) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
    // request li of step j
    auto request = [&](lds_char_t* st, int j, int li) {
      const int jj = li >> 1, i = wave + jj * C::NW, at = 2 * (j & 31) + i * C::RPR / 16;
      const uint64_t from = li & 1 ? v_at : k_at;
      const uint64_t base = (uint64_t)lane_of((uint32_t)(from >> 32), at) << 32 | lane_of((uint32_t)from, at);
      const __amdgpu_buffer_rsrc_t rows = make_rsrc((const void*)base, lane_of(li & 1 ? v_bytes : k_bytes, at));
      buf_load16_lds(rows, st + (li & 1 ? C::TILE : 0) + i * 1024, li & 1 ? roff_v[jj] : roff_k[jj], 0);
    };

    f32x16_t oacc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) oacc[d][v] = 0.f;
    const f32x16_t zero16 = {};
    float m_i = kLowest, l_i = 0.f;

    // Softmax of one step in micro-steps: value v is slot 16 (v >> 3) + 8 half + (v & 7).
    constexpr int NMICRO = 18;
    struct Soft {
      float mx, alpha, neg_m, ls, pv;
      bool moved;
    };
    auto soft_micro = [&](int u, Soft& sm, const f32x16_t& sc, i32x4_t (&pk)[2]) {
      if (u == 0) {
        const float a = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), b2 = fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7]));
        const float c2 = fmaxf(fmaxf(sc[8], sc[9]), fmaxf(sc[10], sc[11])), d2 = fmaxf(fmaxf(sc[12], sc[13]), fmaxf(sc[14], sc[15]));
        sm.mx = fmaxf(fmaxf(a, b2), fmaxf(c2, d2));
        sm.ls = 0.f;
      } else if (u == 1) {
        sm.mx = fmaxf(sm.mx, other_half(sm.mx)) * p.scale_log2;
        // row by row: whether its neighbours in the wave move changes nothing for one that stays
        const bool move = sm.mx > m_i + PP::SLACK;
        sm.moved = __builtin_amdgcn_ballot_w64(move) != 0;
        const float m_new = move ? sm.mx : m_i;
        sm.alpha = fast_exp2(m_i - m_new);
        m_i = m_new;
        sm.neg_m = PP::UP - m_new;
      } else {
        const int v = u - 2;
        const float pe = fast_exp2(fmaf(sc[v], p.scale_log2, sm.neg_m));
        sm.ls += pe;
        if (v & 1) pk[v >> 3][(v & 7) >> 1] = (int)Elem<T>::pack2(sm.pv, pe);
        else sm.pv = pe;
      }
    };
    // a step some of whose slots are not there
    auto mask = [&](f32x16_t& sc, int i) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int key = first + i * C::BN + hh * 16;
        const int there = kv.locate(b, key).page < 0 ? 0 : min(max(last - key, 0), 16);
#pragma unroll
        for (int v = 0; v < 8; ++v)
          if (8 * half + v >= there) sc[8 * hh + v] = -__builtin_inff();
      }
    };
    auto all_there = [&](int i) { return (((i >> 5) == window ? whole : whole_before) >> (2 * (i & 31)) & 3) == 3; };

    auto load_op = [&](const lds_char_t* s_next, const lds_char_t* s_cur, int o) -> i32x4_t {
      if (o < KS) return *(lds_i32x4_t*)(s_next + k_off(o));
      const int t = (o - KS) / DB, db = (o - KS) % DB;
      const lds_char_t* base = s_cur + C::TILE + t * 16 * ROWB;
      const u32x2_t lo = lds_read_tr16(base + v_off(db, 0)), hi = lds_read_tr16(base + v_off(db, 1));
      return i32x4_t{(int)lo[0], (int)lo[1], (int)hi[0], (int)hi[1]};
    };
    auto mfma_op = [&](int o, i32x4_t a, f32x16_t& sn, const i32x4_t (&pk)[2]) {
      if (o < KS) sn = mfma32(a, qreg[o], o == 0 ? zero16 : sn, T());
      else oacc[(o - KS) % DB] = mfma32(a, pk[(o - KS) / DB], oacc[(o - KS) % DB], T());
    };
    auto rescale = [&](float alpha) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        asm volatile("" : "+v"(oacc[d]));  // not to be computed ahead of the branch around it
#pragma unroll
        for (int v = 0; v < 16; ++v) oacc[d][v] *= alpha;
      }
    };
    // step i: scores of step i + 1 with the softmax of step i between them, then its
    // products with V, the requests of step i + 3 between those
    auto step = [&](auto kk, int i, f32x16_t& sc, f32x16_t& sn) {
      constexpr int k = decltype(kk)::value;
      if (((i + 3) & 31) == 0) look_up(i + 3);
      ring_sync<C::LOADS>();  // step i + 1 has landed, step i + 2 may be in flight
      pin();
      const lds_char_t *s_next = stage(IC<k + 1>{}), *s_cur = stage(IC<k>{});
      lds_char_t* s_req = stage(IC<k + 3>{});
      if (!all_there(i)) mask(sc, i);
      i32x4_t opr[PF];
#pragma unroll
      for (int o = 0; o < PF; ++o) opr[o] = load_op(s_next, s_cur, o);
      Soft sm;
      i32x4_t pk[2];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int o = 0; o < KS; ++o) {
        mfma_op(o, opr[o % PF], sn, pk);
        if (o + PF < NOP) opr[o % PF] = load_op(s_next, s_cur, o + PF);
#pragma unroll
        for (int u = o * NMICRO / KS; u < (o + 1) * NMICRO / KS; ++u) soft_micro(u, sm, sc, pk);
        __builtin_amdgcn_sched_barrier(0);
      }
      l_i = l_i * sm.alpha + sm.ls;
      asm volatile("" : "+v"(pk[0]), "+v"(pk[1]), "+v"(l_i));  // used here: the softmax stays above
      if (sm.moved) rescale(sm.alpha);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int o = KS; o < NOP; ++o) {
        mfma_op(o, opr[o % PF], sn, pk);
        if (o + PF < NOP) opr[o % PF] = load_op(s_next, s_cur, o + PF);
#pragma unroll
        for (int li = 0; li < C::LOADS; ++li)
          if (KS + li * 2 * DB / C::LOADS == o) request(s_req, i + 3, li);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto last_step = [&](auto kk, int i, f32x16_t& sc) {
      const lds_char_t* s_cur = stage(kk);
      if (!all_there(i)) mask(sc, i);
      Soft sm;
      i32x4_t pk[2];
#pragma unroll
      for (int u = 0; u < NMICRO; ++u) soft_micro(u, sm, sc, pk);
      l_i = l_i * sm.alpha + sm.ls;
      rescale(sm.alpha);
      f32x16_t none;
#pragma unroll
      for (int o = KS; o < NOP; ++o) mfma_op(o, load_op(s_cur, s_cur, o), none, pk);
    };

    if (ntiles > 0) {
      look_up(0);
      wait_vmem();
      // steps 0, 1, 2; a step beyond the last reads zeros
#pragma unroll
      for (int li = 0; li < C::LOADS; ++li) request(stage(IC<0>{}), 0, li);
#pragma unroll
      for (int li = 0; li < C::LOADS; ++li) request(stage(IC<1>{}), 1, li);
#pragma unroll
      for (int li = 0; li < C::LOADS; ++li) request(stage(IC<2>{}), 2, li);
      ring_sync<2 * C::LOADS>();
      f32x16_t sa, sb;
      {
        const lds_char_t* s0 = stage(IC<0>{});
        const i32x4_t none[2] = {};
#pragma unroll
        for (int o = 0; o < KS; ++o) mfma_op(o, load_op(s0, s0, o), sa, none);
      }
      int i = 0;
      for (; i + 4 < ntiles; i += 4) {
        step(IC<0>{}, i, sa, sb);
        step(IC<1>{}, i + 1, sb, sa);
        step(IC<2>{}, i + 2, sa, sb);
        step(IC<3>{}, i + 3, sb, sa);
      }
      const int rest = ntiles - i;  // 1..4
      if (rest >= 2) step(IC<0>{}, i, sa, sb);
      if (rest >= 3) step(IC<1>{}, i + 1, sb, sa);
      if (rest >= 4) step(IC<2>{}, i + 2, sa, sb);
      if (rest == 1) last_step(IC<0>{}, i, sa);
      else if (rest == 2) last_step(IC<1>{}, i + 1, sb);
      else if (rest == 3) last_step(IC<2>{}, i + 2, sa);
      else last_step(IC<3>{}, i + 3, sb);
    }
    ring_sync<0>();  // nothing in flight, and nobody reads the ring any more

    // lane (row col, half) holds elements 32 db + 8 jj + 4 half + 0..3
    const float l = (l_i + other_half(l_i)) * PP::DOWN;
    if (r < p.R) {
      const int64_t at = ((int64_t)(x + b) * kv.heads + hk) * p.R + r;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          f32x4_t o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = oacc[d][4 * jj + e] * PP::DOWN;
          *(f32x4_t*)(p.part_o + at * D + 32 * d + 8 * jj + 4 * half) = o;
        }
      if (half == 0) {
        p.part_ml[2 * at] = m_i;
        p.part_ml[2 * at + 1] = l;
      }
    }
  }
}

// The prefix's pass and, with the launch's last blocks, that over the sequences' own
// slots, which starts wherever the first one's workgroups end: 16 rows at a time, or many
// rows like the prefix's where every row sees every slot.
enum class OwnPass { kAll, kCausal, kRows };

template <typename T, int D, OwnPass OWN>
__global__ __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) void prefix_rows_kernel(PagedAttnParams shared, PagedAttnParams p,
                                                                                         int rows_blocks) {
  using C = PrefixCfg<D>;
  __shared__ __attribute__((aligned(1024))) char stg0[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char stg1[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char stg2[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char stg3[C::STAGE];
  constexpr int O = 16 * PagedCfg<D>::OP;
  static_assert((O + 32) * 4 <= C::STAGE);
  struct Lds {  // a wave's part is one stage
    __device__ __forceinline__ float* o(int w) const { return (float*)(w == 0 ? stg0 : w == 1 ? stg1 : w == 2 ? stg2 : stg3); }
    __device__ __forceinline__ float* m(int w) const { return o(w) + O; }
    __device__ __forceinline__ float* l(int w) const { return o(w) + O + 16; }
  };
  const PrefixRing ring{(lds_char_t*)stg0, (lds_char_t*)stg1, (lds_char_t*)stg2, (lds_char_t*)stg3};
  const int own = (int)blockIdx.x - rows_blocks;
  if (own >= 0) {
    if constexpr (OWN != OwnPass::kRows) paged_attn_body<T, D, 1, false, OWN == OwnPass::kCausal>(p, own, Lds{});
    else prefix_rows_body<T, D>(p, own, ring);
  } else {
    prefix_rows_body<T, D>(shared, (int)blockIdx.x, ring);
  }
}

template <typename T, int D>
static hipError_t prefix_rows_d(const PagedAttnParams& shared, const PagedAttnParams& p, hipStream_t s) {
  auto blocks = [](const PagedAttnParams& a) { return (a.splits * a.kv.heads + 7) / 8 * 8 * a.row_groups; };
  const int rows = blocks(shared);
  const dim3 grid((unsigned)(rows + blocks(p))), block(256);
  if (prefix_own_rows(p.R, p.causal, p.S)) hipLaunchKernelGGL((prefix_rows_kernel<T, D, OwnPass::kRows>), grid, block, 0, s, shared, p, rows);
  else if (p.causal && p.S > 1) hipLaunchKernelGGL((prefix_rows_kernel<T, D, OwnPass::kCausal>), grid, block, 0, s, shared, p, rows);
  else hipLaunchKernelGGL((prefix_rows_kernel<T, D, OwnPass::kAll>), grid, block, 0, s, shared, p, rows);
  return hipGetLastError();
}

template <typename T>
static hipError_t prefix_rows_t(const PagedAttnParams& shared, const PagedAttnParams& p, int D, hipStream_t s) {
  switch (D) {
    case 64: return prefix_rows_d<T, 64>(shared, p, s);
    case 128: return prefix_rows_d<T, 128>(shared, p, s);
    case 256: return prefix_rows_d<T, 256>(shared, p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_prefix_rows(const PagedAttnParams& shared, const PagedAttnParams& p, int dtype, int D, hipStream_t s) {
  return dtype == 0 ? prefix_rows_t<__bf16>(shared, p, D, s) : prefix_rows_t<_Float16>(shared, p, D, s);
}

// More than 16 rows per key head (one row tile of paged_attn_kernel) go here, whose
// K and V pass through LDS once for 128 rows. 40 heads of 128 over 32760 slots: 135
// against 136 us for 24 rows, 136 - 144 for 32, 140 - 167 for 48, 159 - 304 for 128; 64-wide
// heads 80 - 81 us for 32 rows, 105 - 169 for 128; 16 heads of 256 113 - 121 for 17, 150 - 389
// for 128. Up to 16 rows 124 to 134 there against 130 to 135 here.
bool prefix_rows_takes(int D, int64_t R) { return (D == 64 || D == 128 || D == 256) && R > kPrefixRowsFrom; }
// Own slots of more than 32 rows whose tokens all see the same: 4 continuations by a frame
// of 1560 tokens (12 heads, 1560 to 3120 own slots, behind 4000) 322 us against 737 with 16
// rows per workgroup, 40 rows of 8 x 40 heads (1000 to 2000) 95 - 117, 48 of 4 x 16 64-wide
// ones 32 - 29. Causal blocks go 16 at a time: the LDS kernel masks slots for all rows
// alike, not row by row. The same frame, causal, takes 897 us.
bool prefix_own_rows(int64_t R, bool causal, int64_t S) { return !(causal && S > 1) && R > kPrefixOwnRowsFrom; }
// Workgroups per CU that the cut aims at; a CU holds 3, 2, 1. Fewer are fewer pieces to
// leave and join, and leave room for the own slots: 128-wide heads 159 us with one
// against 205 with two for 128 rows as above (88 - 98 for 96 samples behind two
// prefixes); 64-wide ones 111, 105 and 107 us with one, two and three.
int prefix_rows_resident(int D) { return D == 64 ? 2 : 1; }

}  // namespace dmad
