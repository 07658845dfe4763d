// Parameters and launchers of the per-head norm and rotation, the paged
// key-value cache, its attention and its eviction.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kv_pages.h"

namespace dmad {

// One of q, k, v in [B, S, H, D] by strides (elements).
struct QkOperand {
  const void* x;  // null: absent (H = 0)
  const void* t;  // tangent (forward) or the gradient of the output (backward)
  const void* w;  // [D] weight, or null
  void* out;      // contiguous [B, S, H, D]; in an append null for k and v, which go to the pages
  void* tout;
  int64_t xb, xs, xh, tb, ts, th;
  int H, passes;  // heads, and wave passes that cover them
};

struct QkNormRopeParams {
  QkOperand op[3];  // q, k, v
  const float* freqs;      // angles: [rows][D/2], or null
  int64_t freqs_b;         // stride of a batch entry (0: shared)
  int freqs_rows;          // rows of the table (append: indexed by position)
  int B, S, D;
  int passes, per_wave;    // passes per token, and per wave
  int64_t units;           // waves' worth of work: tokens * ceil(passes / per_wave)
  float eps;
  bool past_caches;        // tangents, backward: more than the caches hold (qk_past_caches)
  bool by_sequence;        // append: a workgroup per sequence (qk_append_split)
  float* partial;          // backward: [blocks][2][D] sums of the weights' gradients
  KvPages kv;              // append
};

enum class QkMode { kPrimal, kTangent, kAppend };
// Whether a call that reads and writes that many bytes does so past the caches.
bool qk_past_caches(int64_t bytes);
// Decides whether an append runs a workgroup per sequence, and cuts it so.
void qk_append_split(QkNormRopeParams& p);
hipError_t launch_qk_norm_rope(const QkNormRopeParams& p, int dtype, int wdtype, QkMode mode, hipStream_t s);

// Blocks of the backward pass (rows of `partial`).
int64_t qk_norm_rope_bwd_blocks(int64_t units);
hipError_t launch_qk_norm_rope_bwd(const QkNormRopeParams& p, int dtype, int wdtype, void* dwq, void* dwk, hipStream_t s);

// ---------------------------------------------------------------- attention
constexpr int kPagedTile = 128;  // slots per workgroup step: 32 for each of 4 waves

struct PagedAttnParams {
  KvPages kv;
  const void* q;           // [B, S, Hq, D] by strides (elements)
  int64_t qb, qs, qh;
  void* o;                 // contiguous [B, S, Hq, D]
  float* lse;              // [B, Hq, S]
  int S, G, R;             // new tokens, query heads per key head, rows per key head (S * G)
  int row_groups;          // workgroups that share a key head's rows
  int causal;
  int splits;              // pieces of all sequences together, per head and row group
  float scale_log2;
  float* part_o;           // [splits + B][heads][R][D], or null: no sequence has more than a tile
  float* part_ml;          // [splits + B][heads][R][2]: maximum (log2 domain) and sum
  float* scores;           // [B][heads][R][M P], log2 domain; null: weights are not accumulated
  float* lse2;             // [B][heads][R], log2 domain (with scores)
  int keep_parts;          // every segment stays in part_o and part_ml, for a join with another cache's
};
// Rows of a workgroup of paged attention at head dim D, of R rows per key head.
int paged_attn_rows(int D, int R);
// Its workgroups per CU that a launch aims at.
int paged_attn_resident(int D);
hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, int D, hipStream_t s);
// The same for many rows per key head (prefix_rows.hip), partials only: rows per
// workgroup, whether a call is one of these, and its workgroups per CU.
constexpr int kPrefixRows = 128;
constexpr int kPrefixRowsFrom = 16;
bool prefix_rows_takes(int D, int64_t R);
// Whether such a call's own slots, of R rows per key head, are one too.
constexpr int kPrefixOwnRowsFrom = 32;
bool prefix_own_rows(int64_t R, bool causal, int64_t S);
int prefix_rows_resident(int D);
hipError_t launch_prefix_rows(const PagedAttnParams& shared, const PagedAttnParams& p, int dtype, int D, hipStream_t s);
// Attention over prefixes and over each sequence's own slots behind its prefix:
// sequence b of p follows prefix b / (p.kv.B / shared.kv.B), whose rows in
// `shared` are those of its sequences one after the other. Both keep_parts.
hipError_t launch_prefix_attn(const PagedAttnParams& shared, const PagedAttnParams& p, int dtype, int D, hipStream_t s);

// ---------------------------------------------------------------- eviction
// Up to this many slots per sequence the selection keeps its keys in LDS (128 KiB).
constexpr int kSelectInLds = 32 * 1024;

struct KvEvictParams {
  KvPages kv;
  int D, keep, recent, sink;
  int max_moves;       // bound on the slots that move, per sequence and head
  uint32_t* keys;      // [B][heads][M P], for more than kSelectInLds slots
  int32_t* moves;      // [B][heads][2][max_moves]: destination slots, source slots
  int32_t* counts;     // [B][heads] slots that move; 0 where nothing is evicted
  int32_t* ends;       // [B] lengths afterwards
};
hipError_t launch_kv_evict(const KvEvictParams& p, hipStream_t s);

}  // namespace dmad
