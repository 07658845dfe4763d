// Parameters and launchers of the operators around a block's attention: gate,
// residual and norm in one pass, and rotations by position.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dmad {

// One [B, S, C] operand by strides (elements), rows contiguous.
struct NormRows {
  const void* p;  // null: absent
  int64_t b, s;
};
// One [B, F, C] vector per group of tokens, rows contiguous.
struct NormVec {
  const void* p;  // null: absent
  int64_t b, f;
};

constexpr int kNormSums = 3;  // sums over tokens that the small operands' gradients are made of

struct GatedNormParams {
  NormRows x, y;             // y absent: no branch
  NormRows tx, ty;           // tangents (forward), or the gradients of x' and of n (backward; either may be absent)
  NormVec gate, scale, shift, tgate, tscale, tshift;
  const void *weight, *bias, *post;  // [C], or null
  void *xo, *txo, *no, *tno;         // contiguous [B, S, C]; backward: xo, txo are the gradients of x and y
  int B, S, F, T, C;         // T = S / F tokens per group
  int64_t rows;              // B S
  int layer;                 // the norm subtracts the mean
  float eps, rs;             // rs: scale of the branch
  int past_caches;           // more than the caches hold
  int split;                 // workgroups per group of tokens
  // backward: either each leaves its sums in partial
  // [B F split][kNormSums][C], or (partial null, split 1) writes the group's
  // gradients itself
  float* partial;
  void *dgate, *dscale, *dshift;     // contiguous [B, F, C], or null
  void *dweight, *dbias, *dpost;     // [C], or null
};

// Widest rows.
constexpr int kNormMaxC = 8192;
// Waves of a workgroup for rows of C channels, waves that a pass aims at, and waves per CU in
// a round of the forward and of the backward pass. The backward's are what a CU holds; of the
// forward's it would hold 32 (28 with a norm after the branch; with tangents 20 and 16).
int norm_waves(int C);
enum class NormPass { kForward, kTangent, kBackward };
constexpr int kNormFwdWaves = 40960, kNormTangentWaves = 65536, kNormFwdHeld = 20, kNormBwdHeld = 16;

hipError_t launch_gated_norm(const GatedNormParams& p, int dtype, int wdtype, hipStream_t s);
// Workgroups per group of tokens.
int gated_norm_split(int64_t groups, int T, int C, NormPass pass);
hipError_t launch_gated_norm_bwd(const GatedNormParams& p, int dtype, int wdtype, hipStream_t s);

// ---------------------------------------------------------------- rotations by position

// One of q, k in [B, S, H, D] by strides (elements).
struct RotaryOperand {
  const void* x;  // null: absent (H = 0)
  const void* t;  // tangent, or null
  void* out;      // contiguous [B, S, H, D]
  void* tout;
  int64_t xb, xs, xh, tb, ts, th;
  int H;
};

struct RotaryParams {
  RotaryOperand op[2];  // q, k
  const void* positions;       // [B, S] by strides, int32 or int64
  int64_t pos_b, pos_s;
  int pos64;
  const double* frequencies;   // [R / 2] radians per position
  int B, S, D, R;
  int64_t tokens;              // B S
  int interleaved;             // pairs of neighbours; otherwise element i with i + R / 2
  float factor;                // times the sines and cosines
  int sign;                    // -1: the transposed rotation
  int vec;                     // elements per access: 8, 4, 2 or 1 (rotary_vec)
  int per_head, per_token;     // units (two accesses each) of a head's row, and of a token
  uint32_t head_mul;           // x / per_head = (x head_mul) >> 32 for x < per_token * tile (0: per_head is 1)
  uint32_t token_mul;          // and by per_token
  int tile;                    // tokens per workgroup
  int past_caches;
};
// Sets vec, per_head, per_token, the multipliers and tile from the rest; `align`
// is the largest power of two that divides every operand's strides, offsets and
// addresses, in elements. False where the sizes are too large.
bool rotary_plan(RotaryParams& p, int elem_size, int align);
hipError_t launch_rotary(const RotaryParams& p, int dtype, hipStream_t s);

}  // namespace dmad
