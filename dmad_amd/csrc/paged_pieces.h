// How paged attention's work is cut over the sequences of a cache, on the device.
#pragma once
#include "kv_cache.h"
#include "lanes.h"

namespace dmad {

// Running sum over the lanes, the lane's own included: within rows of 16
// lanes, then the row before's last lane, then lane 31's.
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = scan_step<0x111, 0xf>(x);  // from 1, 2, 4 and 8 lanes below
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  x = scan_step<0x118, 0xf>(x);
  x = scan_step<0x142, 0xa>(x);  // lane 15 to rows 1, 3
  x = scan_step<0x143, 0xc>(x);  // lane 31 to rows 2, 3
  return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// How the work is cut. Each sequence is a run of 128-slot tiles (one at least),
// the runs follow one another, and piece x takes tiles [x chunk, (x + 1) chunk)
// of that line, whatever sequences they belong to: equal work for every
// workgroup of a ragged batch. A piece's part of a sequence is a segment; with
// the pieces and the sequences both in order, x + b numbers the segments
// without a clash. Every read of a length may find another value where a caller
// writes them meanwhile: pieces and sequences are kept in range whatever the
// lengths were, so that such a call gives wrong results and nothing worse.
__device__ __forceinline__ int paged_tiles(int n) { return max(1, (n + kPagedTile - 1) / kPagedTile); }

// Lengths of all sequences, a lane each; the first 64 are read once.
struct PagedLengths {
  const KvPages& kv;
  int lane, first;
  __device__ __forceinline__ PagedLengths(const KvPages& k, int l) : kv(k), lane(l), first(l < k.B ? k.length(l) : 0) {}
  // length of sequence b0 + lane (b0 a multiple of 64), and its tiles (0 beyond the last)
  __device__ __forceinline__ int at(int b0) const { return b0 == 0 ? first : b0 + lane < kv.B ? kv.length(b0 + lane) : 0; }
  __device__ __forceinline__ int tiles(int b0) const { return b0 + lane < kv.B ? paged_tiles(at(b0)) : 0; }
  __device__ __forceinline__ int total() const {
    int t = 0;
    for (int b0 = 0; b0 < kv.B; b0 += 64) t += tiles(b0);
    return wave_total(t);
  }
};

// A sequence and where its run of tiles begins.
struct PagedRun {
  int b, n, base;
};
__device__ __forceinline__ PagedRun run_of_tile(const PagedLengths& len, int tile) {
  int before = 0;
  for (int b0 = 0; b0 < len.kv.B; b0 += 64) {
    // one reading: a tile is never before its sequence's first
    const int n = len.at(b0), end = before + wave_scan(b0 + len.lane < len.kv.B ? paged_tiles(n) : 0);
    const uint64_t past = __ballot(end > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int m = __builtin_amdgcn_readlane(n, at);
      return PagedRun{b0 + at, m, __builtin_amdgcn_readlane(end, at) - paged_tiles(m)};
    }
    before = __builtin_amdgcn_readlane(end, 63);
  }
  return PagedRun{len.kv.B, 0, before};  // beyond the last tile: not asked for
}
__device__ __forceinline__ PagedRun run_of_sequence(const PagedLengths& len, int b) {
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) before += b0 + len.lane < b ? len.tiles(b0) : 0;
  return PagedRun{b, len.kv.length(b), wave_total(before)};
}

// Piece x, segment by segment.
struct PagedPiece {
  const KvPages& kv;
  PagedRun run;
  int tile, stop, end;  // this segment's first tile, the piece's end, the segment's end
  __device__ __forceinline__ PagedPiece(const KvPages& k, int splits, int x, int lane) : kv(k), run{0, 0, 0}, tile(0), stop(0), end(0) {
    const PagedLengths len(kv, lane);
    const int total = len.total(), chunk = max(1, (total + splits - 1) / splits);
    tile = x * chunk;
    stop = min(total, tile + chunk);
    if (tile < stop) run = run_of_tile(len, tile);
    if (run.b >= kv.B) stop = tile;
    end = min(stop, run.base + paged_tiles(run.n));
  }
  __device__ __forceinline__ bool done() const { return tile >= stop; }
  __device__ __forceinline__ bool last() const { return end >= stop; }
  __device__ __forceinline__ void next() {
    tile = end;
    if (run.b + 1 >= kv.B) stop = tile;
    if (done()) return;
    run = PagedRun{run.b + 1, kv.length(run.b + 1), run.base + paged_tiles(run.n)};
    end = min(stop, run.base + paged_tiles(run.n));
  }
  // the segment's slots, and whether it is the whole sequence
  __device__ __forceinline__ int first_slot() const { return (tile - run.base) * kPagedTile; }
  __device__ __forceinline__ int end_slot() const { return min(run.n, (end - run.base) * kPagedTile); }
  __device__ __forceinline__ bool whole() const { return tile == run.base && end == run.base + paged_tiles(run.n); }
};

}  // namespace dmad
