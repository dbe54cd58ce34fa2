// Which rows a workgroup of the packed-sequence attention owns.  Needs nothing but a wave's ballots and lane reads, so a
// test can run it on the host.
#pragma once

namespace ogv {

// Tile slot t of sequence-major tiles of BM rows: the slots of sequence b begin at cu[b] * G / BM + b, which
// leaves every sequence room for ceil(len * G / BM) tiles, needs no table and bounds their number by
// M * G / BM + B.  A whole wave searches (64 probes a round).  Offsets are clamped to [0, M], the first one
// to 0.  The search takes them for sorted; where they are not it may end at a sequence whose slots do not hold t, so
// what it found counts only if the tile has rows: no offset array leads outside the tensors.
struct Seq {
  int b, tile, start, len, start2, len2;   // rows of the tiled side, rows of the other side
};
__device__ __forceinline__ int cu_at(const int* __restrict__ cu, int b, int M) {
  return b <= 0 ? 0 : min(max(cu[b], 0), M);
}
// cu / M: the side that is tiled, G * its rows in tiles of BM; cu2 / M2: the other side.  False: the slot has no rows
// (those behind the last sequence are in the last one's tiles).
__device__ __forceinline__ bool find_tile(const int* __restrict__ cu, const int* __restrict__ cu2, int B, int M, int M2, int G, int BM,
                                          int t, int lane, Seq& s) {
  int at, end, at2, end2;
  if (B < 64) {   // the offsets fit a wave: one load each, everything else from registers
    const int x = cu_at(cu, min(lane, B), M), y = cu_at(cu2, min(lane, B), M2);
    const bool ok = lane < B && (int)(((long)x * G) / BM) + lane <= t;
    const int hits = __popcll(__ballot(ok));
    s.b = __builtin_amdgcn_readfirstlane(hits > 0 ? hits - 1 : 0);
    at = __builtin_amdgcn_readlane(x, s.b), end = __builtin_amdgcn_readlane(x, s.b + 1);
    at2 = __builtin_amdgcn_readlane(y, s.b), end2 = __builtin_amdgcn_readlane(y, s.b + 1);
  } else {
    int lo = 0, n = B;   // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + 63) >> 6, idx = lo + lane * step;
      const bool ok = lane * step < n && (int)(((long)cu_at(cu, idx, M) * G) / BM) + idx <= t;
      const int hits = __popcll(__ballot(ok));
      const int j = hits > 0 ? hits - 1 : 0;
      n = min(step, n - j * step);
      lo += j * step;
    }
    s.b = __builtin_amdgcn_readfirstlane(lo);
    at = __builtin_amdgcn_readfirstlane(cu_at(cu, s.b, M)), end = __builtin_amdgcn_readfirstlane(cu_at(cu, s.b + 1, M));
    at2 = __builtin_amdgcn_readfirstlane(cu_at(cu2, s.b, M2)), end2 = __builtin_amdgcn_readfirstlane(cu_at(cu2, s.b + 1, M2));
  }
  s.start = at, s.len = max(end - at, 0), s.start2 = at2, s.len2 = max(end2 - at2, 0);
  s.tile = t - ((int)(((long)at * G) / BM) + s.b);
  return s.tile >= 0 && (long)s.tile * BM < (long)(s.b == B - 1 ? M - at : s.len) * G;
}

}  // namespace ogv
