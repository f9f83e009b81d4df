// How coli_cuda_delta_prompt cuts packed prompts into launches and passes, so that the
// records between its two kernels stay within a fixed workspace (host code, no HIP).
#pragma once

#include <stddef.h>

namespace sw {

constexpr int kChunk = 64;                           // tokens of a chunk
constexpr size_t kDeltaRecords = (size_t)512 << 20;  // bytes of a pass's records

inline long long chunks_of(int rows) { return ((long long)rows + kChunk - 1) / kChunk; }

// Sequences of a launch, `most` at most: a chunk of each fits the workspace, or it is one
// sequence, whose chunk may be larger by itself.
inline int delta_sequences(int most, size_t chunk_bytes) {
  const size_t fit = kDeltaRecords / chunk_bytes;
  return fit < 1 ? 1 : fit < (size_t)most ? (int)fit : most;
}

// Of n sequences, longest first, those that have a chunk number `first`.
inline int delta_live(const int *rows, int n, long long first) {
  int live = 0;
  while (live < n && chunks_of(rows[live]) > first) live++;
  return live;
}

// Chunks of each sequence in the pass that begins at chunk `first`: the most whose
// records fit, a sequence counted only as far as it goes (127 one-token prompts beside
// one of 8,191 are one pass, not 64 of two chunks each).  0 where none is left.
inline long long delta_pass(const int *rows, int n, long long first, size_t chunk_bytes) {
  const int live = delta_live(rows, n, first);
  if (live == 0) return 0;
  const long long fit = (long long)(kDeltaRecords / chunk_bytes);
  long long lo = 1, hi = chunks_of(rows[0]) - first;
  while (lo < hi) {
    const long long mid = (lo + hi + 1) / 2;
    long long records = 0;
    for (int s = 0; s < live; s++) {
      const long long left = chunks_of(rows[s]) - first;
      records += left < mid ? left : mid;
    }
    if (records <= fit)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

}  // namespace sw
