// Arithmetic of the packed-sequence attention that the kernels and the host share and that needs no GPU: division by
// multiplication, tile numbers, a row's token within a tile, and the cut of a list's chunks into key ranges. Plain C++, so that a
// host program can include it by itself and check the same lines that the kernels run.
#pragma once
#include <cmath>
#include <cstdint>

#if defined(__HIP__)
#define ES_RULE __host__ __device__ __forceinline__
#else
#define ES_RULE inline
#endif

namespace es {

// x / d for 0 <= x < 2^31 by one multiplication: mul = ceil(2^(32 + sh) / d) with 2^sh < d <= 2^(sh + 1), whose error
// mul * d - 2^(32 + sh) < d <= 2^(sh + 1) keeps x * error under 2^(32 + sh). d = 1: mul = 0.
struct FastDiv {
  unsigned mul;
  int sh;
};
inline FastDiv fast_div(int d) {
  if (d <= 1) return FastDiv{0u, 0};
  int sh = 0;
  while ((2 << sh) < d) ++sh;
  return FastDiv{(unsigned)(((1ull << (32 + sh)) + d - 1) / d), sh};
}
ES_RULE int divide(FastDiv f, int x) {
  return f.mul == 0 ? x : (int)((unsigned)(((uint64_t)(unsigned)x * f.mul) >> 32) >> f.sh);
}

// Tile numbers: a sequence that starts at row `start` (of one of the token tensors) has those from first_tile on; a launch has
// tile_numbers of them.
template <int M>
ES_RULE int first_tile(int start, int G, int b) {
  return start * G / M + b;
}
template <int M>
ES_RULE long long tile_numbers(int B, int T, int G) {
  return (long long)T * G / M + B + 1;
}

// The token of a list's row, both counted from the first token of a tile of 64 rows; half: the row + 1/2. (Exact: rows up to
// G + 63, G up to 4096, the nearest border 1 / (2 G) away.)
ES_RULE int token_of(float half, float inv_g) { return (int)(half * inv_g); }

// ceil(x / y) of positive values by y's reciprocal: up to one in 2^22 off on either side, which moves a range's border but
// leaves the plan the same on every wave
ES_RULE float parts(float x, float inv_y) { return ceilf(x * inv_y - 1e-5f); }

// A list's ranges a tile and chunks a range, `per` chunks a range or more; inv: reciprocal of a float.
struct Cut {
  float ranges, size;
  template <class Inverse>
  ES_RULE Cut(int tiles, int chunks, int rows, float per, Inverse inv) {
    ranges = fmaxf(parts((float)chunks, inv(fmaxf(per, rows <= 32 ? 4.0f : 8.0f))), 1.0f);
    size = tiles > 0 ? parts((float)chunks, inv(ranges)) : 0.0f;
  }
};
// The fair share: chunks a range where all tiles' chunks fill the GPU once.
ES_RULE float fair_share(float chunks, float inv_slots) { return fmaxf(ceilf(chunks * inv_slots), 1.0f); }
// The first chunk of a tile's range
ES_RULE int range_begin(int chunks, int range, int ranges) { return (int)((long long)chunks * range / ranges); }

// Workgroups of a ranged launch that the GPU holds at once: 256 CUs, two workgroups each at D = 128 (64 KB of staging), three
// at D = 64 (134 registers: at 128, for four, the wide loop reloads spilled ones).
inline int resident(int D) { return D == 64 ? 768 : 512; }
// Items a head of a ranged launch: at most one a tile more than the ranges' chunks fill.
inline long long range_items(long long tiles, int Hk, int D) { return tiles + resident(D) / Hk + 1; }

}  // namespace es
