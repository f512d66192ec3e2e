// Shared by the packed-sequence attention kernels (packed_fwd.hip, packed_bwd.hip): which rows a workgroup owns, the tile
// layouts for head dims 64 and 128, and the host checks.
//
// Grouped heads: the G = H / Hk query heads of a kv head and the queries of a sequence form one list of rows,
// row = token * G + head in group, and a tile is a run of rows of that list. A tile of M rows then reads each key once for
// all heads of the group, and a kv head's gradients are plain sums over the rows of one list.
//
// Sequences are found on the device from cu_q / cu_k, so a call needs no length on the host: sequence b gets the tile
// numbers from floor(start_b * G / M) + b on, which leaves room for its ceil(len_b * G / M) tiles before the next one's
// (floor(x + y) + 1 >= floor(x) + ceil(y)); numbers that no tile has are workgroups that leave at once, at most one a
// sequence. Rows behind the last sequence form a sequence of their own, number B, without keys.
#pragma once
#include "../../include/packed_hip.h"
#include "elem.h"

namespace es {

namespace {

constexpr float PK_LN2 = 0.6931471805599453f;
constexpr int TILE = 128;                       // query rows of a forward tile
constexpr int BIAS_ROWS = ES_PACKED_BIAS_ROWS;  // entries of the LDS bias table: G * (2 R + 1)

// x / d for 0 <= x < 2^31 by one multiplication: mul = ceil(2^(32 + sh) / d) with 2^sh < d <= 2^(sh + 1), whose error
// mul * d - 2^(32 + sh) < d <= 2^(sh + 1) keeps x * error under 2^(32 + sh). d = 1: mul = 0.
struct FastDiv {
  unsigned mul;
  int sh;
};
static inline FastDiv fast_div(int d) {
  if (d <= 1) return FastDiv{0u, 0};
  int sh = 0;
  while ((2 << sh) < d) ++sh;
  return FastDiv{(unsigned)(((1ull << (32 + sh)) + d - 1) / d), sh};
}
__device__ __forceinline__ int divide(FastDiv f, int x) { return f.mul == 0 ? x : (int)(__umulhi((unsigned)x, f.mul) >> f.sh); }

// rows of sequence b in one of the token tensors
__device__ __forceinline__ int seq_start(const int* cu, int b, int B, int T) {
  if (cu == nullptr) return b >= B ? T : b * (T / B);
  return b <= 0 ? 0 : min(max(cu[b], 0), T);
}

// The sequence of tile number w where sequence b's numbers start at floor(start_b * G / M) + b; every lane of the wave
// calls it, one load a lane for 64 sequences.
template <int M>
__device__ __forceinline__ int seq_of_tile(const int* cu, int B, int T, int G, int w) {
  const int l = lane_id();
  int count = 0;
  for (int b0 = 0; b0 <= B; b0 += 64) {
    const int b = b0 + l;
    const bool in = b <= B && seq_start(cu, min(b, B), B, T) * G / M + b <= w;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    count += __builtin_popcountll(m);
    if (m != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(max(count - 1, 0));
}
template <int M>
__host__ __device__ __forceinline__ long long tile_numbers(int B, int T, int G) {
  return (long long)T * G / M + B + 1;
}

// Tile number w of a launch without ranges: the sequences in descending order of weight(b), so that the tiles with the most
// work start first and those that start last are short (workgroups are dispatched in order), each with its tiles(b) tiles.
// Up to 64 sequences (the rows behind the last one included): each lane takes one and adds up the tiles of those before it.
// More: their own order, by seq_of_tile. false: no tile has this number.
template <int M, class TILES, class WEIGHT>
__device__ __forceinline__ bool tile_of(const int* cu, int B, int T, int G, int w, const TILES& tiles, const WEIGHT& weight,
                                        int& b, int& t) {
  if (B < 64) {
    const int l = lane_id();
    const int mine = l <= B ? tiles(l) : 0, heavy = l <= B ? weight(l) : -1;
    int base = 0;
    for (int j = 0; j <= B; ++j) {
      const int tj = __builtin_amdgcn_readlane(mine, j), hj = __builtin_amdgcn_readlane(heavy, j);
      base += hj > heavy || (hj == heavy && j < l) ? tj : 0;
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(l <= B && base <= w && w < base + mine);
    if (hit == 0) return false;
    b = __builtin_ctzll(hit);
    t = w - __builtin_amdgcn_readlane(base, b);
    return true;
  }
  b = seq_of_tile<M>(cu, B, T, G, w);
  t = w - (__builtin_amdgcn_readfirstlane(seq_start(cu, b, B, T)) * G / M + b);
  return t >= 0 && t < __builtin_amdgcn_readfirstlane(tiles(b));
}

struct Seq {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Seq sequence(const int* cu_q, const int* cu_k, int B, int Tq, int Tk, int b) {
  Seq s;
  s.q0 = __builtin_amdgcn_readfirstlane(seq_start(cu_q, b, B, Tq));
  s.k0 = __builtin_amdgcn_readfirstlane(seq_start(cu_k, b, B, Tk));
  if (b >= B) {  // rows behind the last sequence
    s.nq = Tq - s.q0;
    s.nk = 0;
    return s;
  }
  s.nq = max(__builtin_amdgcn_readfirstlane(seq_start(cu_q, b + 1, B, Tq)) - s.q0, 0);
  s.nk = max(__builtin_amdgcn_readfirstlane(seq_start(cu_k, b + 1, B, Tk)) - s.k0, 0);
  return s;
}

// rows of the list of sequence b (b == B: the rows behind the last sequence), and its keys
__device__ __forceinline__ int list_rows(const int* cu_q, int B, int Tq, int G, int b) {
  const int q0 = seq_start(cu_q, b, B, Tq);
  return b >= B ? (Tq - q0) * G : max(seq_start(cu_q, b + 1, B, Tq) - q0, 0) * G;
}
__device__ __forceinline__ int list_keys(const int* cu_k, int B, int Tk, int b) {
  return b >= B ? 0 : max(seq_start(cu_k, b + 1, B, Tk) - seq_start(cu_k, b, B, Tk), 0);
}

// Tiles of D-column rows in LDS, 16-byte chunks XOR-swizzled so that sixteen consecutive rows read at one chunk, and four
// rows read at four consecutive chunks, touch every bank once. D = 128: 256-byte rows (common.h). D = 64: two 128-byte rows
// share a line of all banks, so bit 0 of the row is part of the position and bits 1 to 3 are mixed into the chunk.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? swz(row) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int tile_at(int row, int c) {
  return row * (D * 2) + ((c ^ swizzle<D>(row)) << 4);
}

// s_waitcnt vmcnt(N) and a compiler barrier: the transfers issued before the last N have landed
template <int N>
__device__ __forceinline__ void wait_transfers() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}
// this wave's LDS reads have returned: what they read may be overwritten
__device__ __forceinline__ void wait_lds() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
}

// The bias of a head group by clamped distance in log2 units: tab[g * (2 R + 1) + d + R], filled by the whole workgroup.
__device__ __forceinline__ void fill_bias(float* tab, const float* bias, const int* buckets, int num_buckets, int R, int G,
                                          int H, int hk) {
  const int n = 2 * R + 1;
  for (int i = threadIdx.x; i < G * n; i += blockDim.x) {
    const int g = i / n, bk = min(max(buckets[i - g * n], 0), num_buckets - 1);
    tab[i] = bias[(size_t)bk * H + hk * G + g] * LOG2E;
  }
  __syncthreads();
}

}  // namespace

// ------------------------------------------------------------------------------------------------ host checks
static inline int packed_check(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k,
                               const float* bias, const int* buckets, int num_buckets, int R, int B, int Tq, int Tk,
                               int H, int Hk, int D, float scale) {
  ES_REQUIRE(B > 0 && Tq >= 0 && Tk >= 0, ES_ERR_INVALID, "packed: B must be positive, Tq and Tk not negative");
  ES_REQUIRE(H > 0 && Hk > 0 && H % Hk == 0, ES_ERR_INVALID, "packed: H must be a positive multiple of Hk");
  ES_REQUIRE(D == 64 || D == 128, ES_ERR_UNSUPPORTED, "packed: head dim must be 64 or 128");
  ES_REQUIRE(H <= 4096, ES_ERR_UNSUPPORTED, "packed: at most 4096 heads");
  ES_REQUIRE((Tq == 0 || q) && (Tk == 0 || (k && v)), ES_ERR_INVALID, "packed: null q / k / v");
  ES_REQUIRE((cu_q || Tq % B == 0) && (cu_k || Tk % B == 0), ES_ERR_INVALID,
             "packed: without cu_q / cu_k the rows must divide into B equal sequences");
  ES_REQUIRE(scale > 0.0f && scale < 1e30f, ES_ERR_INVALID, "packed: scale must be positive and finite");
  ES_REQUIRE(((long long)Tq * H + 128LL * (B + 1)) < (1LL << 30) && (long long)Tk + 64LL * (B + 1) < (1LL << 30),
             ES_ERR_UNSUPPORTED, "packed: too many rows");
  if (bias) {
    ES_REQUIRE(buckets && num_buckets > 0 && R >= 0, ES_ERR_INVALID, "packed: a bias needs buckets");
    ES_REQUIRE(R <= BIAS_ROWS && (long long)(H / Hk) * (2 * R + 1) <= BIAS_ROWS, ES_ERR_UNSUPPORTED,
               "packed: (H / Hk) * (2 R + 1) must be at most 816");
  }
  return ES_OK;
}

}  // namespace es
