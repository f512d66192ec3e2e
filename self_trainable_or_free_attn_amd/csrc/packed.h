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
#include "packed_rules.h"

#include <initializer_list>

namespace es {

namespace {

constexpr float PK_LN2 = 0.6931471805599453f;
constexpr int TILE = 128;                       // query rows of a forward tile
constexpr int BIAS_ROWS = ES_PACKED_BIAS_ROWS;  // G * (2 R + 1) at most
// With one head a group the table repeats its ends for BIAS_PAD distances more on either side: the 32 keys of a run that is
// not all at -R and below or all at R and beyond stand within 31 + 31 of that range, and need no clamp.
constexpr int BIAS_PAD = 64, BIAS_TABLE = BIAS_ROWS + 2 * BIAS_PAD;
// Finite bias values are held to this magnitude (see fill_bias).
constexpr float BIAS_MAX = ES_PACKED_BIAS_MAX;
constexpr long long MAX_GRID = 1LL << 24;  // workgroups of a launch: its threads are counted in 32 bits

// rows of sequence b in one of the token tensors
__device__ __forceinline__ int seq_start(const int* cu, int b, int B, int T) {
  if (cu == nullptr) return b >= B ? T : b * (T / B);
  return b <= 0 ? 0 : min(max(cu[b], 0), T);
}

// The sequence of tile number w (numbers by first_tile); every lane of the wave
// calls it, one load a lane for 64 sequences.
template <int M>
__device__ __forceinline__ int seq_of_tile(const int* cu, int B, int T, int G, int w) {
  const int l = lane_id();
  int count = 0;
  for (int b0 = 0; b0 <= B; b0 += 64) {
    const int b = b0 + l;
    const bool in = b <= B && first_tile<M>(seq_start(cu, min(b, B), B, T), G, b) <= w;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(in);
    count += __builtin_popcountll(m);
    if (m != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(max(count - 1, 0));
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

// Tile number w of a launch without ranges: the sequences in descending order of their other length (keys where tiles are of
// rows, rows where KEYS), so that the tiles with the most work start first and those that start last are short (workgroups are
// dispatched in order), each with its tiles. Up to 64 sequences (the rows behind the last one included): each lane takes one
// and adds up the tiles of those before it. More: their own order, by seq_of_tile. false: no tile has this number. lens: the
// keys of each sequence, held to `cap`, in the place of cu_k.
template <int M, bool KEYS>
__device__ __forceinline__ bool tile_of(const int* cu_q, const int* cu_k, int B, int Tq, int Tk, int G, int w, Seq& s, int& b,
                                        int& t, const int* lens = nullptr, int cap = 0) {
  if (B < 64) {
    const int l = min(lane_id(), B), last = KEYS ? Tk : Tq;
    Seq x;
    x.q0 = seq_start(cu_q, l, B, Tq);
    x.k0 = seq_start(cu_k, l, B, Tk);
    x.nq = l < B ? max(seq_start(cu_q, l + 1, B, Tq) - x.q0, 0) : 0;
    x.nk = l < B ? max(seq_start(cu_k, l + 1, B, Tk) - x.k0, 0) : 0;
    if (lens != nullptr) x.nk = l < B ? min(max(lens[l], 0), cap) : 0;
    if (l == B) (KEYS ? x.nk : x.nq) = last - (KEYS ? x.k0 : x.q0);
    const int tiles = ((KEYS ? x.nk : x.nq * G) + M - 1) / M, weight = KEYS ? x.nq : x.nk;
    int base = 0;
    for (int j = 0; j <= B; ++j) {
      const int tj = __builtin_amdgcn_readlane(tiles, j), wj = __builtin_amdgcn_readlane(weight, j);
      base += wj > weight || (wj == weight && j < l) ? tj : 0;
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(base <= w && w < base + tiles);
    if (hit == 0) return false;
    b = __builtin_ctzll(hit);  // (lanes past B repeat lane B's)
    t = w - __builtin_amdgcn_readlane(base, b);
    s.q0 = __builtin_amdgcn_readlane(x.q0, b);
    s.nq = __builtin_amdgcn_readlane(x.nq, b);
    s.k0 = __builtin_amdgcn_readlane(x.k0, b);
    s.nk = __builtin_amdgcn_readlane(x.nk, b);
    return true;
  }
  b = KEYS ? seq_of_tile<M>(cu_k, B, Tk, 1, w) : seq_of_tile<M>(cu_q, B, Tq, G, w);
  s = sequence(cu_q, cu_k, B, Tq, Tk, b);
  if (lens != nullptr) s.nk = b < B ? __builtin_amdgcn_readfirstlane(min(max(lens[b], 0), cap)) : 0;
  if (KEYS && b >= B) {
    s.nk = Tk - s.k0;
    s.nq = 0;
  }
  t = w - (KEYS ? first_tile<M>(s.k0, 1, b) : first_tile<M>(s.q0, G, b));
  return t >= 0 && t * M < (KEYS ? s.nk : s.nq * G);
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

// Two or three workgroups share a SIMD, a wave each: s_setprio(1) around a wave's runs of products lets it issue them before the
// other waves' exponentials, whose instructions then fill the gaps; at one priority the two take turns and the matrix unit waits.
// (Measured where it is used.)

// The bias of a head group by distance in log2 units, filled by the whole workgroup (which waits at a barrier before it reads
// it): bias_at(g, d) with d clamped to -R .. R, or for G = 1 within BIAS_PAD of that. Values like -1e9 or the lowest float, as
// masks have them, leave a float32 score no bits of its product; where all keys of a row have one, the probabilities are taken
// against a maximum rounded by more than the exponent's range and overflow. At 2^17 a score still has steps of 2^-6, and keys
// with any other value beside them vanish all the same. -inf stays.
__device__ __forceinline__ int bias_width(int G, int R) { return 2 * R + 1 + (G == 1 ? 2 * BIAS_PAD : 0); }
__device__ __forceinline__ int bias_row(int G, int R, int g) { return g * bias_width(G, R) + R + (G == 1 ? BIAS_PAD : 0); }
__device__ __forceinline__ void fill_bias(float* tab, const float* bias, const int* buckets, int num_buckets, int R, int G,
                                          int H, int hk) {
  const int n = bias_width(G, R);
  for (int i = threadIdx.x; i < G * n; i += blockDim.x) {
    const int g = i / n, d = min(max(i - bias_row(G, R, g), -R), R), bk = min(max(buckets[d + R], 0), num_buckets - 1);
    const float x = bias[(size_t)bk * H + hk * G + g];
    tab[i] = (fabsf(x) < INFINITY ? fminf(fmaxf(x, -BIAS_MAX), BIAS_MAX) : x) * LOG2E;
  }
}
// x[r] = x[r] * sc + bias of the key at distance d0 + 8 (r / 4) + r % 4; row: the table at distance 0
__device__ __forceinline__ void add_bias(f32x16& x, float sc, const float* row, int d0, int G, int R) {
  if (G == 1) {
    row += d0;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], sc, row[8 * (r / 4) + r % 4]);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], sc, row[min(max(d0 + 8 * (r / 4) + r % 4, -R), R)]);
  }
}

}  // namespace

// ------------------------------------------------------------------------------------------------ host checks
static inline bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

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
               "packed: (H / Hk) * (2 R + 1) must be at most 784");
  }
  return ES_OK;
}

}  // namespace es
