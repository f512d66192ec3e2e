// Attention of new tokens over paged caches of 16 and 4 bits (gfx950, bf16 / fp16): where the tiles of packed_tiles.h get their
// keys from, and tiles of their own for few rows over a cache of 4 bits.
//
// Page numbers: a page holds 16 rows or a multiple of that, so sixteen keys that start at a multiple of sixteen stand in one page.
// Each lane of a wave holds the page number of one such group, a window of 64 groups (the next window's numbers are on their way),
// and the wave takes the one that it needs by a lane read: no load stands between a chunk and its transfers.
// Groups whose page number is outside the cache are missing: their scores become -inf, their values zeros.
#include "packed_tiles.h"
#include "paged.h"
#include "paged_rules.h"

#include <algorithm>
#include <type_traits>

namespace es {

namespace {

__device__ __forceinline__ int cached_keys(const FwdArgs& a, int b) {
  return b >= a.B ? 0 : __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.paged.cap));
}
// tokens that stand past the last page
__device__ __forceinline__ int keys_over(const FwdArgs& a, int b) {
  return b >= a.B ? 0 : __builtin_amdgcn_readfirstlane(max(a.lens[b], a.paged.cap)) - a.paged.cap;
}

// Page numbers of 64 groups of sixteen keys, a lane each: narrow tiles, whose waves take every fourth run of 32 keys, hold those of
// 32 runs of their own, wide ones those of sixteen chunks. -1: missing; 0 where the sequence has no keys.
struct PageWindow {
  int cur, next, first, step;  // the window's first run or chunk, and how many it spans
  unsigned long long gone;
  bool narrow;

  __device__ __forceinline__ int fetch(const FwdArgs& a, const Job& j, int from) const {
    const int l = lane_id(), g = narrow ? 2 * (from + 4 * (l >> 1)) + (l & 1) : 4 * from + l;
    if (16 * g >= j.nk) return 0;
    const int p = j.table[(16 * g) >> a.paged.shift];
    return p >= 0 && p < a.paged.num_pages ? p : -1;
  }
  __device__ __forceinline__ void start(const FwdArgs& a, const Job& j, int from, bool narrow_) {
    narrow = narrow_;
    step = narrow ? 128 : 16;
    first = from;
    cur = fetch(a, j, first);
    next = fetch(a, j, first + step);
    gone = __builtin_amdgcn_ballot_w64(cur < 0);
  }
  // moves on to the window that holds run (chunk) x, which is in this one or the first of the next; its slot
  __device__ __forceinline__ int slot(const FwdArgs& a, const Job& j, int x) {
    if (x - first >= step) {
      first += step;
      cur = next;
      gone = __builtin_amdgcn_ballot_w64(cur < 0);
      next = fetch(a, j, first + step);
    }
    return narrow ? (x - first) >> 2 : x - first;
  }
  // page number of group i of the window
  __device__ __forceinline__ int page(int i) const { return __builtin_amdgcn_readlane(cur, i); }
  __device__ __forceinline__ unsigned missing(int i, unsigned mask) const { return (unsigned)(gone >> i) & mask; }
};

// the scores of missing groups of sixteen keys; bits: two groups
__device__ __forceinline__ void mask_groups(f32x16& s, unsigned bits) {
  if (bits == 0) return;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (bits >> (r / 8) & 1) s[r] = -INFINITY;
}

// 16 bits: transfers of sixteen rows each from their page, rows past the sequence's keys and of missing pages read as zeros
template <int D>
struct Pages {
  static constexpr bool HOLES = true, STAGED = false, FINE = true;
  static constexpr int LPR = D / 8, NI = D / 32;  // NI transfers of 64 / LPR rows: sixteen rows
  PageWindow window;
  unsigned src[2 * NI], stride, now, then;
  int wv;
  __device__ __forceinline__ Pages(const FwdArgs& a, const Job& j, int l, int wave, bool narrow) : now(0), then(0), wv(wave) {
    stride = (unsigned)a.paged.row_stride * 2;
#pragma unroll
    for (int i = 0; i < 2 * NI; ++i) {  // (the row within its group; its place in LDS goes by the row within the tile)
      const int R = i * (64 / LPR) + l / LPR, at = (narrow ? 0 : 16 * wv) + R;
      src[i] = (unsigned)(R & 15) * stride + (unsigned)(((l % LPR) ^ swizzle<D>(at)) * 16);
    }
    window.start(a, j, narrow ? 2 * j.c0 + wv : j.c0, narrow);
  }
  // group g of the sequence in page `page`: what holds it, and the bytes of it that are there
  __device__ __forceinline__ size_t group(const FwdArgs& a, const Job& j, int g, int page, unsigned& bytes) const {
    const int left = min(16, j.nk - 16 * g);
    bytes = page < 0 || left <= 0 ? 0u : (unsigned)(left - 1) * stride + D * 2;
    return (size_t)max(page, 0) * a.paged.page_stride +
           (size_t)((16 * g) & ((1 << a.paged.shift) - 1)) * a.paged.row_stride;
  }
  __device__ __forceinline__ void wide(const FwdArgs& a, const Job& j, int c, unsigned dst) {
    const int slot = window.slot(a, j, c);
    then = window.missing(4 * slot, 15u);
    unsigned bytes;
    const size_t at = group(a, j, 4 * c + wv, window.page(4 * slot + wv), bytes);
    const srd_t rk = make_srd(j.k + at, bytes), rv = make_srd(j.v + at, bytes);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rk, dst + i * 1024, src[i], 0u);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rv, dst + BK * D * 2 + i * 1024, src[i], 0u);
  }
  __device__ __forceinline__ void settle(char*) {}
  __device__ __forceinline__ void run(const FwdArgs& a, const Job& j, bool v, int u, unsigned dst) {
    const int slot = window.slot(a, j, u);
    then = window.missing(2 * slot, 3u);
    const e16_t* base = v ? j.v : j.k;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      unsigned bytes;
      const size_t at = group(a, j, 2 * u + t, window.page(2 * slot + t), bytes);
      const srd_t r = make_srd(base + at, bytes);
#pragma unroll
      for (int i = 0; i < NI; ++i) dma16_at(r, dst + (NI * t + i) * 1024, src[NI * t + i], 0u);
    }
  }
  __device__ __forceinline__ void enter() { now = then; }
  __device__ __forceinline__ void enter_run(int) { now = then; }  // (called before the next run's transfers)
  __device__ __forceinline__ void mask(f32x16& s, int run) const { mask_groups(s, now >> (2 * run) & 3u); }
};

// 4 bits, wide tiles: a thread loads 32 codes of a row and their scale a chunk ahead (D = 128: of keys and of values) and writes
// them as token values where the transfers of 16 bits would have put them. Lanes have the rows in an order in which eight
// neighbours write to different banks (in the order of memory, a row to four lanes, 1.5e7 cycles of conflicts instead of 7e5, and
// 32760 tokens, 24 heads, 7180 us instead of 7110).
template <int D>
struct Codes {
  static constexpr bool HOLES = true, STAGED = true, FINE = true;
  static constexpr int PARTS = D == 128 ? 2 : 1;
  PageWindow window;
  uint4 code[PARTS];
  unsigned scale[PARTS], now, then;
  int tensor, row, part, wv;  // D = 64: two waves have the keys, two the values
  __device__ __forceinline__ Codes(const FwdArgs& a, const Job& j, int l, int wave, bool) : now(0), then(0), wv(wave) {
    tensor = D == 128 ? 0 : wv >> 1;
    row = D == 128 ? 16 * wv + ((l & 1) | (l >> 1 & 3) << 2 | (l >> 3 & 1) << 1)
                   : 32 * (wv & 1) + (2 * (l & 7) | (l >> 3 & 1) | (l & 16));
    part = l >> (D == 128 ? 4 : 5);
    window.start(a, j, j.c0, false);
  }
  __device__ __forceinline__ void wide(const FwdArgs& a, const Job& j, int c, unsigned) {
    const int slot = window.slot(a, j, c);
    then = window.missing(4 * slot, 15u);
    int page = window.page(4 * slot + (D == 128 ? wv : 2 * (wv & 1)));
    if (D == 64) page = row & 16 ? window.page(4 * slot + 2 * (wv & 1) + 1) : page;
    const int key = BK * c + row;
    const bool there = key < j.nk && page >= 0;
    const size_t at = (((size_t)max(page, 0) * a.Hk + j.hk) << a.paged.shift) + (key & ((1 << a.paged.shift) - 1));
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const uint8_t* codes = tensor + p ? a.paged.codes[1] : a.paged.codes[0];
      const uint8_t* scales = tensor + p ? a.paged.scales[1] : a.paged.scales[0];
      code[p] = make_uint4(0, 0, 0, 0);
      scale[p] = 127;
      if (there) {
        code[p] = *reinterpret_cast<const uint4*>(codes + at * (D / 2) + 16 * part);
        scale[p] = scales[at * (D / 32) + part];
      }
    }
  }
  __device__ __forceinline__ void settle(char* base) const {
    const int at = tile_at<D>(row, 4 * part);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      char* tile = base + (tensor + p) * BK * D * 2;
      const float s = __uint_as_float(scale[p] << 23);
      const unsigned w[4] = {code[p].x, code[p].y, code[p].z, code[p].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<ev8*>(tile + (at ^ (16 * i))) = decode8(w[i], s);
    }
  }
  __device__ __forceinline__ void enter() { now = then; }
  __device__ __forceinline__ void mask(f32x16& s, int run) const { mask_groups(s, now >> (2 * run) & 3u); }
};

// ------------------------------------------------------------------------------------------------ few rows over 4 bits
// MFMA 16x16x32. Operand layouts (checked on the GPU): A (16x32): lane l holds A[l % 16][8 (l / 16) + 0..7], B (32x16): lane l
// holds B[8 (l / 16) + 0..7][l % 16], C (16x16): lane l, register r holds C[4 (l / 16) + r][l % 16].
__device__ __forceinline__ f32x4 emfma16(ev8 a, ev8 b, f32x4 c) {
#ifdef ES_ELEM_F16
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#endif
}

// sums and maxima over the four lanes l % 16 + 16 i
__device__ __forceinline__ float2 lane_pair16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_rows16(float x) {
  const float2 h = lane_pair16(x);
  return max_xor32(fmaxf(h.x, h.y));
}
__device__ __forceinline__ float sum_rows16(float x) {
  const float2 h = lane_pair16(x);
  return sum_xor32(h.x + h.y);
}

// V rows of a run in a wave's LDS: 16-byte chunk c of row r at c ^ values_swizzle(r). Eight lanes write a chunk each of eight rows,
// and sixteen lanes read four rows at two neighbouring chunks: both touch every bank once. (With the rows of the wide tiles and a
// row to four lanes, LDS was busy 58 % of the time, 48 tokens against 8000 keys, 32 heads over 8; so 20 %.)
template <int D>
__device__ __forceinline__ int values_swizzle(int row) {
  return (row & 3) << 1 | (row >> 2 & 1) | (D == 128 ? row & 8 : 0);
}
template <int D>
__device__ __forceinline__ int values_at(int row, int c) {
  return row * (D * 2) + ((c ^ values_swizzle<D>(row)) << 4);
}

// Up to 16 NR rows; every wave has the same rows and takes every fourth run of 32 keys, the four states are merged at the end.
// S^T = K Q^T of two groups of sixteen keys, channels in the order in which a lane's bytes hold them: lane (key l % 16, quarter
// l / 16) loads a quarter of its key's row in one piece and feeds it to the products without LDS. The exponentials of both groups
// are the B operand of O^T += V^T P^T with the keys in the order 4 q + 0..3, 16 + 4 q + 0..3 of quarter q. V goes through the
// wave's own LDS as token values, from where it is read transposed. No barrier in the loop.
// P goes into the products as its 16-bit value and, rounded again, what that leaves (FINE in packed_tiles.h, for caches of 16
// bits): launches of few rows wait for HBM, and outputs then have no error but their own rounding (48 tokens against 1 to 16000
// keys over 4 bits: relative error 4.7e-4 instead of 6.8e-4, with probabilities in float32 4.7e-4; 97.1 us instead of 96.4, and at
// most 7 % more, 64 tokens against 8000 keys of 64 channels). Wide tiles, which the matrix units bound, round P once.
template <int D, int NR>
__device__ __forceinline__ void narrow4_tile(const FwdArgs& a, const Job& j, char* lds, float* stats) {
  constexpr int NKS = D / 32, NDB = D / 16, ROW = D * 2, WORDS = D / 32;  // words of 8 codes a lane and group
  constexpr int LDS_WAVE = NR * 32 * ROW;
  const int tid = threadIdx.x, l = tid & 63, c = l & 15, g = l >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = j.nq * a.G, last = min(j.r0 + 16 * NR, rows) - 1;
  const int seen_min = keys_seen(a, j, j.r0), seen_max = keys_seen(a, j, last);

  ev8 q[NR][NKS];
  f32x4 o[NR][NDB];
  float lsum[NR], mrun[NR];
  int seen[NR];
  size_t at[NR];
  bool valid[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = j.r0 + 16 * n + c;
    valid[n] = r < rows;
    const int tok = divide(a.div_g, r), head = r - tok * a.G;
    at[n] = ((size_t)(j.q0 + (valid[n] ? tok : 0)) * a.Hk + j.hk) * a.G + (valid[n] ? head : 0);
    seen[n] = valid[n] ? keys_seen(a, j, r) : 0;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const ev8 z = {};
      q[n][ks] = valid[n] ? *reinterpret_cast<const ev8*>(a.q + at[n] * D + (D / 4) * g + 8 * ks) : z;
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[n][db] = f32x4{};
    lsum[n] = 0.0f;
    mrun[n] = -INFINITY;
  }

  PageWindow window;
  const int end = min(2 * j.c1, (seen_max + 31) / 32);
  int u = 2 * j.c0 + wv;
  window.start(a, j, u, true);
  typedef typename std::conditional<D == 128, uint4, uint2>::type Piece;  // a lane's codes of a group
  Piece kc[2], vc[2];
  unsigned ks8[2], vs8[2];
  // a lane's quarter of its key's row: K as the products take it, V as it is written
  const int k_at = c * (D / 2) + g * (D / 8), ks_at = c * (D / 32) + (D == 128 ? g : g >> 1);
  size_t at16[2];  // a run's groups: the first row in the cache
  unsigned missing = 0, missing_next = 0;
  auto places = [&](int u) {
    const int slot = window.slot(a, j, u);
    missing_next = window.missing(2 * slot, 3u);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      at16[t] = (((size_t)max(window.page(2 * slot + t), 0) * a.Hk + j.hk) << a.paged.shift) +
                ((32 * u + 16 * t) & ((1 << a.paged.shift) - 1));
  };
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      kc[t] = *reinterpret_cast<const Piece*>(a.paged.codes[0] + at16[t] * (D / 2) + k_at);
      ks8[t] = a.paged.scales[0][at16[t] * (D / 32) + ks_at];
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      vc[t] = *reinterpret_cast<const Piece*>(a.paged.codes[1] + at16[t] * (D / 2) + k_at);
      vs8[t] = a.paged.scales[1][at16[t] * (D / 32) + ks_at];
    }
  };
  char* vb = lds + wv * LDS_WAVE;
  const int tr = values_at<D>(4 * g + (c >> 2), (c & 3) >> 1) + (c & 1) * 8, put = values_at<D>(c, WORDS * g);
  if (u < end) {
    places(u);
    load_k();
    load_v();
  }
  for (; u < end; u += 4) {
    const bool more = u + 4 < end;
    missing = missing_next;
    f32x4 s[NR][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float scale = __uint_as_float(ks8[t] << 23);
      unsigned w[WORDS];
      __builtin_memcpy(w, &kc[t], sizeof(w));
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][t] = f32x4{};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const ev8 k = decode8(w[ks], scale);
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][t] = emfma16(k, q[n][ks], s[n][t]);
      }
    }
    // V of this run to LDS, then the next run's loads
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = 32 * u + 16 * t + c;
      const bool there = key < j.nk && !(missing >> t & 1);
      const float scale = __uint_as_float((there ? vs8[t] : 127u) << 23);
      unsigned w[WORDS];
      __builtin_memcpy(w, &vc[t], sizeof(w));
#pragma unroll
      for (int i = 0; i < WORDS; ++i)
        *reinterpret_cast<ev8*>(vb + 16 * t * ROW + (put ^ (16 * i))) = decode8(w[i], scale);
    }
    asm volatile("" ::: "memory");
    if (more) {
      places(u + 4);
      load_k();
      load_v();
    }
    ev8 p[NR], rest[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (missing || 32 * (u + 1) > seen_min) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int left = missing >> t & 1 ? 0 : seen[n] - 32 * u - 16 * t - 4 * g;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r >= left) s[n][t][r] = -INFINITY;
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      mx = max_rows16(mx) * a.scale;
      if (mx > mrun[n] + SLACK) {  // (as in Rows::raise)
        const float next = mrun[n] == -INFINITY ? mx : mrun[n] + ceilf(mx - mrun[n]), alpha = exp2f_fast(mrun[n] - next);
        lsum[n] *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[n][db] *= alpha;
        mrun[n] = next;
      }
      const float shift = P_SHIFT - (mrun[n] == -INFINITY ? 0.0f : mrun[n]);
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = exp2f_fast(fmaf(s[n][i >> 2][i & 3], a.scale, shift));
      p[n] = epack8(e);
      rest[n] = rest8(e, p[n]);
      lsum[n] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    }
    ev8 before;  // (a block's second product behind the next block's first: neither waits for the other)
#pragma unroll
    for (int db = 0; db <= NDB; ++db) {
      ev8 v = {};
      if (db < NDB) v = ecat_tr(lds_read_tr(vb, tr ^ (32 * db)), lds_read_tr(vb + 16 * ROW, tr ^ (32 * db)));
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        if (db < NDB) o[n][db] = emfma16(v, p[n], o[n][db]);
        if (db > 0) o[n][db - 1] = emfma16(before, rest[n], o[n][db - 1]);
      }
      before = v;
    }
    asm volatile("" ::: "memory");
  }

  // merge of the four waves' states: each wave finishes a quarter of the channels
  static_assert(NR * NDB * 4 * 64 * 4 <= LDS_WAVE, "a wave's O fits its LDS");
  float* mine = reinterpret_cast<float*>(vb);
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int i = 0; i < NDB * 4; ++i) mine[(n * NDB * 4 + i) * 64 + l] = o[n][i >> 2][i & 3];
    const float sum = sum_rows16(lsum[n]);
    if (g == 0) {
      stats[((wv * NR + n) * 2) * 16 + c] = mrun[n];
      stats[((wv * NR + n) * 2 + 1) * 16 + c] = sum;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float w[4], top = -INFINITY, tot = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, stats[((i * NR + n) * 2) * 16 + c]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = stats[((i * NR + n) * 2) * 16 + c];
      w[i] = m == -INFINITY ? 0.0f : exp2f_fast(m - top);
      tot += w[i] * stats[((i * NR + n) * 2 + 1) * 16 + c];
    }
    const float inv = j.part != nullptr ? 1.0f : tot == 0.0f ? 0.0f : 1.0f / tot;
    const int r = 16 * n + c;
#pragma unroll
    for (int x = 0; x < NDB / 4; ++x) {
      const int db = wv * (NDB / 4) + x, col = 16 * db + 4 * g;
      f32x4 acc = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* other = reinterpret_cast<const float*>(lds + i * LDS_WAVE);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(w[i], other[(n * NDB * 4 + 4 * db + e) * 64 + l], acc[e]);
      }
      if (j.part != nullptr) *reinterpret_cast<f32x4*>(j.part + 2 * j.part_rows + r * D + col) = acc;
      else if (valid[n]) store_row<D>(a, at[n], col, acc * inv);
    }
    if (wv == 0 && g == 0) {
      if (j.part != nullptr) {
        j.part[r] = top;
        j.part[j.part_rows + r] = tot;
      } else if (valid[n]) {
        a.lse[at[n]] = tot == 0.0f ? -INFINITY : (top - P_SHIFT + log2f(tot)) * PK_LN2;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ kernels
// Rows a tile of a launch: TOKENS, up to sixteen (4 bits) or 32 (16 bits) rows, which are narrow tiles, or 128 (64), of which those
// with up to 32 rows are.
template <int BITS>
constexpr int TOKENS = BITS == 4 ? 16 : 32;

template <int D, int BITS, int M>
__device__ __forceinline__ void paged_tile(const FwdArgs& a, const Job& j, char* lds, float* stats) {
  if constexpr (BITS == 16 && M == TOKENS<16>) {
    narrow_tile<D, false, Pages<D>>(a, j, lds, stats, nullptr);
  } else if constexpr (BITS == 16) {
    run_tile<D, false, M, Pages<D>>(a, j, lds, stats, nullptr);
  } else if constexpr (M == TOKENS<4>) {
    narrow4_tile<D, 1>(a, j, lds, stats);
  } else {
    if (j.nq * a.G - j.r0 <= 32) narrow4_tile<D, 2>(a, j, lds, stats);
    else wide_tile<D, false, M, Codes<D>>(a, j, lds, stats, nullptr);
  }
}

// the job of a tile of sequence b, its keys and rows
template <int D, int BITS>
__device__ __forceinline__ void paged_job(const FwdArgs& a, Job& j, int q0, int nq, int b, int nk, int over, int hk) {
  j.table = a.paged.table + (size_t)(b < a.B ? b : 0) * a.paged.max_pages;
  if (BITS == 16) {
    j.k = a.paged.k + (size_t)hk * a.paged.head_stride;
    j.v = a.paged.v + (size_t)hk * a.paged.head_stride;
  }
  j.q0 = q0;
  j.nq = nq;
  j.nk = nk;
  j.over = over;
  j.hk = hk;
  j.causal = a.causal;
}

// LDS: two chunks (16 bits, narrow: a run a wave) of keys and values; 4 bits, TOKENS: a run of values a wave
template <int D, int M>
constexpr int paged_lds() { return M == TOKENS<4> ? 4 * 32 * D * 2 : 4 * BK * D * 2; }
// Workgroups that a CU holds. (TOKENS over 4 bits: 157 registers; at 128, for four, the loop reloads spilled ones, and 48 tokens
// against 8000 keys, 32 heads over 8, take 107 us instead of 88.)
#define ES_PAGED_RESIDENT(D, M) ((M) == 16 || (D) == 64 ? 3 : 2)

// whole tiles: grid tiles * Hk, a tile's heads on neighbouring workgroups
template <int D, int BITS, int M>
__global__ __launch_bounds__(256, ES_PAGED_RESIDENT(D, M)) void paged_whole_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[paged_lds<D, M>()];
  __shared__ float stats[4 * 128];
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  int b, t;
  Seq s;
  Job j;
  if (!tile_of<M, false>(a.cu_q, nullptr, a.B, a.Tq, 0, a.G, w, s, b, t, a.lens, a.paged.cap)) return;
  j.r0 = ((s.nq * a.G + M - 1) / M - 1 - t) * M;
  paged_job<D, BITS>(a, j, s.q0, s.nq, b, s.nk, keys_over(a, b), hk);
  j.part = nullptr;
  j.c0 = 0;
  j.c1 = tile_chunks<M>(a, j);
  paged_tile<D, BITS, M>(a, j, lds, stats);
}

// ------------------------------------------------------------------------------------------------ tokens: equal shares
// Launches of narrow tiles are bound by HBM, and a workgroup reads keys as fast as any other: all tiles of a head, sequence by
// sequence, laid end to end by the chunks that they read, are cut into as many equal shares as the GPU holds workgroups. Each
// workgroup does its share: the rest of a tile, whole tiles, the beginning of a tile. Whole tiles are finished by it, pieces leave
// partials (two a share at most) that a second launch adds in order. So one long history among short ones takes what it costs and
// not the time of one workgroup (200 tokens against 1 to 40000 keys, 32 heads over 8: 16 bits 766 us whole tiles, 704 key ranges,
// 535 shares; 4 bits 468, 256, 167).
// Every wave derives its share's borders from the lengths by itself, so they stay on the device: costs are whole numbers (units of
// 1 / cost_unit chunks, TILE_COST more for a tile's beginning and end), and a border is a function of its place alone, so all waves
// agree on it. A border near a tile's own (SNAP of a share) moves there, which saves a partial; where all tiles are about as long
// as a share or shorter and no share needs more than one, all of them do. In launches so small that shares are left over, each
// tile has some of its own: no workgroup then has two pieces, one after the other (7 tokens against 3 to 9923 keys, 24 heads over
// 3, 17.9 us instead of 20.4; 18 against 1 to 25716 over 4 bits, 16 heads over 2, 21.2 instead of 23.0). TILE_COST 2 and shares of
// 4 chunks instead of LEAST = 6 at least: 12 tokens against 6 to 23354 keys, 3 heads, 33.0 us instead of 28.1; 100 against 1 to
// 40000, 16 heads of 64 over 2, 47.7 instead of 43.3; the large cases above the same. SNAP 0: 200 tokens of 1 to 40000 keys over
// 4 bits 171.5 us instead of 166.9, others up to 1 % slower; 0.25: in 16 bits 564 instead of 544, though 256 against 2000 over 4
// bits 118 instead of 123. WHOLE 1: 63 tokens against 2000 keys 114 us instead of 101; 2: 48 against 8000 over 4 bits 117 instead
// of 87, though in 16 bits 269 instead of 293. A lane has LISTS sequences one behind the other, so up to 255 are read once. (Over
// 16 bits 28 scalar registers are spilled to lanes at D = 64 and 35 at D = 128.)
struct Share {
  int tile, chunk;  // tile number as in packed.h (first_tile of its sequence and its place there), chunk within it
};
constexpr int END = 0x7fffffff;
constexpr int LISTS = 4;
constexpr float TILE_COST = 4.0f, LEAST = 6.0f, SNAP = 0.1f, WHOLE = 1.3f;

// rows and keys of sequence b (b == B: the rows behind the last one, without keys)
__device__ __forceinline__ int paged_rows_of(const FwdArgs& a, int b) { return list_rows(a.cu_q, a.B, a.Tq, a.G, b); }
__device__ __forceinline__ int paged_keys_of(const FwdArgs& a, int b) {
  return b >= a.B ? 0 : min(max(a.lens[min(b, a.B - 1)], 0), a.paged.cap);
}

template <int M>
struct Shares {
  const FwdArgs& a;
  int mine[LISTS], upto, from;  // of the first 64 * LISTS sequences: costs of this lane's, their sum with and without them
  int share, count;             // cost of a share; shares
  bool whole, even;             // no tile is cut; every tile has shares of its own

  // a tile's cost, and the tiles, of sequence b. (Causal tiles of more rows than one tile has count as if they saw all keys: these
  // are sequences of several tiles, which launches of tokens rarely have.)
  __device__ __forceinline__ int cost(int b, int& tiles) const {
    if (b > a.B) return tiles = 0;
    tiles = (paged_rows_of(a, b) + M - 1) / M;
    const int each = max((int)(((float)((paged_keys_of(a, b) + BK - 1) / BK) + TILE_COST) * a.cost_unit), 1);
    return even ? own_shares(each) * share : each;
  }
  __device__ __forceinline__ int own_shares(int each) const {
    return max((int)ceilf((float)each / (float)share - (WHOLE - 1.0f)), 1);
  }

  __device__ __forceinline__ Shares(const FwdArgs& args) : a(args), even(false) {
    int total = 0, all_tiles = 0, each_of[LISTS], tiles_of[LISTS];
    float most = 0.0f;
    for (int b0 = 0; b0 <= a.B; b0 += 64 * LISTS) {
      int x[LISTS], sum = 0;
#pragma unroll
      for (int k = 0; k < LISTS; ++k) {
        int tiles;
        const int each = cost(b0 + lane_id() * LISTS + k, tiles);
        x[k] = each * tiles;
        each_of[k] = each;
        tiles_of[k] = tiles;
        most = fmaxf(most, tiles > 0 ? (float)each : 0.0f);
        all_tiles += tiles;
        sum += x[k];
      }
      const int scan = total + wave_scan(sum);
      if (b0 == 0) {
#pragma unroll
        for (int k = 0; k < LISTS; ++k) mine[k] = x[k];
        upto = scan;
        from = scan - sum;
      }
      total = __builtin_amdgcn_readlane(scan, 63);
    }
    most = wave_max_dpp(most);
    share = max((total + a.shares - 1) / a.shares, a.least_share);
    count = total > 0 ? (total + share - 1) / share : 1;
    whole = most <= WHOLE * (float)share && __builtin_amdgcn_readlane(wave_scan(all_tiles), 63) <= a.shares;
    if (share > a.least_share || a.B >= 64 * LISTS) return;
    int own = 0;
#pragma unroll
    for (int k = 0; k < LISTS; ++k) own += own_shares(each_of[k]) * tiles_of[k];
    const int scan = wave_scan(own), all = __builtin_amdgcn_readlane(scan, 63);
    if (all > a.shares) return;
    even = true;
    count = max(all, 1);
    upto = scan * share;
    from = upto - own * share;
#pragma unroll
    for (int k = 0; k < LISTS; ++k) mine[k] = own_shares(each_of[k]) * tiles_of[k] * share;
  }

  // the border in front of share w, its sequence and place there
  __device__ __forceinline__ Share border(int w, int& seq, int& place) const {
    seq = place = 0;
    if (w <= 0) return Share{first_tile<M>(0, a.G, 0), 0};
    if (w >= count) return Share{END, 0};
    const int x = w * share;
    int lane_from = from, lane_upto = upto, y = 0, front = 0, tiles;
    int each[LISTS];
#pragma unroll
    for (int k = 0; k < LISTS; ++k) each[k] = mine[k];
    for (int b0 = 0; b0 <= a.B; b0 += 64 * LISTS) {
      if (b0 > 0) {
        int sum = 0;
#pragma unroll
        for (int k = 0; k < LISTS; ++k) {
          each[k] = cost(b0 + lane_id() * LISTS + k, tiles);
          each[k] *= tiles;
          sum += each[k];
        }
        lane_upto = front + wave_scan(sum);
        lane_from = lane_upto - sum;
      }
      const unsigned long long past = __builtin_amdgcn_ballot_w64(lane_upto > x);
      if (past) {
        const int l = __builtin_ctzll(past);
        int at = lane_from, k = 0;  // the lane's sequence that x falls into
#pragma unroll
        for (int i = 0; i < LISTS - 1; ++i)
          if (k == i && at + each[i] <= x) {
            at += each[i];
            k = i + 1;
          }
        seq = min(b0 + l * LISTS + __builtin_amdgcn_readlane(k, l), a.B);
        y = x - __builtin_amdgcn_readlane(at, l);
        break;
      }
      front = __builtin_amdgcn_readlane(lane_upto, 63);
    }
    const int tile_cost = cost(seq, tiles);
    place = place_in(y, tile_cost, tiles);
    y -= place * tile_cost;
    const int number = first_tile<M>(seq_start(a.cu_q, seq, a.B, a.Tq), a.G, seq) + place;
    const float snap = SNAP * (float)share;
    if (whole ? 2 * y <= tile_cost : (float)y < snap) return Share{number, 0};
    if (whole || (float)(tile_cost - y) < snap) {
      ++place;
      return Share{number + 1, 0};
    }
    const int rows = paged_rows_of(a, seq), nk = paged_keys_of(a, seq), nq = divide(a.div_g, rows);
    const int len = seq < a.B ? max(a.lens[seq], 0) : 0, last = min((place + 1) * M, rows) - 1;
    const int seen = a.causal ? min(max(divide(a.div_g, last) + 1 - nq + len, 0), nk) : nk;
    const int chunks = (seen + BK - 1) / BK;
    return Share{number, max(min((int)((float)y / (float)tile_cost * (float)chunks), chunks - 1), 0)};
  }
};

// grid: shares * Hk, a share's heads on neighbouring workgroups (workgroup i runs on XCD i % 8: with eight kv heads each XCD's L2
// then holds one head's keys)
template <int D, int BITS, int M>
__global__ __launch_bounds__(256, ES_PAGED_RESIDENT(D, M)) void paged_shares_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[paged_lds<D, M>()];
  __shared__ float stats[4 * 128];
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  const Shares<M> shares(a);
  int seq, place, other_seq, other_place;
  const Share from = shares.border(w, seq, place), to = shares.border(w + 1, other_seq, other_place);
  if (hk == 0 && threadIdx.x == 0) {
    int4* borders = reinterpret_cast<int4*>(a.plan);
    const int rows = from.chunk > 0 ? min(paged_rows_of(a, seq) - place * M, M) : 0;  // (of a cut tile)
    borders[w] = make_int4(from.tile, from.chunk, seq_start(a.cu_q, seq, a.B, a.Tq), 64 * place + rows);
    if (w == a.shares - 1) borders[w + 1] = make_int4(END, 0, 0, 0);
  }
  int tile = __builtin_amdgcn_readfirstlane(from.tile), chunk = __builtin_amdgcn_readfirstlane(from.chunk);
  const int last_tile = __builtin_amdgcn_readfirstlane(to.tile), last_chunk = __builtin_amdgcn_readfirstlane(to.chunk);
  if (tile == END) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  place = __builtin_amdgcn_readfirstlane(place);
  while (seq <= a.B && (tile < last_tile || (tile == last_tile && chunk < last_chunk))) {
    const Seq s = sequence(a.cu_q, nullptr, a.B, a.Tq, 0, seq);
    if (place * M >= s.nq * a.G) {
      ++seq;
      place = chunk = 0;
      if (seq <= a.B) tile = first_tile<M>(__builtin_amdgcn_readfirstlane(seq_start(a.cu_q, seq, a.B, a.Tq)), a.G, seq);
      continue;
    }
    Job j;
    paged_job<D, BITS>(a, j, s.q0, s.nq, seq, cached_keys(a, seq), keys_over(a, seq), hk);
    j.r0 = place * M;
    const int chunks = tile_chunks<M>(a, j);
    j.c0 = min(chunk, chunks);
    j.c1 = tile == last_tile ? min(last_chunk, chunks) : chunks;
    j.part_rows = M;
    j.part = j.c0 == 0 && j.c1 == chunks ? nullptr : partial<D>(a.part, M, a, 2 * w + (j.c0 == 0), hk);
    if (j.part == nullptr || j.c0 < j.c1) {
      paged_tile<D, BITS, M>(a, j, lds, stats);
      __syncthreads();
    }
    ++place;
    ++tile;
    chunk = 0;
  }
}

// O of rows r0 + 0 .. of a tile that was cut: sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over the n pieces, whose partials (M
// rows each) are numbered in `pieces`. D / 4 lanes a row and piece, SIDE pieces of a row side by side, each side with a maximum of
// its own, the sides added in order. A workgroup does merge_rows_of(D, SIDE) rows.
constexpr int merge_rows_of(int D, int side) { return 256 / (D / 4 * side); }
template <int D, int M, int SIDE>
__device__ __forceinline__ void merge_rows(const FwdArgs& a, const int* pieces, int n, int hk, int q0, int row0, int r0, int rows) {
  constexpr int LPR = D / 4, RPB = merge_rows_of(D, SIDE);
  const int lane = threadIdx.x % LPR, c = lane * 4, side = threadIdx.x / LPR % SIDE, local = threadIdx.x / (LPR * SIDE);
  const int r = min(r0 + local, rows - 1);
  float top = -INFINITY, sum = 0.0f;
  f32x4 acc = {};
  for (int i = side; i < n; i += 4 * SIDE) {  // (four pieces in flight)
    f32x4 o[4];
    float m[4], z[4], most = top;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = f32x4{};
      m[e] = -INFINITY;
      z[e] = 0.0f;
      if (i + e * SIDE >= n) continue;
      const float* p = partial<D>(a.part, M, a, pieces[i + e * SIDE], hk);
      o[e] = *reinterpret_cast<const f32x4*>(p + 2 * M + r * D + c);
      m[e] = p[r];
      z[e] = p[M + r];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) most = fmaxf(most, m[e]);
    if (most == -INFINITY) continue;
    const float old = exp2f_fast(top - most);
    acc *= old;
    sum *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = exp2f_fast(m[e] - most);
      acc += f * o[e];
      sum = fmaf(f, z[e], sum);
    }
    top = most;
  }
  if constexpr (SIDE > 1) {
    __shared__ f32x4 sums[SIDE][RPB][LPR];
    __shared__ float2 weights[SIDE][RPB];  // maximum, sum
    sums[side][local][lane] = acc;
    if (lane == 0) weights[side][local] = make_float2(top, sum);
    __syncthreads();
    if (side != 0) return;
    float2 s[SIDE];
#pragma unroll
    for (int i = 0; i < SIDE; ++i) {
      s[i] = weights[i][local];
      top = fmaxf(top, s[i].x);
    }
    acc = f32x4{};
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < SIDE; ++i) {
      const float f = s[i].x == -INFINITY ? 0.0f : exp2f_fast(s[i].x - top);
      acc += f * sums[i][local][lane];
      sum = fmaf(f, s[i].y, sum);
    }
  }
  if (r0 + local >= rows) return;
  const int row = row0 + r, tok = divide(a.div_g, row);
  const size_t at = ((size_t)(q0 + tok) * a.Hk + hk) * a.G + (row - tok * a.G);
  store_row<D>(a, at, c, acc * (sum == 0.0f ? 0.0f : 1.0f / sum));
  if (c == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top - P_SHIFT + log2f(sum)) * PK_LN2;
}

// Tiles that were cut. Grid: (borders * Hk, rows of a tile / rows of a workgroup): the first border within a tile has it merged,
// so the launch does not grow with the sequences, most of whose tiles are whole, and a border says all that is to be known of its
// tile: one load a lane, then the pieces' (256 tokens against 2000 keys, 32 heads over 8: attention 397 us with a workgroup a tile,
// 365 so; one sequence of 75600 keys among 49, whose tile has half of the borders: 8 us piece after piece, 4.7 so).
template <int D, int M>
__global__ __launch_bounds__(256) void merge_shares_kernel(FwdArgs a) {
  constexpr int RPB = merge_rows_of(D, 4);
  const int w = blockIdx.x / a.Hk + 1, hk = blockIdx.x - (w - 1) * a.Hk, l = lane_id();
  const int4* borders = reinterpret_cast<const int4*>(a.plan);
  int4 x = borders[min(w - 1 + l, a.shares)];
  const int tile = __builtin_amdgcn_readlane(x.x, 1), r0 = blockIdx.y * RPB;
  const bool again = __builtin_amdgcn_readlane(x.x, 0) == tile && __builtin_amdgcn_readlane(x.y, 0) > 0;
  if (__builtin_amdgcn_readlane(x.y, 1) == 0 || again) return;
  const int q0 = __builtin_amdgcn_readlane(x.z, 1), place = __builtin_amdgcn_readlane(x.w, 1), rows = place % 64, t = place / 64;
  if (r0 >= rows) return;
  // the shares that have a piece of it, in order: the one before the border the beginning, in its second slot, the others in their
  // first; two borders may stand at one place
  __shared__ int pieces[256 * ES_PAGED_RESIDENT(D, M) + 1];
  if (threadIdx.x == 0) pieces[0] = 2 * (w - 1) + 1;
  int n = 1;
  for (int i0 = w - 1;; i0 += 62) {  // (lanes 1 to 62, which see the next border)
    if (i0 >= w) x = borders[min(i0 + l, a.shares)];
    const int next = __shfl(x.x, min(l + 1, 63), 64), next_chunk = __shfl(x.y, min(l + 1, 63), 64);
    const bool within = l >= 1 && l <= 62 && i0 + l < a.shares && x.x == tile;
    const bool mine = within && (next != tile || next_chunk > x.y);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(mine);
    if (mine && threadIdx.x < 64) pieces[n + __builtin_popcountll(hit & ((1ull << l) - 1))] = 2 * (i0 + l);
    n += __builtin_popcountll(hit);
    if (!__builtin_amdgcn_readlane((int)within, 62)) break;
  }
  __syncthreads();
  merge_rows<D, M, 4>(a, pieces, n, hk, q0, t * M, r0, rows);
}

// ------------------------------------------------------------------------------------------------ wide tiles: pieces
// Launches with wide tiles are bound by the matrix units, and tiles that read the same keys side by side have them from L2: tiles
// are cut into pieces (paged_rules.h) that fill the GPU about once, one level of all tiles after the other. (Equal shares, whose
// pieces start anywhere: 4096 tokens of 32 heads over 8 alone 228 us, pieces 155. One count of ranges for all tiles of a sequence,
// as packed_tiles.h has it, which takes a causal prompt for twice its work: prompts of 3923, 938 and 3440 tokens, 8 heads of 64
// over one, 114 us, pieces 79; 256 and 512 tokens over 9000 and 512 keys beside two small ones, 24 heads over 8, 65 and 56.)
// P goes into the products of wide tiles as one 16-bit value: errors are 1.3 to 1.4 times those of its own rounding of the output.
// With what the rounding leaves as a second product (narrow tiles) they are not, but 256 to 512 tokens over 9000 keys take 68 us
// instead of 55, 700 over 16384 315 instead of 241, 32760 causal ones 8280 instead of 5980.
// Every wave derives the cut from the lengths by itself, so they stay on the device: of sizes from the fair share on the one with
// the shortest schedule, by a model of it. Items over three quarters of the largest come first, then those over a half, over a
// quarter and the rest, since workgroups are dispatched in order. Lanes have LISTS sequences each, 64 apart; more than 64 * LISTS
// are read once a pass and keep their order.
struct WideItem {
  int list, tile, level, piece, number, per;  // list < 0: none; number: within its class and list
};
// What the first workgroup leaves for the merge, behind it (first partial, first cut tile) of each list.
struct WidePlan {
  int per, cut_tiles;
};
struct Wide {
  WideList x;
  int q0, nq;
  __device__ __forceinline__ int keys(const FwdArgs& a) const { return min(nq - x.behind, a.paged.cap); }
  __device__ __forceinline__ int over(const FwdArgs& a) const { return nq - x.behind - keys(a); }
};
__device__ __forceinline__ Wide wide_of(const FwdArgs& a, int b) {
  Wide w;
  w.q0 = seq_start(a.cu_q, b, a.B, a.Tq);
  w.nq = max((b < a.B ? seq_start(a.cu_q, b + 1, a.B, a.Tq) : a.Tq) - w.q0, 0);
  const int rows = w.nq * a.G, len = b < a.B ? max(a.lens[b], 0) : 0, head = divide(a.div_g, max(min(rows, TILE) - 1, 0)) + 1;
  w.x = wide_list(rows, w.nq, len, min(len, a.paged.cap), head, a.causal);
  return w;
}
// lane `from`'s
__device__ __forceinline__ Wide wide_at(const Wide& w, int from) {
  auto at = [&](int v) { return __builtin_amdgcn_readlane(v, from); };
  return Wide{WideList{at(w.x.rows), at(w.x.tiles), at(w.x.chunks), at(w.x.behind), at(w.x.first)}, at(w.q0), at(w.nq)};
}
// sums of a row of sixteen lanes, on its last one
__device__ __forceinline__ float row_sum(float x) {
  x += __int_as_float(dpp_i<0x111>(__float_as_int(x)));
  x += __int_as_float(dpp_i<0x112>(__float_as_int(x)));
  x += __int_as_float(dpp_i<0x114>(__float_as_int(x)));
  return x + __int_as_float(dpp_i<0x118>(__float_as_int(x)));
}
// x, held to the workspace whatever counts a call has
__device__ __forceinline__ int within(int x, int n) { return (int)min((unsigned)x, (unsigned)(n - 1)); }
constexpr int CUTS = 16;  // sizes of pieces that are looked at
// A plan, page numbers and first keys take about 8 us, a chunk 2.1, with D = 64 1.1; a merge 5 more where tiles are cut.
template <int D>
constexpr float START = D == 128 ? 3.5f : 7.0f;
template <int D>
struct WideLists {
  const FwdArgs& a;
  int lists, classes;
  bool few;  // a row of sixteen lanes has all lists, each row the same
  Wide mine[LISTS];

  __device__ __forceinline__ Wide load(int i) const { return i < lists ? wide_of(a, i) : Wide{}; }
  __device__ __forceinline__ explicit WideLists(const FwdArgs& args)
      : a(args), lists(args.B + 1), classes(lists <= 64 * LISTS ? 4 : 1), few(lists <= 16) {
    mine[0] = load(few ? lane_id() & 15 : lane_id());
#pragma unroll
    for (int k = 1; k < LISTS; ++k) mine[k] = 64 * k < lists ? load(64 * k + lane_id()) : Wide{};
  }
  // each list once
  __device__ __forceinline__ WideList at(int i0, int k) const {
    if (i0 > 0) return load(i0 + 64 * k + lane_id()).x;
    return few && lane_id() >= 16 ? WideList{} : mine[k].x;
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i0 = 0; i0 < lists; i0 += 64 * LISTS) {
#pragma unroll
      for (int k = 0; k < LISTS; ++k)
        if (i0 + 64 * k < lists) f(at(i0, k));
    }
  }
  // items of at most this many chunks are in a class behind class k
  __device__ __forceinline__ int bound(int longest, int k) const { return classes == 1 ? -1 : longest * (3 - k) / 4; }

  struct Load {
    float big, small, later;  // items of class 0, the others' time, pieces above level 0
  };
  __device__ __forceinline__ void add(Load& s, const WideList& x, int per) const {
    const int rest = tiles_within(x, a.G, a.causal, bound(per, 0)), more = later_pieces(x, a.G, a.causal, piece_of(x, per));
    s.big += (float)(x.tiles - rest + more);
    s.small += (float)rest * (0.5f * (float)(min(x.first, x.chunks) + min(x.chunks, bound(per, 0))) + START<D>);
    s.later += (float)more;
  }

  // Chunks a piece. The waves look at some sizes each, with up to 16 lists each row of lanes at one. times: [CUTS] in LDS.
  __device__ __forceinline__ int cut(float* times) const {
    float sum = 0.0f, top = 0.0f;
    each([&](const WideList& x) {
      sum += (float)x.tiles * (0.5f * (float)(x.first + x.chunks) + 0.5f);
      top = fmaxf(top, x.tiles > 0 ? (float)x.chunks : 0.0f);
    });
    const int most = max((int)wave_max_dpp(top), 1);
    const float mean = wave_sum_dpp(sum) * a.inv_slots;
    const int least = max((int)ceilf(fminf(mean, (float)most)), 4);
    if (least >= most) return most;
    const int wave = threadIdx.x >> 6;
    auto size = [&](int i) { return i < CUTS - 1 ? min(least + (least * i + 11) / 12, most) : most; };  // (at last: no tile is cut)
    auto time = [&](const Load& s, int per) {
      const float t = wide_time(s.big, (float)per, s.small, mean, s.later > 0.0f, START<D>, a.inv_slots);
      return s.later <= (float)(a.items - a.tiles) ? t : INFINITY;
    };
    if (few) {
      const int i = 4 * wave + (lane_id() >> 4), per = size(i);
      Load s = {};
      add(s, mine[0].x, per);
      s.big = row_sum(s.big);
      s.small = row_sum(s.small);
      s.later = row_sum(s.later);
      if ((lane_id() & 15) == 15) times[i] = time(s, per);
    } else {
      for (int i = wave; i < CUTS; i += 4) {
        // many lists, each read once a size: one beside no cut, a wave each (600 sequences of two tokens, 16 heads over 4, 244 us
        // with all sizes, 184 so)
        if (classes == 1 && i < CUTS - 2) {
          if (lane_id() == 0) times[i] = INFINITY;
          continue;
        }
        const int per = size(i);
        Load s = {};
        each([&](const WideList& x) { add(s, x, per); });
        s.big = wave_sum_dpp(s.big);
        s.small = wave_sum_dpp(s.small);
        s.later = wave_sum_dpp(s.later);
        if (lane_id() == 0) times[i] = time(s, per);
      }
    }
    __syncthreads();
    int best = most;
    float shortest = times[CUTS - 1];
#pragma unroll
    for (int i = 0; i < CUTS - 1; ++i) {
      const float t = times[i];
      if (t < shortest) {
        shortest = t;
        best = size(i);
      }
    }
    return __builtin_amdgcn_readfirstlane(best);
  }

  __device__ __forceinline__ int cut_tiles_of(const WideList& x, int per) const {
    return x.tiles - tiles_within(x, a.G, a.causal, piece_of(x, per));
  }
  __device__ __forceinline__ int parts_of(const WideList& x, int per) const {
    return cut_tiles_of(x, per) + later_pieces(x, a.G, a.causal, piece_of(x, per));
  }
  // the partial of an item of a cut tile, all of which are in class 0
  __device__ __forceinline__ int part(const WideItem& item, const WideList& own) const {
    int front = 0;  // partials of this lane's lists in front of the item's
    for (int i0 = 0; i0 < item.list; i0 += 64 * LISTS) {
#pragma unroll
      for (int k = 0; k < LISTS; ++k)
        if (i0 + 64 * k < item.list && i0 + 64 * k + lane_id() < item.list) front += parts_of(at(i0, k), item.per);
    }
    const int level0 = own.tiles - tiles_within(own, a.G, a.causal, bound(item.per, 0));
    front = __builtin_amdgcn_readlane(wave_scan(front), 63);
    return within(front + partial_number(item.number, level0, cut_tiles_of(own, item.per)), a.parts);
  }

  // item w, and its list
  __device__ __forceinline__ WideItem find(int w, float* times, Wide& own) const {
    const int per = cut(times), l = lane_id();
    const bool leave = blockIdx.x == 0 && threadIdx.x < 64;
    int2* plan = a.plan + 1;
    int first = 0, cut_tiles = 0, parts = 0, list = -1, kind = 0, number = 0;
    for (int i0 = 0; i0 < lists; i0 += 64 * LISTS) {
      int upto[LISTS][4], count[LISTS][4], base[4] = {}, all = 0;
#pragma unroll
      for (int k = 0; k < LISTS; ++k) {
        if (i0 + 64 * k >= lists) continue;
        const WideList x = at(i0, k);
        int before = tiles_within(x, a.G, a.causal, bound(per, 0));
        count[k][0] = x.tiles - before + later_pieces(x, a.G, a.causal, piece_of(x, per));
#pragma unroll
        for (int c = 1; c < 4; ++c) {
          const int rest = c < 3 ? tiles_within(x, a.G, a.causal, bound(per, c)) : 0;
          count[k][c] = before - rest;
          before = rest;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          upto[k][c] = wave_scan(count[k][c]);
          base[c] += __builtin_amdgcn_readlane(upto[k][c], 63);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = base[c];
        base[c] = first + all;
        all += n;
      }
#pragma unroll
      for (int k = 0; k < LISTS; ++k) {
        if (i0 + 64 * k >= lists) continue;
        const int i = i0 + 64 * k + l;
        if (leave) {
          const WideList x = at(i0, k);
          const int cuts = cut_tiles_of(x, per), cut_upto = wave_scan(cuts);
          const int own_parts = parts_of(x, per), part_upto = wave_scan(own_parts);
          if (i < lists) plan[i] = make_int2(parts + part_upto - own_parts, cut_tiles + cut_upto - cuts);
          parts += __builtin_amdgcn_readlane(part_upto, 63);
          cut_tiles += __builtin_amdgcn_readlane(cut_upto, 63);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int item0 = base[c] + upto[k][c] - count[k][c];
          base[c] += __builtin_amdgcn_readlane(upto[k][c], 63);
          if (item0 <= w && w < item0 + count[k][c]) list = i, kind = c, number = w - item0;
        }
      }
      first += all;
      if (!leave && __builtin_amdgcn_ballot_w64(list >= 0)) break;
    }
    if (leave && l == 0) *reinterpret_cast<WidePlan*>(a.plan) = WidePlan{per, cut_tiles};
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(list >= 0);
    if (hit == 0) return WideItem{-1};
    const int from = __builtin_ctzll(hit);
    list = __builtin_amdgcn_readlane(list, from);
    kind = __builtin_amdgcn_readlane(kind, from);
    number = __builtin_amdgcn_readlane(number, from);
    if (list < 64) own = wide_at(mine[0], from);
    else own = wide_at(wide_of(a, list), 0);
    const int piece = piece_of(own.x, per);
    WideItem item = {list, 0, 0, 0, number, per};
    if (kind > 0) {
      item.tile = tiles_within(own.x, a.G, a.causal, bound(per, kind - 1)) - 1 - number;
      if (item.tile < 0) item.list = -1;  // (counts that decrease, too many to be added up)
    } else if (!piece_at(own.x, a.G, a.causal, piece, bound(per, 0), number, item.tile, item.level)) {
      item.list = -1;
    }
    item.piece = piece;
    return item;
  }
};

// grid: items * Hk
template <int D, int BITS>
__global__ __launch_bounds__(256, ES_PAGED_RESIDENT(D, TILE)) void paged_pieces_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[paged_lds<D, TILE>()];
  __shared__ float stats[4 * 128];
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  __shared__ float times[CUTS];
  Wide own;
  const WideLists<D> all(a);
  const WideItem item = all.find(w, times, own);
  if (item.list < 0) return;
  Job j;
  paged_job<D, BITS>(a, j, own.q0, own.nq, item.list, own.keys(a), own.over(a), hk);
  j.r0 = item.tile * TILE;
  const int chunks = tile_chunks<TILE>(a, j), n = pieces_of(chunks, item.piece);
  j.c0 = range_begin(chunks, item.level, n);
  j.c1 = range_begin(chunks, item.level + 1, n);
  j.part_rows = TILE;
  j.part = n == 1 ? nullptr : partial<D>(a.part, TILE, a, all.part(item, own.x), hk);
  paged_tile<D, BITS, TILE>(a, j, lds, stats);
}

// Their tiles that were cut, numbered list by list, the last ones first. Grid: (as many as there can be * Hk, parts of their rows).
template <int D>
__global__ __launch_bounds__(256) void merge_pieces_kernel(FwdArgs a) {
  constexpr int MOST = 256 * ES_PAGED_RESIDENT(D, TILE) + 2;  // pieces of a tile: as many as fill the GPU
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  const WidePlan plan = *reinterpret_cast<const WidePlan*>(a.plan);
  int2 first = a.plan[1 + min(lane_id(), a.B)];
  if (w >= plan.cut_tiles) return;
  int list = 0;
  for (int i0 = 0; i0 <= a.B; i0 += 64) {  // the last list that starts at or before w and has cut tiles
    if (i0 > 0) first = a.plan[1 + min(i0 + lane_id(), a.B)];
    const unsigned long long upto = __builtin_amdgcn_ballot_w64(i0 + lane_id() <= a.B && first.y <= w);
    if (upto == 0) break;
    list = i0 + 63 - __builtin_clzll(upto);
    if (!(upto >> 63)) break;
  }
  const int2 left = a.plan[1 + list];
  const Wide own = wide_at(wide_of(a, list), 0);
  const int piece = piece_of(own.x, plan.per), t = __builtin_amdgcn_readfirstlane(own.x.tiles - 1 - (w - left.y));
  if (t < 0) return;
  const int rows = min(own.x.rows - t * TILE, TILE), last = divide(a.div_g, t * TILE + rows - 1);
  const int seen = a.causal ? min(max(last + 1 - own.x.behind, 0), own.keys(a)) : own.keys(a);
  const int n = min(pieces_of((seen + BK - 1) / BK, piece), MOST);
  __shared__ int pieces[MOST];
  for (int i = threadIdx.x; i < n; i += 256)
    pieces[i] = within(left.x + piece_number(own.x, a.G, a.causal, piece, piece, t, i), a.parts);
  __syncthreads();
  auto merge = [&](auto side) {
    constexpr int S = decltype(side)::value, RPB = merge_rows_of(D, S);
    for (int r0 = blockIdx.y * RPB; r0 < rows; r0 += gridDim.y * RPB) {
      merge_rows<D, TILE, S>(a, pieces, n, hk, own.q0, t * TILE, r0, rows);
      __syncthreads();
    }
  };
  if (n <= 8) merge(std::integral_constant<int, 1>{});
  else merge(std::integral_constant<int, 4>{});
}

}  // namespace

// What a call launches.
enum PagedForm { WHOLE_TILES, SHARES, PIECES };
struct PagedPlan {
  PagedForm form;
  int M;               // rows a tile
  long long tiles;     // tile numbers of a head
  int shares, items;   // a head: SHARES, PIECES
  int parts;           // a head: PIECES
  size_t plan, bytes;  // workspace: partials, then borders (SHARES) or the cut (PIECES)
};

// `cap`: the keys that a sequence can have, by the width of its table of pages; equal: B sequences of Tq / B tokens. Both are
// what the host knows. Up to 1024 keys a tile is short enough for one workgroup, and a second launch would take as long again.
// Without this form: 4 tokens of 300 keys, 8 heads of 64 over 2, 14.1 us instead of 8.6, of 1000 14.4 instead of 13.2; 48 of 300,
// 32 heads over 8, 27.8 instead of 18.7; a prompt of 1000 34.7 instead of 23.6, eight 113 instead of 115. With it up to 4096 keys:
// 48 tokens of 1500 keys 54 us instead of 62 and a prompt of 1500 36 instead of 48, but 4 tokens of 1500 17 instead of 15, of 2500
// 26 instead of 15. A table that is wider than the histories need pays for the cut: 4 tokens of 1 to 300 keys with one of 32768
// 13.3 us instead of 8.0, 48 of 300 27 instead of 18, eight prompts of 1000 108 instead of 99. So does one more token than
// sequences, which makes all tiles wide: 48 tokens of 1 to 16000 keys 302 us, with one more 317; over 4 bits 96 and 129.
static PagedPlan paged_plan(int B, int Tq, int cap, int H, int Hk, int D, int bits, bool equal) {
  PagedPlan p = {};
  const int G = H / Hk, narrow = bits == 4 ? TOKENS<4> : TOKENS<16>;
  // single tokens (with running counts: no more tokens than sequences) and the like whose rows fit a narrow tile
  const bool tokens = (equal ? (long long)(Tq / B) * G : Tq <= B ? G : narrow + 1) <= narrow;
  p.M = tokens ? narrow : TILE;
  p.tiles = !tokens     ? tile_numbers<TILE>(B, Tq, G)
            : bits == 4 ? tile_numbers<TOKENS<4>>(B, Tq, G)
                        : tile_numbers<TOKENS<16>>(B, Tq, G);
  p.form = cap <= 1024 ? WHOLE_TILES : tokens ? SHARES : PIECES;
  if (p.form == WHOLE_TILES && !tokens && p.tiles * Hk <= (D == 64 ? 768 : 384)) {  // (as for packed sequences)
    p.M = TILE / 2;
    p.tiles = tile_numbers<TILE / 2>(B, Tq, G);
  }
  const int slots = 256 * ES_PAGED_RESIDENT(D, p.M);
  if (p.form == SHARES) {
    p.shares = std::max(slots / Hk, 1);
    p.plan = (size_t)2 * p.shares * Hk * part_floats(p.M, D) * sizeof(float);
    p.bytes = p.plan + (size_t)(p.shares + 1) * sizeof(int4);
  } else if (p.form == PIECES) {
    // later pieces as many as fill the GPU (WideLists::cut); only cut tiles have partials (75600 tokens of 40 heads over 8: 69 MB
    // instead of the 1.6 GB of one for every tile)
    const int later = slots / Hk + 1;
    p.items = (int)(p.tiles + later);
    p.parts = (int)most_partials(p.tiles, later);
    p.plan = (size_t)p.parts * Hk * part_floats(p.M, D) * sizeof(float);
    p.bytes = p.plan + sizeof(WidePlan) + (size_t)(B + 1) * sizeof(int2);
  }
  return p;
}

#ifndef ES_ELEM_F16
extern "C" size_t es_paged_workspace(int B, int Tq, int max_pages, int page_size, int H, int Hk, int D, int bits) {
  if (B <= 0 || Tq <= 0 || max_pages < 0 || page_size <= 0 || H <= 0 || Hk <= 0 || H % Hk || (D != 64 && D != 128)) return 0;
  const int cap = (int)std::min<long long>((long long)max_pages * page_size, 1LL << 30);
  const size_t a = paged_plan(B, Tq, cap, H, Hk, D, bits, false).bytes;  // (with and without running counts)
  return std::max(a, paged_plan(B, Tq, cap, H, Hk, D, bits, true).bytes);
}
#endif

static int paged_fwd(FwdArgs& a, const void* q, const int* pages, const int* lens, const int* cu, void* out, float* lse,
                     void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages, int num_pages, int page_size, int H,
                     int Hk, int D, int causal, float scale, int bits, hipStream_t stream) {
  if (int st = places_check(pages, lens, cu, B, Tq, max_pages, num_pages, page_size, Hk)) return st;
  if (int st = packed_check(q, nullptr, nullptr, cu, lens, nullptr, nullptr, 0, 0, B, Tq, 0, H, Hk, D, scale)) return st;
  if (Tq == 0) return ES_OK;
  ES_REQUIRE(out && lse, ES_ERR_INVALID, "paged: null out / lse");
  ES_REQUIRE(aligned16({q, out, workspace}), ES_ERR_INVALID, "paged: tensors must be aligned to 16 bytes");
  a.q = (const e16_t*)q;
  a.cu_q = cu;
  a.out = (e16_t*)out;
  a.lse = lse;
  a.lens = lens;
  a.B = B;
  a.Tq = Tq;
  a.H = H;
  a.Hk = Hk;
  a.G = H / Hk;
  a.div_g = fast_div(a.G);
  a.causal = causal != 0;
  a.scale = scale * LOG2E;
  a.paged.table = pages;
  a.paged.max_pages = max_pages;
  a.paged.num_pages = num_pages;
  a.paged.shift = log2_of(page_size);
  a.paged.cap = num_pages > 0 ? max_pages * page_size : 0;  // (without pages no sequence has keys)
  const PagedPlan p = paged_plan(B, Tq, max_pages * page_size, H, Hk, D, bits, cu == nullptr);
  a.tiles = (int)p.tiles;
  ES_REQUIRE(p.tiles * Hk < MAX_GRID && (long long)p.items * Hk < MAX_GRID, ES_ERR_UNSUPPORTED, "paged: too many sequences");
  ES_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes), ES_ERR_INVALID, "paged: workspace too small");
  a.part = (float*)workspace;
  a.plan = (int2*)((char*)workspace + p.plan);
  a.items = p.form == SHARES ? 2 * p.shares : p.items;
  a.shares = p.shares;
  a.parts = p.parts;
  a.inv_slots = (float)Hk / (float)(256 * ES_PAGED_RESIDENT(D, p.M));
  // sixteenths of a chunk, or as much more as it takes for all costs of a head to stay below 2^29
  a.cost_unit = (float)std::min(16.0, (double)(1 << 29) / ((double)p.tiles * ((double)a.paged.cap / BK + TILE_COST)));
  a.least_share = std::max((int)(LEAST * a.cost_unit), 1);
  const long long rows_most = std::min<long long>((long long)Tq * a.G, p.M);
  auto launch = [&](auto dim, auto bit, auto rows) {
    constexpr int d = decltype(dim)::value, n = decltype(bit)::value, m = decltype(rows)::value;
    if constexpr (m == TOKENS<n>) {
      if (p.form == SHARES) {
        hipLaunchKernelGGL((paged_shares_kernel<d, n, m>), dim3((unsigned)(p.shares * Hk)), dim3(256), 0, stream, a);
        if (p.shares > 1)
          hipLaunchKernelGGL((merge_shares_kernel<d, m>),
                             dim3((unsigned)((p.shares - 1) * Hk), (unsigned)((rows_most * d + 255) / 256)), dim3(256), 0,
                             stream, a);
        return;
      }
    } else if constexpr (m == TILE) {
      if (p.form == PIECES) {
        hipLaunchKernelGGL((paged_pieces_kernel<d, n>), dim3((unsigned)(p.items * Hk)), dim3(256), 0, stream, a);
        // a tile's rows are shared out over more workgroups, down to one pass each, where the tiles are few (15 sequences of 16
        // tokens, 16 heads over 2, up to 13269 keys: merge 10.0 us with 16 workgroups a tile, 5.0 with 64)
        const long long cuts = std::min<long long>(p.tiles, p.items - p.tiles) * Hk;
        const long long few = merge_rows_of(d, 4), many = merge_rows_of(d, 1);
        const long long parts = std::min((rows_most + few - 1) / few, std::max((rows_most + many - 1) / many, 2048 / cuts));
        hipLaunchKernelGGL((merge_pieces_kernel<d>), dim3((unsigned)cuts, (unsigned)parts), dim3(256), 0, stream, a);
        return;
      }
    }
    hipLaunchKernelGGL((paged_whole_kernel<d, n, m>), dim3((unsigned)(p.tiles * Hk)), dim3(256), 0, stream, a);
  };
  using std::integral_constant;
  auto with_bits = [&](auto dim) {
    auto with_rows = [&](auto bit) {
      if (p.M == TILE) launch(dim, bit, integral_constant<int, TILE>{});
      else if (p.M == TILE / 2) launch(dim, bit, integral_constant<int, TILE / 2>{});
      else launch(dim, bit, integral_constant<int, TOKENS<decltype(bit)::value>>{});
    };
    if (bits == 16) with_rows(integral_constant<int, 16>{});
    else with_rows(integral_constant<int, 4>{});
  };
  if (D == 64) with_bits(integral_constant<int, 64>{});
  else with_bits(integral_constant<int, 128>{});
  return check_launch("es_paged_fwd");
}

}  // namespace es

using namespace es;

extern "C" int ES_VSA_API(es_paged_fwd)(const void* q, const void* k_pages, const void* v_pages, const int* pages,
                                        const int* lens, const int* cu, void* out, float* lse, void* workspace,
                                        size_t workspace_bytes, int B, int Tq, int max_pages, int num_pages, int page_size, int H,
                                        int Hk, int D, int causal, float scale, long long page_stride, long long head_stride,
                                        long long row_stride, hipStream_t stream) {
  if (int st = cache_check(k_pages, v_pages, num_pages, page_size, Hk, D, page_stride, head_stride, row_stride)) return st;
  FwdArgs a = {};
  a.paged.k = (const e16_t*)k_pages;
  a.paged.v = (const e16_t*)v_pages;
  a.paged.page_stride = page_stride, a.paged.head_stride = head_stride, a.paged.row_stride = row_stride;
  return paged_fwd(a, q, pages, lens, cu, out, lse, workspace, workspace_bytes, B, Tq, max_pages, num_pages, page_size, H, Hk, D,
                   causal, scale, 16, stream);
}

extern "C" int ES_VSA_API(es_paged4_fwd)(const void* q, const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                                         const uint8_t* v_scales, const int* pages, const int* lens, const int* cu, void* out,
                                         float* lse, void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages,
                                         int num_pages, int page_size, int H, int Hk, int D, int causal, float scale,
                                         hipStream_t stream) {
  if (int st = cache4_check(k_codes, k_scales, v_codes, v_scales, num_pages)) return st;
  FwdArgs a = {};
  a.paged.codes[0] = k_codes, a.paged.codes[1] = v_codes;
  a.paged.scales[0] = k_scales, a.paged.scales[1] = v_scales;
  return paged_fwd(a, q, pages, lens, cu, out, lse, workspace, workspace_bytes, B, Tq, max_pages, num_pages, page_size, H, Hk, D,
                   causal, scale, 4, stream);
}
