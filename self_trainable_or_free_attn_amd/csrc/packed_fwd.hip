// Forward of attention over packed sequences and over a shared prefix (gfx950, MFMA 32x32x16, bf16 / fp16).
//
// One workgroup of four waves owns a tile of up to 128 (small grids: 64) rows of (token, head in group) (packed.h) and
// streams the keys its rows see in 64-key chunks, online softmax: S^T = K Q^T, so that exp(S^T) is the B operand of O^T +=
// V^T P^T.
//   wide tiles (more than 32 rows): each wave has 32 rows; a chunk is staged once in LDS for all four, the next one's
//     transfers in flight under its products. With 64 rows two waves share 32 rows and take half of each chunk's keys.
//   narrow tiles (up to 32 rows: single tokens with their head group): every wave has the same 32 rows and takes every
//     fourth run of 32 keys, staged in its own quarter of LDS without a barrier; the four softmax states are merged at the
//     end. The next K run is requested when this one's products have read it, the next V run likewise, so one of them is
//     always in flight.
// What bounds them: wide tiles the matrix units and what runs beside them on long sequences (32760 causal tokens of 24 heads
// over 8, D = 128: 5.94 ms, 1110 TFLOP/s; 57 % of the cycles issue a matrix instruction, 55 % vector work, LDS 29 %, no bank
// conflicts), at D = 64 the vector work (as many exponentials for half the products: 8192 causal tokens of 32 heads 0.33 ms,
// 830 TFLOP/s, 44 % matrix, 77 % vector), the transfers where many tiles stream different keys from HBM, and on sequences of
// a few hundred rows the chain of a tile's few chunks. Narrow tiles: HBM (8 tokens, 40 heads over 8, caches of 513 to 75600
// keys: 654 MB in 137 us, 4.8 TB/s, what a large copy reaches).
// 128 rows a wide tile and not 256 on eight waves: those read K and V half as often, but stop at their barriers together (32760
// causal tokens 6.57 -> 6.95 ms; 13770 of 12 heads without a mask 1433 -> 1360 us).
// Key ranges: with few tiles the chunks of a tile are cut into ranges, one workgroup each, that leave unnormalised partials
// (O, running maximum, sum) in the workspace; merge_kernel adds them in order.
#include "packed.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace es {

namespace {

constexpr float SLACK = 8.0f;  // log2 growth of a row's maximum that triggers a rescale of O and the sum
// fp16 probabilities are taken 2^7 higher (up to 2^15 with the slack), which keeps those down to 2^-21 of the maximum out of
// the type's subnormal range; the shift cancels in O / sum and is taken off the LSE
#ifdef ES_ELEM_F16
constexpr float P_SHIFT = 7.0f;
#else
constexpr float P_SHIFT = 0.0f;
#endif

struct FwdArgs {
  const e16_t *q, *k, *v;
  const int *cu_q, *cu_k, *buckets;
  const float* bias;
  e16_t* out;
  float *lse, *part, *part_prefix;
  FastDiv div_g;
  int B, Tq, Tk, H, Hk, G, R, num_buckets, causal;
  int tiles;        // tile numbers of a head
  int items;        // ranged launches: items of a head
  int2* plan;       // ranged launches: (ranges a tile, first item) of each list
  float inv_slots;  // ranged launches: Hk / the workgroups that the GPU holds at once
  float scale;      // log2(e) * softmax scale
  // shared prefix: rows 0 .. P - 1 of k_prefix / v_prefix are seen by every row
  const e16_t *kp, *vp;
  const int* lens;
  int n, P, S;
  int part_rows;  // rows of a sequence's partial
};

// What one workgroup computes: the tile from row r0 on of the list of nq * G rows that starts at token q0, against key rows
// 0 .. nk - 1 behind k / v (this kv head's first row), chunks c0 .. c1 - 1 of them.
struct Job {
  const e16_t *k, *v;
  int q0, nq, nk, hk, r0, c0, c1, causal;
  float* part;  // a partial of `part_rows` rows; nullptr: finished rows go to out / lse
  int part_rows;
};

// floats of a partial of `rows` rows: m, l, O [D] of each
__host__ __device__ constexpr int part_floats(int rows, int D) { return rows * (D + 2); }

// keys that row r of the job's list sees
__device__ __forceinline__ int keys_seen(const FwdArgs& a, const Job& j, int r) {
  return j.causal ? min(max(divide(a.div_g, r) + 1 + j.nk - j.nq, 0), j.nk) : j.nk;
}
// chunks that any of the M rows of the job's tile sees
template <int M>
__device__ __forceinline__ int tile_chunks(const FwdArgs& a, const Job& j) {
  const int last = min(j.nq * a.G, j.r0 + M) - 1;
  return (keys_seen(a, j, last) + BK - 1) / BK;
}

// A lane's row, its softmax state and the exponentials of a 32-key run of S^T.
template <int D, bool BIAS>
struct Rows {
  ev8 q[D / 16];
  f32x16 o[D / 32];
  float lsum, mrun;
  int seen, pos, gb;  // keys seen, position, the row's part of the bias table
  size_t at;          // row of out / lse
  bool valid;

  __device__ __forceinline__ void load(const FwdArgs& a, const Job& j, int r, int hi) {
    valid = r < j.nq * a.G;
    const int tok = divide(a.div_g, r), g = r - tok * a.G;
    at = ((size_t)(j.q0 + (valid ? tok : 0)) * a.Hk + j.hk) * a.G + (valid ? g : 0);
    seen = valid ? keys_seen(a, j, r) : 0;
    pos = tok + j.nk - j.nq;
    gb = bias_row(a.G, a.R, valid ? g : 0);
    const e16_t* p = a.q + at * D + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const ev8 z = {};
      q[ks] = valid ? *reinterpret_cast<const ev8*>(p + 16 * ks) : z;
    }
#pragma unroll
    for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
    lsum = 0.0f;
    mrun = -INFINITY;
  }

  // The scores of keys key0 .. key0 + 31, s * sc + c: bias and mask put in; masked: some row does not see all of them; low /
  // high: the positions of the wave's rows (bias only). Returns the run's maximum (both half waves of a row together).
  __device__ __forceinline__ float scores(const FwdArgs& a, const float* tab, f32x16& s, int key0, int hi, bool masked, int low,
                                          int high, float& sc, float& c) const {
    sc = a.scale;
    c = 0.0f;
    if (BIAS) {
      if (key0 - high >= a.R) {
        c = tab[gb + a.R];
      } else if (key0 + 31 - low <= -a.R) {
        c = tab[gb - a.R];
      } else {
        add_bias(s, sc, tab + gb, key0 + 4 * hi - (valid ? pos : low), a.G, a.R);  // (a position of the wave's)
        sc = 1.0f;
      }
    }
    if (masked) {
      const int left = seen - key0 - 4 * hi;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 >= left) s[r] = -INFINITY;
    }
    // (the maximum of the products is that of the scores: the scale is positive and the rounding monotone)
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    return fmaf(max_xor32(mx), sc, c);
  }

  // Where a maximum passes the one that the terms are taken against by more than SLACK, that one moves up, by whole powers of
  // two: exact for the float32 sums, and for held probabilities but those that become subnormal in fp16 (below 2^-21 of the
  // row's largest term; half a step there is 2^-32 of it). Returns whether this lane's did; alpha: its factor.
  __device__ __forceinline__ bool raise(float mx, float& alpha) {
    if (!(mx > mrun + SLACK)) return false;
    const float next = mrun == -INFINITY ? mx : mrun + ceilf(mx - mrun);
    alpha = exp2f_fast(mrun - next);
    lsum *= alpha;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    mrun = next;
    return true;
  }

  // p = exp(s - maximum) as two B operands
  __device__ __forceinline__ void exponentials(const f32x16& s, float sc, float c, ev8& pa, ev8& pb) {
    c -= (mrun == -INFINITY ? 0.0f : mrun) - P_SHIFT;
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = exp2f_fast(fmaf(s[r], sc, c));
    pa = epack8(&p[0]);
    pb = epack8(&p[8]);
    // (the sum takes the probabilities before their rounding: the LSE is a float32 result of its own)
    float sum[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
    for (int r = 4; r < 16; ++r) sum[r & 3] += p[r];
    lsum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }

  // O^T += V^T P^T of sixteen keys at `v`
  __device__ __forceinline__ void values(const char* v, int t0, int t1, const ev8& p) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
      o[db] = emfma(ecat_tr(lds_read_tr(v, t0 ^ (64 * db)), lds_read_tr(v, t1 ^ (64 * db))), p, o[db]);
  }
};

// LDS offsets of a lane: K rows (A operand of S^T) at k-step ks: k0 ^ 32 ks; V columns (transposed reads) of channel block
// db: t0 / t1 ^ 64 db (exact: the swizzle is an XOR of the 16-byte chunk)
template <int D>
struct Offsets {
  int k0, t0, t1;
  __device__ __forceinline__ Offsets(int l) {
    const int hi = l >> 5, g1 = (l >> 4) & 1, sub = (l & 1) * 8, row = 4 * hi + ((l & 15) >> 2);
    k0 = tile_at<D>(l & 31, hi);
    t0 = tile_at<D>(row, 2 * g1 + ((l & 3) >> 1)) + sub;
    t1 = tile_at<D>(row + 8, 2 * g1 + ((l & 3) >> 1)) + sub;
  }
};

template <int D>
__device__ __forceinline__ void store_row(const FwdArgs& a, size_t at, int col, f32x4 x) {
  ushort4 v4;
  v4.x = f2e(x[0]); v4.y = f2e(x[1]); v4.z = f2e(x[2]); v4.w = f2e(x[3]);
  *reinterpret_cast<ushort4*>(a.out + at * D + col) = v4;
}

// M = 128: 32 rows a wave; M = 64: two row groups x two key halves, whose softmax states are merged at the end
template <int D, bool BIAS, int M>
__device__ __forceinline__ void wide_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, TILE_BYTES = BK * ROW, NI = D / 32, LPR = D / 8;
  const int tid = threadIdx.x, l = tid & 63, hi = l >> 5, lq = l & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = M == TILE ? wv : wv & 1, kh = M == TILE ? 0 : wv >> 1;
  const int r0 = j.r0 + rg * 32, rows = j.nq * a.G;
  Rows<D, BIAS> x;
  x.load(a, j, r0 + lq, hi);
  const Offsets<D> off(l);
  // this wave's rows: the first one sees the fewest keys, the last one the most
  const int first = min(r0, rows - 1), last = min(r0 + 31, rows - 1);
  const int seen_min = keys_seen(a, j, first), seen_max = r0 < rows ? keys_seen(a, j, last) : 0;
  const int low = divide(a.div_g, first) + j.nk - j.nq, high = divide(a.div_g, last) + j.nk - j.nq;

  // a lane's transfers: NI 1 KB runs of 64 / LPR rows each a wave
  const unsigned stride = (unsigned)a.Hk * D * 2;
  unsigned src[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int R = (wv * NI + i) * (64 / LPR) + l / LPR;
    src[i] = (unsigned)R * stride + (unsigned)(((l % LPR) ^ swizzle<D>(R)) * 16);
  }
  const unsigned lds0 = uni(lds_addr(lds) + (unsigned)wv * (NI * 1024u));
  auto issue = [&](int c, int sb) {
    const size_t row = (size_t)c * BK * a.Hk * D;
    const unsigned bytes = (unsigned)(min(BK, j.nk - c * BK) - 1) * stride + ROW;
    const srd_t rk = make_srd(j.k + row, bytes), rv = make_srd(j.v + row, bytes);
    const unsigned dst = lds0 + (unsigned)sb * (2u * TILE_BYTES);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rk, dst + i * 1024, src[i], 0u);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rv, dst + TILE_BYTES + i * 1024, src[i], 0u);
  };
  if (j.c0 < j.c1) issue(j.c0, 0);
  if (BIAS) fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, j.hk);
  dma_wait();
  __syncthreads();
  for (int c = j.c0; c < j.c1; ++c) {
    const int sb = (c - j.c0) & 1;
    const char* kb = lds + sb * 2 * TILE_BYTES;
    const char* vb = kb + TILE_BYTES;
    // K of the wave's first 32 keys is read before the next chunk's transfers are issued: the first products then find their
    // operands ready
    ev8 kf[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) kf[ks] = elds16(kb + kh * (TILE_BYTES / 2), off.k0 ^ (32 * ks));
    if (c + 1 < j.c1) issue(c + 1, sb ^ 1);
    if (M != TILE) {  // (one priority: raised for the products 1700 causal tokens of 16 heads 30 us, so 28)
      const int key0 = c * BK + 32 * kh;
      if (key0 < seen_max) {
        float sc, c0, alpha;
        ev8 pa, pb;
        f32x16 s0 = {};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s0 = emfma(kf[ks], x.q[ks], s0);
        x.raise(x.scores(a, tab, s0, key0, hi, key0 + 32 > seen_min, low, high, sc, c0), alpha);
        x.exponentials(s0, sc, c0, pa, pb);
        const char* v = vb + kh * (TILE_BYTES / 2);
        x.values(v, off.t0, off.t1, pa);
        x.values(v + TILE_BYTES / 4, off.t0, off.t1, pb);
      }
    } else if (c * BK < seen_max) {
      // Two 32-key runs, one behind the other, so that one's products run while the other's exponentials are taken: S of the
      // second under the exponentials of the first, O += V^T P^T of the first under those of the second. (The first run's
      // probabilities are held back over the second's test of the maximum, and scaled with O where that one moves. Against
      // both S first and each run's exponentials before its own products: 32760 causal tokens, 24 heads 6.39 -> 6.08 ms, 8192
      // at D = 64, 32 heads 345 -> 318 us.) Products run at a raised priority (packed.h): 32760 causal tokens 6.08 -> 5.94
      // ms, 13770 of 12 heads without a mask 1332 -> 1225 us, 8192 causal of 32 heads 541 -> 522. At D = 64 it gains without a
      // mask (13770 of 12 heads 720 -> 705, 4096 of 16 92 -> 84) and loses with one (8192 causal of 32 heads 327 -> 332, 4096 of
      // 24 heads with a bias 78 -> 84): the mask is known at run time only, so both have it.
      const bool masked = (c + 1) * BK > seen_min;
      float sc, c0, c1, alpha;
      ev8 pa, pb, qa, qb;
      f32x16 s0 = {}, s1 = {};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s0 = emfma(kf[ks], x.q[ks], s0);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) kf[ks] = elds16(kb + TILE_BYTES / 2, off.k0 ^ (32 * ks));
      x.raise(x.scores(a, tab, s0, c * BK, hi, masked, low, high, sc, c0), alpha);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s1 = emfma(kf[ks], x.q[ks], s1);
      x.exponentials(s0, sc, c0, pa, pb);
#pragma unroll
      for (int i = 0; i < NKS / 2; ++i) {  // (two products, then what fits beside them)
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 14, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (x.raise(x.scores(a, tab, s1, c * BK + 32, hi, masked, low, high, sc, c1), alpha)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pa[e] = (elem_t)((float)pa[e] * alpha);
          pb[e] = (elem_t)((float)pb[e] * alpha);
        }
      }
      __builtin_amdgcn_s_setprio(1);
      x.values(vb, off.t0, off.t1, pa);
      x.values(vb + TILE_BYTES / 4, off.t0, off.t1, pb);
      x.exponentials(s1, sc, c1, qa, qb);
      x.values(vb + TILE_BYTES / 2, off.t0, off.t1, qa);
      x.values(vb + 3 * (TILE_BYTES / 4), off.t0, off.t1, qb);
      __builtin_amdgcn_s_setprio(0);
    }
    dma_wait();
    __syncthreads();
  }

  float tot = sum_xor32(x.lsum);
  if (M != TILE) {  // the second key half hands its state over: O through the staging buffers, [row group][register][lane]
    float* xch = reinterpret_cast<float*>(lds) + rg * (NDB * 16 * 64);
    if (kh == 1) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) xch[(db * 16 + r) * 64 + l] = x.o[db][r];
      stats[rg * 128 + l] = x.mrun;
      stats[rg * 128 + 64 + l] = tot;
    }
    __syncthreads();
    if (kh == 1) return;
    const float m1 = stats[rg * 128 + l], m = fmaxf(x.mrun, m1), msub = m == -INFINITY ? 0.0f : m;
    const float w0 = exp2f_fast(x.mrun - msub), w1 = exp2f_fast(m1 - msub);
    tot = w0 * tot + w1 * stats[rg * 128 + 64 + l];
    x.mrun = m;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) x.o[db][r] = w0 * x.o[db][r] + w1 * xch[(db * 16 + r) * 64 + l];
  }
  if (M == TILE && j.part != nullptr) {
    const int r = wv * 32 + lq;
    if (r0 >= rows) return;
    float* o = j.part + 2 * j.part_rows;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(o + r * D + 32 * db + 8 * i + 4 * hi) =
            f32x4{x.o[db][4 * i], x.o[db][4 * i + 1], x.o[db][4 * i + 2], x.o[db][4 * i + 3]};
    if (hi == 0) {
      j.part[r] = x.mrun;
      j.part[j.part_rows + r] = tot;
    }
    return;
  }
  if (!x.valid) return;
  const float inv = tot == 0.0f ? 0.0f : 1.0f / tot;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store_row<D>(a, x.at, 32 * db + 8 * i + 4 * hi,
                   f32x4{x.o[db][4 * i], x.o[db][4 * i + 1], x.o[db][4 * i + 2], x.o[db][4 * i + 3]} * inv);
  if (hi == 0) a.lse[x.at] = tot == 0.0f ? -INFINITY : (x.mrun - P_SHIFT + log2f(tot)) * PK_LN2;
}

// up to 32 rows; `lds`: 64 KB of staging, `stats`: [4 waves][m | l][64 lanes]
template <int D, bool BIAS>
__device__ __forceinline__ void narrow_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, RUN = 32 * ROW, NI = D / 16, LPR = D / 8;
  const int tid = threadIdx.x, l = tid & 63, hi = l >> 5, lq = l & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = j.r0, rows = j.nq * a.G;
  Rows<D, BIAS> x;
  x.load(a, j, r0 + lq, hi);
  const Offsets<D> off(l);
  const int last = min(r0 + 31, rows - 1);
  const int seen_min = keys_seen(a, j, r0), seen_max = keys_seen(a, j, last);
  const int low = divide(a.div_g, r0) + j.nk - j.nq, high = divide(a.div_g, last) + j.nk - j.nq;

  const unsigned stride = (unsigned)a.Hk * D * 2;
  unsigned src[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int R = i * (64 / LPR) + l / LPR;
    src[i] = (unsigned)R * stride + (unsigned)(((l % LPR) ^ swizzle<D>(R)) * 16);
  }
  char* kb = lds + wv * 2 * RUN;
  char* vb = kb + RUN;
  const unsigned kd = uni(lds_addr(kb)), vd = uni(lds_addr(vb));
  auto issue = [&](const e16_t* base, int u, unsigned dst) {
    const srd_t rs = make_srd(base + (size_t)u * 32 * a.Hk * D, (unsigned)(min(32, j.nk - u * 32) - 1) * stride + ROW);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rs, dst + i * 1024, src[i], 0u);
  };
  const int end = min(2 * j.c1, (seen_max + 31) / 32);
  int u = 2 * j.c0 + wv;
  if (u < end) {
    issue(j.k, u, kd);
    issue(j.v, u, vd);
  }
  if (BIAS) {
    fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, j.hk);
    __syncthreads();
  }
  for (; u < end; u += 4) {
    const bool more = u + 4 < end;
    wait_transfers<NI>();  // K: all but the V run's transfers
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) s = emfma(elds16(kb, off.k0 ^ (32 * ks)), x.q[ks], s);
    wait_lds();
    if (more) issue(j.k, u + 4, kd);
    ev8 pa, pb;
    float sc, c, alpha;
    x.raise(x.scores(a, tab, s, 32 * u, hi, 32 * (u + 1) > seen_min, low, high, sc, c), alpha);
    x.exponentials(s, sc, c, pa, pb);
    if (more) wait_transfers<NI>();
    else wait_transfers<0>();
    x.values(vb, off.t0, off.t1, pa);
    x.values(vb + RUN / 2, off.t0, off.t1, pb);
    wait_lds();
    if (more) issue(j.v, u + 4, vd);
  }

  // merge of the four waves' states: each wave finishes a quarter of the channels
  wait_transfers<0>();
  float* mine = reinterpret_cast<float*>(lds + wv * 2 * RUN);  // [NDB * 16 registers][64 lanes]
  static_assert(NDB * 16 * 64 * 4 <= 2 * RUN, "a wave's O fits its staging");
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) mine[(db * 16 + r) * 64 + l] = x.o[db][r];
  stats[wv * 128 + l] = x.mrun;
  stats[wv * 128 + 64 + l] = sum_xor32(x.lsum);
  __syncthreads();
  float m[4], w[4], M = -INFINITY, tot = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = stats[i * 128 + l];
    M = fmaxf(M, m[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = m[i] == -INFINITY ? 0.0f : exp2f_fast(m[i] - M);
    tot += w[i] * stats[i * 128 + 64 + l];
  }
  const float inv = j.part != nullptr ? 1.0f : tot == 0.0f ? 0.0f : 1.0f / tot;
#pragma unroll
  for (int e = 0; e < NDB; ++e) {
    const int q4 = wv * NDB + e;  // group of four registers: channels 32 (q4 / 4) + 8 (q4 % 4) + 4 hi ..
    f32x4 acc = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* other = reinterpret_cast<const float*>(lds + i * 2 * RUN);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = fmaf(w[i], other[(q4 * 4 + c) * 64 + l], acc[c]);
    }
    const int col = 32 * (q4 >> 2) + 8 * (q4 & 3) + 4 * hi;
    if (j.part != nullptr) *reinterpret_cast<f32x4*>(j.part + 2 * j.part_rows + lq * D + col) = acc;
    else if (x.valid) store_row<D>(a, x.at, col, acc * inv);
  }
  if (wv == 0 && hi == 0) {
    if (j.part != nullptr) {
      j.part[lq] = M;
      j.part[j.part_rows + lq] = tot;
    } else if (x.valid) {
      a.lse[x.at] = tot == 0.0f ? -INFINITY : (M - P_SHIFT + log2f(tot)) * PK_LN2;
    }
  }
}

template <int D, bool BIAS, int M>
__device__ __forceinline__ void run_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  if (j.nq * a.G - j.r0 <= 32) narrow_tile<D, BIAS>(a, j, lds, stats, tab);
  else wide_tile<D, BIAS, M>(a, j, lds, stats, tab);
}

// whole tiles: grid tiles * Hk, a tile's heads on neighbouring workgroups (workgroup i runs on XCD i % 8: with eight kv heads
// each XCD's L2 then holds one head's keys); under a causal mask a sequence's last tiles, which see the most keys, first
template <int D, bool BIAS, int M>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void packed_fwd_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[4 * BK * D * 2];
  __shared__ float stats[4 * 128];
  __shared__ float tab[BIAS ? BIAS_TABLE : 1];
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  int b, t;
  Seq s;
  Job j;
  if (!tile_of<M, false>(a.cu_q, a.cu_k, a.B, a.Tq, a.Tk, a.G, w, s, b, t)) return;
  j.r0 = ((s.nq * a.G + M - 1) / M - 1 - t) * M;
  j.k = a.k + ((size_t)s.k0 * a.Hk + hk) * D;
  j.v = a.v + ((size_t)s.k0 * a.Hk + hk) * D;
  j.q0 = s.q0;
  j.nq = s.nq;
  j.nk = s.nk;
  j.hk = hk;
  j.causal = a.causal;
  j.part = nullptr;
  j.c0 = 0;
  j.c1 = tile_chunks<M>(a, j);
  run_tile<D, BIAS, M>(a, j, lds, stats, tab);
}

// ------------------------------------------------------------------------------------------------ key ranges
// A ranged launch cuts each tile's chunks into ranges of about the same number of chunks, as many as fill the GPU once.
// Every wave derives the plan from the lengths by itself (a load and some DPP sums a 64 sequences), so the lengths stay on
// the device and no launch is spent on it. `lists` lists of rows, list i with tiles(i) tiles of chunks(i) chunks each:
//   list i has ceil(chunks / per) ranges a tile, `per` at least its fair share, all tiles' chunks * Hk / target (and at least
//   four where a tile has up to 32 rows, eight where it has more and its partial costs more). Among the fair share and the
//   chunk counts that cut the longest list into whole numbers of ranges near it the one with the shortest schedule is taken:
//   the longest item times the rounds that the items over half its size need, or all work evenly spread. At the fair share
//   alone the items may be a few more than the GPU holds, and the last ones take as long again (1280 rows against 32760 keys,
//   8 heads, caches of 16 to 4096: 270 us, with the search 250).
// Items are numbered list by list, tile by tile, range by range; up to 64 lists: those with items over half the longest one's
// size first, since workgroups are dispatched in order. The first workgroup leaves the plan for the merge.
struct ListShape {
  int tiles, chunks, rows;
};
struct Ranges {
  int list, ranges, item0;  // the list, its ranges a tile, its first item
};

// sums of the lanes up to this one (DPP row shifts and broadcasts, as wave_sum_dpp)
template <int CTRL, int ROWMASK = 0xF>
__device__ __forceinline__ int dpp_i(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWMASK, 0xF, true);
}
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_i<0x111>(x);
  x += dpp_i<0x112>(x);
  x += dpp_i<0x114>(x);
  x += dpp_i<0x118>(x);
  x += dpp_i<0x142, 0xA>(x);
  x += dpp_i<0x143, 0xC>(x);
  return x;
}

struct Reciprocal {
  __device__ __forceinline__ float operator()(float x) const { return __builtin_amdgcn_rcpf(x); }
};
__device__ __forceinline__ Cut cut(const ListShape& x, float per) { return Cut(x.tiles, x.chunks, x.rows, per, Reciprocal()); }

// The shapes of the lists, a lane each; up to 64 are read once.
template <class F>
struct Lists {
  const F& shape;
  int lists;
  ListShape mine;
  __device__ __forceinline__ Lists(const F& f, int n) : shape(f), lists(n), mine{0, 0, 0} {
    if (lane_id() < n) mine = f(lane_id());
  }
  __device__ __forceinline__ ListShape at(int i0) const {
    if (i0 == 0) return mine;
    return i0 + lane_id() < lists ? shape(i0 + lane_id()) : ListShape{0, 0, 0};
  }

  // `per`, and the longest item's chunks. (Sums in float32: every wave computes the same ones.)
  __device__ __forceinline__ float range_chunks(const FwdArgs& a, float& longest_item) const {
    float sum = 0.0f, most = 0.0f;
    for (int i0 = 0; i0 < lists; i0 += 64) {
      const ListShape x = at(i0);
      sum += wave_sum_dpp((float)x.tiles * (float)x.chunks);
      most = fmaxf(most, wave_max_dpp(x.tiles > 0 ? (float)x.chunks : 0.0f));
    }
    const float fair = fair_share(sum, a.inv_slots);
    const int near = (int)parts(most, __builtin_amdgcn_rcpf(fair));
    float best = fair, least = INFINITY;
    longest_item = most;
    for (int n = max(near - 2, 1); n <= near; ++n) {
      const float per = fmaxf(parts(most, __builtin_amdgcn_rcpf((float)n)), fair);
      float size = 0.0f, big = 0.0f, work = 0.0f;
      for (int i0 = 0; i0 < lists; i0 += 64) size = fmaxf(size, wave_max_dpp(cut(at(i0), per).size));
      for (int i0 = 0; i0 < lists; i0 += 64) {
        const ListShape x = at(i0);
        const Cut c = cut(x, per);
        const float items = (float)x.tiles * c.ranges;
        big += wave_sum_dpp(2.0f * c.size > size ? items : 0.0f);
        work += wave_sum_dpp(items * c.size);
      }
      const float time = fmaxf(ceilf(big * a.inv_slots) * size, work * a.inv_slots);
      if (time < 0.98f * least) {  // (more ranges for a shorter schedule only)
        least = time;
        best = per;
        longest_item = size;
      }
    }
    return best;
  }

  // the list that holds item w, ranges = 0: none; `plan`: where the first workgroup leaves (ranges, first item) of each list
  __device__ __forceinline__ Ranges find(const FwdArgs& a, int w) const {
    float longest;
    const float per = range_chunks(a, longest);
    const bool leave = blockIdx.x == 0 && threadIdx.x < 64;
    int first = 0;
    Ranges found = {0, 0, 0};
    for (int i0 = 0; i0 < lists; i0 += 64) {
      const ListShape x = at(i0);
      const Cut c = cut(x, per);
      const int i = i0 + lane_id(), ranges = (int)c.ranges, items = i < lists ? x.tiles * ranges : 0;
      const bool late = lists <= 64 && 2.0f * c.size <= longest;
      const int early_upto = wave_scan(late ? 0 : items), early = __builtin_amdgcn_readlane(early_upto, 63);
      const int late_upto = wave_scan(late ? items : 0);
      const int item0 = first + (late ? early + late_upto : early_upto) - items;
      if (leave && i < lists) a.plan[i] = make_int2(ranges, item0);
      const unsigned long long hit = __builtin_amdgcn_ballot_w64(item0 <= w && w < item0 + items);
      if (hit) {
        const int from = __builtin_ctzll(hit);
        found = Ranges{i0 + from, __builtin_amdgcn_readlane(ranges, from), __builtin_amdgcn_readlane(item0, from)};
        if (!leave) break;
      }
      first += early + __builtin_amdgcn_readlane(late_upto, 63);
    }
    return found;
  }
};
__device__ __forceinline__ Ranges planned(const FwdArgs& a, int list) {
  const int2 p = a.plan[list];
  return Ranges{list, __builtin_amdgcn_readfirstlane(p.x), __builtin_amdgcn_readfirstlane(p.y)};
}

// packed sequences: list b, the rows behind the last sequence being list B
struct PackedLists {
  const FwdArgs& a;
  __device__ __forceinline__ ListShape operator()(int b) const {
    const int rows = list_rows(a.cu_q, a.B, a.Tq, a.G, b), nk = list_keys(a.cu_k, a.B, a.Tk, b);
    return ListShape{(rows + TILE - 1) / TILE, (nk + BK - 1) / BK, rows};
  }
};
// shared prefix: list 0 holds all rows of the batch against the prefix, list 1 + b sequence b's rows against its own cache
struct SharedLists {
  const FwdArgs& a;
  __device__ __forceinline__ ListShape operator()(int i) const {
    const int rows = (i == 0 ? a.B * a.n : a.n) * a.G;
    const int nk = i == 0 ? a.P : min(max(a.lens[i - 1], 0), a.S);
    return ListShape{(rows + TILE - 1) / TILE, (nk + BK - 1) / BK, rows};
  }
};

// item w of a list: its job's tile and chunks
__device__ __forceinline__ void take_range(const FwdArgs& a, Job& j, const Ranges& r, int w) {
  const int i = w - r.item0, range = i % r.ranges;
  j.r0 = i / r.ranges * TILE;
  const int chunks = tile_chunks<TILE>(a, j);
  j.c0 = range_begin(chunks, range, r.ranges);
  j.c1 = range_begin(chunks, range + 1, r.ranges);
}

// Partial `item` of a launch, all kv heads of an item side by side. Shared prefix: the prefix's items have a part of their own,
// with whole tiles; those of the sequences are as long as their lists. (Running lengths that decrease, which the header rules
// out, may name more items than the launch has: the merge then reads the last one.)
template <int D>
__device__ __forceinline__ float* partial(float* base, int rows, const FwdArgs& a, int item, int hk) {
  item = min(max(item, 0), a.items - 1);
  return base + ((size_t)item * a.Hk + hk) * part_floats(rows, D);
}

// grid: items * Hk, a token's heads on neighbouring workgroups
template <int D, bool BIAS>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_ranges_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[4 * BK * D * 2];
  __shared__ float stats[4 * 128];
  __shared__ float tab[BIAS ? BIAS_TABLE : 1];
  const int w = blockIdx.x / a.Hk;
  const PackedLists shape{a};
  const Lists<PackedLists> lists(shape, a.B + 1);
  const Ranges r = lists.find(a, w);
  if (r.ranges == 0) return;
  const Seq s = sequence(a.cu_q, a.cu_k, a.B, a.Tq, a.Tk, r.list);
  Job j;
  j.hk = blockIdx.x - w * a.Hk;
  j.k = a.k + ((size_t)s.k0 * a.Hk + j.hk) * D;
  j.v = a.v + ((size_t)s.k0 * a.Hk + j.hk) * D;
  j.q0 = s.q0;
  j.nq = s.nq;
  j.nk = s.nk;
  j.causal = a.causal;
  take_range(a, j, r, w);
  j.part_rows = TILE;
  j.part = r.ranges == 1 ? nullptr : partial<D>(a.part, TILE, a, w, j.hk);
  run_tile<D, BIAS, TILE>(a, j, lds, stats, tab);
}

// A tile of the prefix's list holds rows of several sequences, so a prefix is read once for 128 rows of the batch and not
// once a sequence. Single tokens are HBM bound (the prefix is read once, every cache once). More of them are bound by the
// matrix work of places that are not always filled: 16 samples of 16 tokens, prefix 32760, 40 heads over 8 issue a matrix
// instruction in 37 % of the cycles at 1.43 of 2 waves a SIMD (long whole tiles 57 % at 1.92), though the items' chunks are
// spread within 2 %.
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void shared_prefix_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[4 * BK * D * 2];
  __shared__ float stats[4 * 128];
  const int w = blockIdx.x / a.Hk;
  const SharedLists shape{a};
  const Lists<SharedLists> lists(shape, a.B + 1);
  const Ranges r = lists.find(a, w);
  if (r.ranges == 0) return;
  Job j;
  j.hk = blockIdx.x - w * a.Hk;
  if (r.list == 0) {
    j.k = a.kp + (size_t)j.hk * D;
    j.v = a.vp + (size_t)j.hk * D;
    j.q0 = 0;
    j.nq = a.B * a.n;
    j.nk = a.P;
    j.causal = 0;
  } else {
    const int b = r.list - 1;
    j.k = a.k + ((size_t)b * a.S * a.Hk + j.hk) * D;
    j.v = a.v + ((size_t)b * a.S * a.Hk + j.hk) * D;
    j.q0 = b * a.n;
    j.nq = a.n;
    j.nk = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
    j.causal = 1;
  }
  take_range(a, j, r, w);
  j.part_rows = r.list == 0 ? TILE : a.part_rows;
  j.part = r.list == 0 ? partial<D>(a.part_prefix, TILE, a, w - r.item0, j.hk) : partial<D>(a.part, a.part_rows, a, w, j.hk);
  run_tile<D, false, TILE>(a, j, lds, stats, nullptr);
}

// O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a row's partials in order: D / 4 lanes a row, which first take one
// partial's m and l each and then, eight partials in flight, four channels each. SHARED: a row's prefix partials, then those
// of its own cache. Grid: (tile numbers * Hk, merge_rows). Latency bound: 4 to 12 us.
template <int D, bool SHARED>
__global__ __launch_bounds__(256) void merge_kernel(FwdArgs a) {
  constexpr int LPR = D / 4, RPB = 256 / LPR;
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk;
  int list, t, q0, nq;
  Ranges own, pre = {0, 0, 0};
  if (SHARED) {
    const int tiles = (a.n * a.G + TILE - 1) / TILE;
    list = 1 + w / tiles;
    t = w % tiles;
    q0 = (list - 1) * a.n;
    nq = a.n;
    if (t * TILE + (int)blockIdx.y * RPB >= nq * a.G) return;
    own = planned(a, list);
    pre = planned(a, 0);
  } else {
    list = seq_of_tile<TILE>(a.cu_q, a.B, a.Tq, a.G, w);
    const Seq s = sequence(a.cu_q, a.cu_k, a.B, a.Tq, a.Tk, list);
    q0 = s.q0;
    nq = s.nq;
    t = w - first_tile<TILE>(q0, a.G, list);
    if (t < 0 || t * TILE + (int)blockIdx.y * RPB >= nq * a.G) return;
    own = planned(a, list);
    if (own.ranges == 1) return;  // (finished by its only range)
  }
  const int rows = min(nq * a.G - t * TILE, TILE), lane = threadIdx.x % LPR, c = lane * 4, n = pre.ranges + own.ranges;
  const int own_rows = SHARED ? a.part_rows : TILE;
  for (int r = blockIdx.y * RPB + threadIdx.x / LPR; r < rows; r += gridDim.y * RPB) {
    const int all = q0 * a.G + t * TILE + r, rp = SHARED ? all % TILE : 0;  // the row among all rows of the batch
    // a row's partial i: m at [row], l at [rows + row], O behind them
    auto part = [&](int i, int& stored, int& row) -> const float* {
      const bool p = SHARED && i < pre.ranges;
      stored = p ? TILE : own_rows;
      row = p ? rp : r;
      return p ? partial<D>(a.part_prefix, TILE, a, all / TILE * pre.ranges + i, hk)
               : partial<D>(a.part, own_rows, a, own.item0 + t * own.ranges + i - pre.ranges, hk);
    };
    int stored, row;
    float M = -INFINITY;
    for (int i = lane; i < n; i += LPR) {
      const float* p = part(i, stored, row);
      M = fmaxf(M, p[row]);
    }
#pragma unroll
    for (int m = LPR / 2; m >= 1; m >>= 1) M = fmaxf(M, __shfl_xor(M, m, 64));
    const float msub = M == -INFINITY ? 0.0f : M;
    f32x4 acc = {};
    float sum = 0.0f;
    for (int i0 = 0; i0 < n; i0 += LPR) {
      const int count = min(n - i0, LPR);
      float f = 0.0f, l = 0.0f;
      if (lane < count) {
        const float* p = part(i0 + lane, stored, row);
        f = exp2f_fast(p[row] - msub);
        l = p[stored + row];
      }
      for (int i = 0; i < count; i += 8) {
        f32x4 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float* p = part(min(i + e, count - 1) + i0, stored, row);
          x[e] = *reinterpret_cast<const f32x4*>(p + 2 * stored + row * D + c);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float fe = i + e < count ? __shfl(f, i + e, LPR) : 0.0f, le = __shfl(l, min(i + e, count - 1), LPR);
          acc += fe * x[e];
          sum = fmaf(fe, le, sum);
        }
      }
    }
    const int lrow = t * TILE + r, tok = divide(a.div_g, lrow);
    const size_t at = ((size_t)(q0 + tok) * a.Hk + hk) * a.G + (lrow - tok * a.G);
    store_row<D>(a, at, c, acc * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (c == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (M - P_SHIFT + log2f(sum)) * PK_LN2;
  }
}

}  // namespace

}  // namespace es

using namespace es;

// Key ranges are worth a second launch where the tiles do not fill the GPU and a tile may have many chunks. `equal`: the keys
// divide into B equal sequences; otherwise the host knows their sum alone, and the longest may have anything from Tk / B of
// them to all. It is taken to have Tk / sqrt(B) then, halfway in the logarithm: with all of them batches of short sequences
// went to ranges that cut nothing (us whole and in ranges, D = 128, causal: 8 x 512 tokens of 4 heads 13 and 23, 100 x 64 of
// one head 7.5 and 16, 4 x 1024 of 4 heads 18 and 31; 32 tokens against 40 keys each 8 and 10-12), with Tk / B a long
// sequence among short ones is not cut (8000 + 7 x 64 tokens of one head 91 and 46; tokens against 8000 + 31 x 40 keys 69 and
// 14).
// Single tokens and the like (up to 32 rows a sequence on average, whose partials are small): from 1024 keys on. (8 tokens, 8
// heads over 2, against 300 keys each 8 and 12, 1000 12.4 and 12.9; 2000 + 31 x 40 20 and 12.) From 64 sequences on the plan
// is read once a pass, so the longest one has to be longer (64 tokens against 256 keys 7 and 17, 128 against 2000 + 127 x 20
// 19 and 31).
// One sequence, or no more keys than rows (then the longest sequence has the most tiles): a launch of whole tiles takes
// WHOLE_CHUNK_US a chunk of the longest one, ranges RANGE_CHUNK_US a chunk and item and RANGE_US more for their plan,
// partials and merge. (us in ranges and whole, D = 128, causal: 200 tokens of 32 heads over 8 against 1000 keys 24 and 19,
// 2000 keys 26 and 31, 4000 keys 34 and 54; 2000 tokens of 2 heads over one 24 and 29, of 8 heads 36 and 31; 3000 of 8 58 and
// 45; 5000 of 4 heads 61 and 67, of 8 heads over 8 117 and 77; 1500 of 10 over 2 35 and 25. At D = 64 all three are about 3 /
// 4 of that.)
// Otherwise some sequences may have most of the keys and few of the tiles: from 4096 keys in all (equal sequences: each), or
// where the tiles take a quarter of the GPU's places or fewer from 1280 of the longest. (us whole and in ranges, 64 tokens
// each of 8 heads: against 4000 + 3 x 100 keys 49 and 20, 2500 + 2 x 80 34 and 23, 4 x 2000 29 and 22, 4 x 1000 17 and 21, 4
// x 500 12 and 19, 16 x 300 11 and 17, 4000 + 15 x 100 51 and 21.)
constexpr double WHOLE_CHUNK_US = 0.77, RANGE_CHUNK_US = 0.003125, RANGE_US = 15.0;
static bool ranged(long long tiles, int B, int Tq, int Tk, int H, int Hk, int D, bool equal) {
  const long long items = tiles * Hk;
  const double chunks = (double)(Tk / BK), longest = equal ? chunks / B : chunks / std::sqrt((double)B);
  if (items >= 2 * resident(D)) return false;
  if ((long long)Tq * (H / Hk) <= 32LL * B) return longest >= (B < 64 ? 16.0 : 0.625 * B);
  if (B == 1 || Tk <= Tq) return longest * WHOLE_CHUNK_US >= RANGE_US + longest * RANGE_CHUNK_US * (double)items;
  return 4 * items <= resident(D) ? longest >= 20.0 : (equal ? longest : chunks) >= 64.0;
}

// Tiles of 64 rows instead of 128, which take about two thirds of the time each and are twice as many, as long as the GPU holds
// them all at once (512 at D = 128, 1024 at D = 64), under a causal mask half again as many. (us with 128 and 64 rows, D = 128:
// 1462 causal tokens of 4 heads over one 32 and 23, 1700 of 16 heads 38 and 29, of 36 45 and 45, of 48 50 and 58; 1024 tokens
// without a mask of 16 heads 25 and 19, of 32 27 and 26, of 36 37 and 40. D = 64: causal, 16 heads 28 and 21, 48 heads 35 and
// 32, 60 heads 38 and 37; without a mask, 44 heads 25 and 22, 64 heads 27 and 28.)
static bool small_tiles(long long tiles, int Hk, int D, bool causal) {
  return tiles * Hk * (causal ? 2 : 3) <= (D == 64 ? 1536 : 768);
}

// Workgroups a tile of the merge: a row each thread group, as far as a sequence can have rows.
static unsigned merge_rows(long long rows, int D) { return (unsigned)((std::min<long long>(rows, TILE) * D / 4 + 255) / 256); }

// Workspace of a shared-prefix call: partials of the sequences, partials of the prefix, plan; of a packed one: partials, plan.
struct Layout {
  long long items;               // a head
  size_t prefix, plan, bytes;    // offsets
  int rows;                      // of a sequence's partial
};
static Layout packed_layout(long long tiles, int B, int Hk, int D) {
  Layout l = {range_items(tiles, Hk, D), 0, 0, 0, TILE};
  l.plan = (size_t)l.items * Hk * part_floats(TILE, D) * sizeof(float);
  l.bytes = l.plan + (size_t)(B + 1) * sizeof(int2);
  return l;
}
static Layout shared_layout(int B, int n, int H, int Hk, int D) {
  const long long list = (long long)n * (H / Hk), tiles = (B * list + TILE - 1) / TILE, own = B * ((list + TILE - 1) / TILE);
  Layout l = {range_items(tiles + own, Hk, D), 0, 0, 0, (int)std::min<long long>((list + 31) / 32 * 32, TILE)};
  l.prefix = (size_t)l.items * Hk * part_floats(l.rows, D) * sizeof(float);
  l.plan = l.prefix + (size_t)range_items(tiles, Hk, D) * Hk * part_floats(TILE, D) * sizeof(float);
  l.bytes = l.plan + (size_t)(B + 1) * sizeof(int2);
  return l;
}

#ifndef ES_ELEM_F16
extern "C" size_t es_packed_fwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D) {
  if (B <= 0 || Tq <= 0 || Tk < 0 || H <= 0 || Hk <= 0 || H % Hk) return 0;
  const long long tiles = tile_numbers<TILE>(B, Tq, H / Hk);
  // (for either kind of running lengths: NULL or given)
  return ranged(tiles, B, Tq, Tk, H, Hk, D, false) || ranged(tiles, B, Tq, Tk, H, Hk, D, true)
             ? packed_layout(tiles, B, Hk, D).bytes : 0;
}
extern "C" size_t es_shared_prefix_workspace(int B, int n, int P, int S, int H, int Hk, int D) {
  if (B <= 0 || n <= 0 || P < 0 || S < 0 || H <= 0 || Hk <= 0 || H % Hk) return 0;
  return shared_layout(B, n, H, Hk, D).bytes;
}
#endif

extern "C" int ES_VSA_API(es_packed_fwd)(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k,
                                         const float* bias, const int* buckets, int num_buckets, int R, void* out,
                                         float* lse, void* workspace, size_t workspace_bytes, int B, int Tq, int Tk, int H,
                                         int Hk, int D, int causal, float scale, hipStream_t stream) {
  if (int st = packed_check(q, k, v, cu_q, cu_k, bias, buckets, num_buckets, R, B, Tq, Tk, H, Hk, D, scale)) return st;
  if (Tq == 0) return ES_OK;
  ES_REQUIRE(out && lse, ES_ERR_INVALID, "packed: null out / lse");
  ES_REQUIRE(aligned16({q, k, v, out, workspace}), ES_ERR_INVALID, "packed: tensors must be aligned to 16 bytes");
  FwdArgs a = {};
  a.q = (const e16_t*)q;
  a.k = (const e16_t*)k;
  a.v = (const e16_t*)v;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.bias = bias;
  a.buckets = buckets;
  a.num_buckets = num_buckets;
  a.R = bias ? R : 0;
  a.out = (e16_t*)out;
  a.lse = lse;
  a.B = B;
  a.Tq = Tq;
  a.Tk = Tk;
  a.H = H;
  a.Hk = Hk;
  a.G = H / Hk;
  a.div_g = fast_div(a.G);
  a.causal = causal != 0;
  a.scale = scale * LOG2E;
  a.tiles = (int)tile_numbers<TILE>(B, Tq, a.G);
  ES_REQUIRE((long long)a.tiles * Hk < MAX_GRID, ES_ERR_UNSUPPORTED, "packed: too many sequences");
  if (ranged(a.tiles, B, Tq, Tk, H, Hk, D, cu_k == nullptr)) {
    ES_REQUIRE(workspace && workspace_bytes >= es_packed_fwd_workspace(B, Tq, Tk, H, Hk, D), ES_ERR_INVALID,
               "packed: workspace too small");
    a.part = (float*)workspace;
    const Layout l = packed_layout(a.tiles, B, Hk, D);
    a.plan = (int2*)((char*)workspace + l.plan);
    a.inv_slots = (float)Hk / (float)resident(D);
    a.items = (int)l.items;
    const dim3 grid((unsigned)(l.items * Hk)), merge((unsigned)(a.tiles * Hk), merge_rows((long long)Tq * a.G, D));
    if (D == 64) {
      if (bias) hipLaunchKernelGGL((packed_ranges_kernel<64, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_ranges_kernel<64, false>), grid, dim3(256), 0, stream, a);
      hipLaunchKernelGGL((merge_kernel<64, false>), merge, dim3(256), 0, stream, a);
    } else {
      if (bias) hipLaunchKernelGGL((packed_ranges_kernel<128, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_ranges_kernel<128, false>), grid, dim3(256), 0, stream, a);
      hipLaunchKernelGGL((merge_kernel<128, false>), merge, dim3(256), 0, stream, a);
    }
    return check_launch("es_packed_fwd");
  }
  const bool small = small_tiles(a.tiles, Hk, D, causal != 0);
  if (small) a.tiles = (int)tile_numbers<TILE / 2>(B, Tq, a.G);
  const dim3 grid((unsigned)(a.tiles * Hk));
  auto launch = [&](auto dim, auto with_bias) {
    constexpr int d = decltype(dim)::value;
    constexpr bool b = decltype(with_bias)::value;
    if (small) hipLaunchKernelGGL((packed_fwd_kernel<d, b, TILE / 2>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((packed_fwd_kernel<d, b, TILE>), grid, dim3(256), 0, stream, a);
  };
  using std::integral_constant;
  if (D == 64) {
    if (bias) launch(integral_constant<int, 64>{}, std::true_type{});
    else launch(integral_constant<int, 64>{}, std::false_type{});
  } else {
    if (bias) launch(integral_constant<int, 128>{}, std::true_type{});
    else launch(integral_constant<int, 128>{}, std::false_type{});
  }
  return check_launch("es_packed_fwd");
}

extern "C" int ES_VSA_API(es_shared_prefix_fwd)(const void* q, const void* k_prefix, const void* v_prefix, const void* k,
                                                const void* v, const int* lens, void* out, float* lse, void* workspace,
                                                size_t workspace_bytes, int B, int n, int P, int S, int H, int Hk, int D,
                                                float scale, hipStream_t stream) {
  ES_REQUIRE(B > 0 && n > 0 && P >= 0 && S >= 0, ES_ERR_INVALID, "shared prefix: B and n must be positive, P and S not negative");
  ES_REQUIRE((long long)B * n < (1LL << 30) && S < (1 << 30), ES_ERR_UNSUPPORTED, "shared prefix: too many rows");
  ES_REQUIRE(lens && out && lse && workspace && (S == 0 || (k && v)), ES_ERR_INVALID, "shared prefix: null tensor pointer");
  if (int st = packed_check(q, k_prefix, v_prefix, nullptr, lens, nullptr, nullptr, 0, 0, B, B * n, P, H, Hk, D, scale))
    return st;
  ES_REQUIRE(aligned16({q, k_prefix, v_prefix, k, v, out, workspace}), ES_ERR_INVALID,
             "shared prefix: tensors must be aligned to 16 bytes");
  ES_REQUIRE(workspace_bytes >= es_shared_prefix_workspace(B, n, P, S, H, Hk, D), ES_ERR_INVALID,
             "shared prefix: workspace too small");
  FwdArgs a = {};
  a.q = (const e16_t*)q;
  a.kp = (const e16_t*)k_prefix;
  a.vp = (const e16_t*)v_prefix;
  a.k = (const e16_t*)k;
  a.v = (const e16_t*)v;
  a.lens = lens;
  a.out = (e16_t*)out;
  a.lse = lse;
  a.part = (float*)workspace;
  a.B = B;
  a.n = n;
  a.P = P;
  a.S = S;
  a.H = H;
  a.Hk = Hk;
  a.G = H / Hk;
  a.div_g = fast_div(a.G);
  a.scale = scale * LOG2E;
  const Layout l = shared_layout(B, n, H, Hk, D);
  const long long own = (long long)B * (((long long)n * a.G + TILE - 1) / TILE);
  ES_REQUIRE(l.items * Hk < MAX_GRID, ES_ERR_UNSUPPORTED, "shared prefix: too many sequences");
  a.part_prefix = (float*)((char*)workspace + l.prefix);
  a.plan = (int2*)((char*)workspace + l.plan);
  a.part_rows = l.rows;
  a.inv_slots = (float)Hk / (float)resident(D);
  a.items = (int)l.items;
  const dim3 grid((unsigned)(l.items * Hk)), merge((unsigned)(own * Hk), merge_rows((long long)n * a.G, D));
  if (D == 64) {
    hipLaunchKernelGGL((shared_prefix_kernel<64>), grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL((merge_kernel<64, true>), merge, dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((shared_prefix_kernel<128>), grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL((merge_kernel<128, true>), merge, dim3(256), 0, stream, a);
  }
  return check_launch("es_shared_prefix_fwd");
}
