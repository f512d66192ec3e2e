// Tiles of the forward attention kernels over packed sequences, shared prefixes (packed_fwd.hip) and paged caches (paged_fwd.hip):
// the rows of a tile, their online softmax, the cut of tiles into key ranges and the merge of those (gfx950, MFMA 32x32x16).
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
#pragma once
#include "packed.h"

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

// Paged caches: lens (in FwdArgs) keys of each sequence, held to `cap`, in the pages that its row of `table` names.
struct PagedArgs {
  const int* table;
  const e16_t *k, *v;                                // 16 bits, with the strides of a page, a head and a row in values
  const uint8_t *codes[2], *scales[2];               // 4 bits: keys, values
  long long page_stride, head_stride, row_stride;
  int max_pages, num_pages, shift, cap;              // a page has 1 << shift rows
};

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
  PagedArgs paged;
  // paged caches (paged_fwd.hip): shares of a head, the least cost of one, units of cost a chunk; partials of a head
  int shares, least_share, parts;
  float cost_unit;
};

// What one workgroup computes: the tile from row r0 on of the list of nq * G rows that starts at token q0, against key rows
// 0 .. nk - 1 behind k / v (this kv head's first row), chunks c0 .. c1 - 1 of them.
struct Job {
  const e16_t *k, *v;
  int q0, nq, nk, hk, r0, c0, c1, causal;
  int over = 0;      // paged: tokens of the sequence past its last page, whose keys nothing holds
  const int* table;  // paged: the sequence's page numbers
  float* part;  // a partial of `part_rows` rows; nullptr: finished rows go to out / lse
  int part_rows;
};

// floats of a partial of `rows` rows: m, l, O [D] of each
__host__ __device__ constexpr int part_floats(int rows, int D) { return rows * (D + 2); }

// keys that row r of the job's list sees
__device__ __forceinline__ int keys_seen(const FwdArgs& a, const Job& j, int r) {
  return j.causal ? min(max(divide(a.div_g, r) + 1 - j.nq + j.nk + j.over, 0), j.nk) : j.nk;
}
// chunks that any of the M rows of the job's tile sees
template <int M>
__device__ __forceinline__ int tile_chunks(const FwdArgs& a, const Job& j) {
  const int last = min(j.nq * a.G, j.r0 + M) - 1;
  return (keys_seen(a, j, last) + BK - 1) / BK;
}

// eight values less their held ones, held
__device__ __forceinline__ ev8 rest8(const float* p, const ev8& held) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[i] - (float)held[i];
  return epack8(x);
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

  // p = exp(s - maximum) as two B operands; ra, rb: what their rounding leaves, as two more
  __device__ __forceinline__ void exponentials(const f32x16& s, float sc, float c, ev8& pa, ev8& pb, ev8* ra = nullptr,
                                               ev8* rb = nullptr) {
    c -= (mrun == -INFINITY ? 0.0f : mrun) - P_SHIFT;
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = exp2f_fast(fmaf(s[r], sc, c));
    pa = epack8(&p[0]);
    pb = epack8(&p[8]);
    if (ra != nullptr) {
      *ra = rest8(&p[0], pa);
      *rb = rest8(&p[8], pb);
    }
    // (the sum takes the probabilities before their rounding: the LSE is a float32 result of its own)
    float sum[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
    for (int r = 4; r < 16; ++r) sum[r & 3] += p[r];
    lsum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }

  // O^T += V^T P^T of sixteen keys at `v`; rest: of what the rounding of P left, too
  __device__ __forceinline__ void values(const char* v, int t0, int t1, const ev8& p, const ev8* rest = nullptr) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const ev8 x = ecat_tr(lds_read_tr(v, t0 ^ (64 * db)), lds_read_tr(v, t1 ^ (64 * db)));
      o[db] = emfma(x, p, o[db]);
      if (rest != nullptr) o[db] = emfma(x, *rest, o[db]);
    }
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

// Where a tile's keys come from. `Rowwise`: rows in order behind j.k / j.v. (paged_fwd.hip has the others.)
//   wide(a, j, c, dst)       starts the transfers of this wave's quarter of chunk c to LDS address dst (K, then V)
//   settle(base)             what the transfers leave to do once they have landed (STAGED: nothing)
//   run(a, j, v, u, dst)     narrow tiles: starts those of K (v: V) of the 32-key run u, all of them by this wave
//   enter / mask             HOLES: keys that a sequence counts may be missing, 16 at a time; their scores become -inf
//   FINE                     narrow tiles multiply V by what the rounding of P leaves, too (wide ones, which the matrix units
//                            bound, round P once: an error about as large as that of the output's own rounding)
template <int D>
struct Rowwise {
  static constexpr bool HOLES = false, STAGED = false, FINE = false;
  static constexpr int LPR = D / 8, NI = D / 32;
  int l, wv;
  unsigned src[2 * NI], stride;
  __device__ __forceinline__ Rowwise(const FwdArgs& a, const Job&, int lane, int wave, bool narrow) : l(lane), wv(wave) {
    stride = (unsigned)a.Hk * D * 2;
    // a lane's transfers: 1 KB runs of 64 / LPR rows each
#pragma unroll
    for (int i = 0; i < 2 * NI; ++i) {
      const int R = ((narrow ? 0 : wv * NI) + i) * (64 / LPR) + l / LPR;
      src[i] = (unsigned)R * stride + (unsigned)(((l % LPR) ^ swizzle<D>(R)) * 16);
    }
  }
  __device__ __forceinline__ void wide(const FwdArgs& a, const Job& j, int c, unsigned dst) {
    const size_t row = (size_t)c * BK * a.Hk * D;
    const unsigned bytes = (unsigned)(min(BK, j.nk - c * BK) - 1) * stride + D * 2;
    const srd_t rk = make_srd(j.k + row, bytes), rv = make_srd(j.v + row, bytes);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rk, dst + i * 1024, src[i], 0u);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16_at(rv, dst + BK * D * 2 + i * 1024, src[i], 0u);
  }
  __device__ __forceinline__ void settle(char*) {}
  __device__ __forceinline__ void run(const FwdArgs& a, const Job& j, bool v, int u, unsigned dst) {
    const e16_t* base = v ? j.v : j.k;
    const srd_t rs =
        make_srd(base + (size_t)u * 32 * a.Hk * D, (unsigned)(min(32, j.nk - u * 32) - 1) * stride + D * 2);
#pragma unroll
    for (int i = 0; i < 2 * NI; ++i) dma16_at(rs, dst + i * 1024, src[i], 0u);
  }
  __device__ __forceinline__ void enter() {}
  __device__ __forceinline__ void enter_run(int) {}
  __device__ __forceinline__ void mask(f32x16&, int) const {}
};

// M = 128: 32 rows a wave; M = 64: two row groups x two key halves, whose softmax states are merged at the end
template <int D, bool BIAS, int M, class KEYS>
__device__ __forceinline__ void wide_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, TILE_BYTES = BK * ROW;
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

  KEYS keys(a, j, l, wv, false);
  const unsigned lds0 = uni(lds_addr(lds) + (unsigned)wv * (TILE_BYTES / 4));
  auto issue = [&](int c, int sb) { keys.wide(a, j, c, lds0 + (unsigned)sb * (2u * TILE_BYTES)); };
  if (j.c0 < j.c1) issue(j.c0, 0);
  if (BIAS) fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, j.hk);
  if (KEYS::STAGED && j.c0 < j.c1) keys.settle(lds);
  dma_wait();
  __syncthreads();
  for (int c = j.c0; c < j.c1; ++c) {
    const int sb = (c - j.c0) & 1;
    keys.enter();
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
        keys.mask(s0, kh);
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
      keys.mask(s0, 0);
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
      keys.mask(s1, 1);
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
    if (KEYS::STAGED && c + 1 < j.c1) keys.settle(lds + (sb ^ 1) * 2 * TILE_BYTES);
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
template <int D, bool BIAS, class KEYS>
__device__ __forceinline__ void narrow_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, RUN = 32 * ROW, NI = D / 16;
  const int tid = threadIdx.x, l = tid & 63, hi = l >> 5, lq = l & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = j.r0, rows = j.nq * a.G;
  Rows<D, BIAS> x;
  x.load(a, j, r0 + lq, hi);
  const Offsets<D> off(l);
  const int last = min(r0 + 31, rows - 1);
  const int seen_min = keys_seen(a, j, r0), seen_max = keys_seen(a, j, last);
  const int low = divide(a.div_g, r0) + j.nk - j.nq, high = divide(a.div_g, last) + j.nk - j.nq;

  KEYS keys(a, j, l, wv, true);
  char* kb = lds + wv * 2 * RUN;
  char* vb = kb + RUN;
  const unsigned kd = uni(lds_addr(kb)), vd = uni(lds_addr(vb));
  const int end = min(2 * j.c1, (seen_max + 31) / 32);
  int u = 2 * j.c0 + wv;
  if (u < end) {
    keys.run(a, j, false, u, kd);
    keys.run(a, j, true, u, vd);
  }
  if (BIAS) {
    fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, j.hk);
    __syncthreads();
  }
  for (; u < end; u += 4) {
    const bool more = u + 4 < end;
    keys.enter_run(u);
    wait_transfers<NI>();  // K: all but the V run's transfers
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) s = emfma(elds16(kb, off.k0 ^ (32 * ks)), x.q[ks], s);
    wait_lds();
    if (more) keys.run(a, j, false, u + 4, kd);
    ev8 pa, pb, ra, rb;
    float sc, c, alpha;
    keys.mask(s, 0);
    x.raise(x.scores(a, tab, s, 32 * u, hi, 32 * (u + 1) > seen_min, low, high, sc, c), alpha);
    x.exponentials(s, sc, c, pa, pb, KEYS::FINE ? &ra : nullptr, KEYS::FINE ? &rb : nullptr);
    if (more) wait_transfers<NI>();
    else wait_transfers<0>();
    x.values(vb, off.t0, off.t1, pa, KEYS::FINE ? &ra : nullptr);
    x.values(vb + RUN / 2, off.t0, off.t1, pb, KEYS::FINE ? &rb : nullptr);
    wait_lds();
    if (more) keys.run(a, j, true, u + 4, vd);
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

template <int D, bool BIAS, int M, class KEYS = Rowwise<D>>
__device__ __forceinline__ void run_tile(const FwdArgs& a, const Job& j, char* lds, float* stats, float* tab) {
  if (j.nq * a.G - j.r0 <= 32) narrow_tile<D, BIAS, KEYS>(a, j, lds, stats, tab);
  else wide_tile<D, BIAS, M, KEYS>(a, j, lds, stats, tab);
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
