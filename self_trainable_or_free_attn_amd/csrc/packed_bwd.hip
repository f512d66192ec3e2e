// Backward of attention over packed sequences (gfx950, MFMA 32x32x16, bf16 / fp16).
//
// With P = exp(S - lse) and dS = P (dP - delta), dP = dO V^T, delta = rowsum(dO O) (rows that see no key: P = 0):
//   bwd_q       one workgroup per (64 rows, kv head): dQ = scale dS K over the keys, 2 row groups x 2 key halves, S^T and
//               dP^T with rows on lanes; with a bias it also sums dS by clamped distance. It leaves lse in log2 units (+inf
//               for rows without keys) and delta for bwd_kv, laid out by kv head and row of the list (token, head in group),
//               so that a row tile's values are contiguous, the fp16 factor of P and its inverse in them.
//   bwd_kv      one workgroup per (64 keys, kv head): dV = P^T dO and dK = scale dS^T Q over all rows of the list that see
//               the keys, which sums over the heads of a group without atomics. Four waves = 2 key halves x 2 row halves
//               of each staged 64-row tile; S and dP come out with keys on lanes, so that P and dS are B operands.
//               With few (key tile, kv head) pairs the rows of each are cut into ranges, one workgroup each, whose float32
//               sums kv_sums adds in order.
//   bias_sums   those sums over the row tiles and into buckets
// Every sum has a fixed order, so the same inputs give the same bits. The scores are computed twice (7 products for 5): a
// single pass would need dQ in float32 atomics or a dQ partial a key tile.
// delta: O carries the roundings of its probabilities and its own, so rowsum(dO O) is off by up to 2^-8 (bf16) of |dO| |O|,
// the same for all keys of a row. Over n keys of about equal weight that shifts a row's dQ by 1 / sqrt(n) of what the
// rounding of dS does, but with few keys it adds to it, and sums of unrounded dS (the bias gradient) have no other error.
// So bwd_q takes delta = sum P dP / sum P over the keys in a pass of its own before the main one where a tile sees up to
// EXACT_CHUNKS * 64 keys, and always with a bias, and stores it for bwd_kv, which runs after it. (Relative errors against 64
// bits, causal sequences of 1 to 1200 tokens, bf16: dQ 2.55e-3 -> 2.36e-3, dK 2.52e-3 -> 2.34e-3, which is that of the
// rounding of dS and the result, the bias gradient 1.3e-3 -> 2e-7; fp16: 3.3e-4 -> 2.9e-4, 3.4e-4 -> 8e-7.)
// Bounds: the matrix units on long sequences. Clips of 13770, 11880 and 4096 tokens without a mask, 12 heads, D = 128: bwd_q
// 2.87 ms, 1120 TFLOP/s of its three products (61 % of the cycles issue a matrix instruction, LDS 31 %), bwd_kv 4.13 ms, 1030
// TFLOP/s of its four (51 %; it waits the most, for its transfers and at the tile's barrier, with two workgroups a CU at 255
// registers), in fp16 3.20 and 4.62 ms; causal prompts of 1 to 6553 tokens, 24 heads over 8: 0.65 and 0.88 ms. At D = 64 as
// many exponentials go with half the products: the clips take 1.50 and 2.21 ms, 64 and 51 % matrix issue beside 74 and 62 %
// vector work. What bounds short sequences is the chain of a tile's few chunks: transfers, two products, exponentials, two
// products.
// dS is rounded to the token type without the softmax scale (applied to the finished sums). In fp16 it is rounded times a power
// of two of its row (dQ) or key (dK), see fit.
#include "packed.h"

#include <algorithm>
#include <cmath>

namespace es {

namespace {

// fp16: the probabilities of dV = P^T dO are taken 2^14 higher, out of the type's subnormal range for all down to 2^-28; dS
// and the finished sum take the factor back exactly. dS follows dO and V, which may be of any size (scaled losses), so it is
// taken times 2^DS_LOG2 at first and `fit` keeps it in range.
#ifdef ES_ELEM_F16
constexpr bool DS_SCALED = true;
constexpr float P_SHIFT = 14.0f, P_BACK = 1.0f / 16384.0f;
constexpr int DS_LOG2 = 40;
#else
constexpr bool DS_SCALED = false;
constexpr float P_SHIFT = 0.0f, P_BACK = 1.0f;
constexpr int DS_LOG2 = 0;
#endif
constexpr int EXACT_CHUNKS = 8;

// A lane's dS as fp16 operands: values times 2^e, e of its row or key and the same in both half waves. Where one passes 2^15, e
// falls so that the largest comes to 2^7 .. 2^8, and the sums so far fall with it (exact in float32). So no operand overflows
// whose sum float32 holds, and the type's subnormal steps (2^-24, half of one a rounding) put a dS off by no more than 2^-32 of
// the lane's largest, or, where e is still 40, by 2^-65. The 2^7 between the two borders make a change rare: in the first tile,
// then only for values 128 times as large. P 2^40 |dP - delta| stays below 2^80. An infinite dS (from an infinite dO) stays one.
// (Whole backward in fp16 without and with it, us: 13770 tokens of 12 heads 4320 and 4610, 8192 causal of 24 over 8 1490 and
// 1560, of 16 heads at D = 64 1019 and 1089, 500 of 24 heads with a bias at D = 64 41.8 and 43.1.)
template <int N>
__device__ __forceinline__ bool fit(float (&ds)[16], f32x16 (&acc)[N], int& change) {
  float mx = fabsf(ds[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
  mx = max_xor32(mx);
  if (!(mx > 32768.0f)) return false;
  change = 8 - __builtin_amdgcn_frexp_expf(mx);
  const float f = __builtin_ldexpf(1.0f, change);
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
  for (int db = 0; db < N; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= f;
  return true;
}

struct BwdArgs {
  const e16_t *q, *k, *v, *dout, *out;
  const float *lse, *bias;
  const int *cu_q, *cu_k, *buckets;
  e16_t *dq, *dk, *dv;
  float *dbias;
  float *lse2, *delta;  // [Hk][Tq * G]
  float* dist;          // [row tile numbers][Hk][G * (2 R + 1)]: dS by clamped distance
  FastDiv div_g;
  float inv_g;  // 1 / G
  int B, Tq, Tk, H, Hk, G, R, num_buckets, causal;
  int q_tiles, k_tiles;  // tile numbers of a head
  int ranges;            // row ranges of bwd_kv
  float* part;           // their sums [range][Tk][Hk][dV | dK][D]
  float scale_log2, scale;
};

// *p += x without waiting for it (ds_add_f32); lanes of one instruction must not share an address where order matters
__device__ __forceinline__ void lds_add(float* p, float x) {
  __builtin_amdgcn_ds_faddf((__attribute__((address_space(3))) float*)p, x, 0, 0, false);
}

// Tiles of 64 keys x 64 rows: a wave's 32 x 32 of S and dP, its key's K and V rows and two sums of D x 32 just fit the
// registers of two waves a SIMD (three at D = 64; four would spill: 8192 tokens of 16 heads, whole backward 1081 -> 1367 us).
// (dP's products under the exponentials, as bwd_q has them, spill: 4428 -> 4500 us at 13770 tokens, 12 heads. Staging dO later
// than Q computes the row addresses twice: whole backward 4.31 -> 4.43 ms.) With the products of both kernels at a raised
// priority (packed.h) the whole backward of 13770 tokens of 12 heads takes 4.26 ms, not 4.40, of 8192 causal tokens of 24 heads
// over 8 1611 us, not 1661, at D = 64 1063, not 1076. Not in bwd_q with a bias, whose vector work is the longer part (2303 tokens
// of 24 heads, D = 64, whole backward 82.5 us without, 85.5 with).
template <int D, bool BIAS>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_bwd_kv_kernel(BwdArgs a) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, TILE_BYTES = BK * ROW, NI = D / 32, LPR = D / 8;
  __shared__ __attribute__((aligned(16))) char qd_s[2][2][TILE_BYTES];  // [buffer][Q | dO]
  __shared__ __attribute__((aligned(16))) float st_s[2][2][BK];         // [buffer][lse2 | delta]
  // [buffer][position of the row | its part of the bias table]
  __shared__ __attribute__((aligned(16))) int pos_s[BIAS ? 2 : 1][2][BIAS ? BK : 1];
  __shared__ float tab[BIAS ? BIAS_TABLE : 1];
  const int item = blockIdx.x / a.ranges, range = blockIdx.x - item * a.ranges, w = item / a.Hk, hk = item - w * a.Hk;
  int b, kb;
  Seq s;  // (key rows behind the last sequence: no rows, so zero gradients)
  if (!tile_of<BK, true>(a.cu_q, a.cu_k, a.B, a.Tq, a.Tk, a.G, w, s, b, kb)) return;
  const int rows = s.nq * a.G, shift = s.nk - s.nq;
  const int row_tiles = (rows + BK - 1) / BK;
  // causal: the first row that sees this tile's first key
  const int first_tile = a.causal ? min(max(kb * BK - shift, 0) * a.G / BK, row_tiles) : 0;
  const int beg = first_tile + (int)((long long)(row_tiles - first_tile) * range / a.ranges);
  const int end = first_tile + (int)((long long)(row_tiles - first_tile) * (range + 1) / a.ranges);
  const int tid = threadIdx.x, l = tid & 63, hi = l >> 5, lq = l & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qh = wv >> 1, kh = wv & 1;
  const int key = kb * BK + 32 * kh + lq;
  const bool kvalid = key < s.nk;
  const size_t krow = ((size_t)(s.k0 + (kvalid ? key : 0)) * a.Hk + hk) * D;
  ev8 kreg[NKS], vreg[NKS];  // this lane's key row
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const ev8 z = {};
    kreg[ks] = kvalid ? *reinterpret_cast<const ev8*>(a.k + krow + 8 * hi + 16 * ks) : z;
    vreg[ks] = kvalid ? *reinterpret_cast<const ev8*>(a.v + krow + 8 * hi + 16 * ks) : z;
  }
  // Row tile i: Q and dO rows (16 of each a wave) through a resource based at the tile's first token, and, wave 0, its lse2
  // and delta. Rows of a list are `row / G` tokens of H * D values and `row % G` heads apart.
  const size_t list = (size_t)hk * a.Tq * a.G + (size_t)s.q0 * a.G;
  const unsigned lds_q = uni(lds_addr(&qd_s[0][0][0]) + (unsigned)wv * (NI * 1024u));
  // A lane's transfer r moves 16 bytes of tile row R + RPT r, R = 16 wv + l / LPR, whose chunk the swizzle moves by one XOR a
  // step: of its address in a list without gaps one register holds step 0 (`lane_at`). A token's rows are (H - G) rows further
  // apart than that, and the row's token within the tile is (rows since the first token's + 1/2) / G in float32 (exact: rows
  // up to G + 63, G up to 4096, the nearest border 1 / (2 G) away). Few registers matter here: with more the compiler spills
  // some, and a reload in this loop waits for every transfer before it (a tile's transfers took 2970 cycles instead of 920).
  constexpr int RPT = 64 / LPR, XOR = D == 128 ? 16 : 32;
  auto token_in_tile = [&](int row) { return token_of((float)row + 0.5f, a.inv_g); };  // of rows since the first token's
  int lane_at = (wv * 16 + l / LPR) * ROW + (((l % LPR) ^ swizzle<D>(l / LPR)) << 4);
  auto issue = [&](int i, int sb) {
    const int t0 = divide(a.div_g, i * BK), toks = min(s.nq - t0, BK + 1), rel = i * BK - t0 * a.G;
    const size_t base = ((size_t)(s.q0 + t0) * a.H + hk * a.G) * D;
    const unsigned bytes = (unsigned)((toks - 1) * a.H + a.G) * ROW;
    const srd_t rq = make_srd(a.q + base, bytes), rd = make_srd(a.dout + base, bytes);
    const unsigned gap = (unsigned)(a.H - a.G) * ROW;
    const float first = (float)rel + 0.5f;
    const unsigned qd = lds_q + (unsigned)sb * (2u * TILE_BYTES);
#pragma unroll
    for (int r = 0; r < NI; ++r) {
      const unsigned tok = (unsigned)token_of((float)(lane_at / ROW) + (first + (float)(RPT * r)), a.inv_g);
      const unsigned at = __umul24(tok, gap) + (unsigned)((lane_at ^ (XOR * r)) + (RPT * r + rel) * ROW);
      dma16_at(rq, qd + r * 1024, at, 0u);
      dma16_at(rd, qd + TILE_BYTES + r * 1024, at, 0u);
    }
    // (rows past the list's end read as zeros: their P is finite and meets zeros of dO, dP and delta, and `masked` covers
    // the case of a bias that makes it infinite)
    if (wv < 2)
      dma4(make_srd((wv == 0 ? a.lse2 : a.delta) + list + (size_t)i * BK, (unsigned)min(rows - i * BK, BK) * 4u),
           st_s[sb][wv], 4u * l, 0u);
    if (BIAS && a.G > 1 && wv == 2) {
      const int tok = token_in_tile(rel + l);
      pos_s[sb][0][l] = t0 + tok + shift;
      pos_s[sb][1][l] = bias_row(a.G, a.R, rel + l - tok * a.G);
    }
  };
  // LDS offsets of this wave's row half (packed_fwd.hip: Offsets)
  int aoff = qh * (TILE_BYTES / 2) + tile_at<D>(lq, hi);
  int toff0, toff1;
  {
    const int g1 = (l >> 4) & 1, sub = (l & 1) * 8, rowA = 4 * hi + ((l & 15) >> 2);
    toff0 = qh * (TILE_BYTES / 2) + tile_at<D>(rowA, 2 * g1 + ((l & 3) >> 1)) + sub;
    toff1 = qh * (TILE_BYTES / 2) + tile_at<D>(rowA + 8, 2 * g1 + ((l & 3) >> 1)) + sub;
  }
  f32x16 acc_v[NDB], acc_k[NDB];  // this lane's key: dV and dK over this row half
#pragma unroll
  for (int db = 0; db < NDB; ++db) acc_v[db] = acc_k[db] = f32x16{};

  if (beg < end) issue(beg, 0);
  if (BIAS) fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, hk);
  dma_wait();
  __syncthreads();
  float ds_mul = ldexpf(P_BACK, DS_LOG2);  // acc_k sums dS Q times ds_mul / P_BACK
  // (lanes past the last key: whatever they sum up belongs to their own column and is not stored)
  for (int i = beg; i < end; ++i) {
    const int sb = (i - beg) & 1;
    // the rows of Q are read before the next tile's transfers are issued: S then finds its operands ready
    ev8 qf[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[ks] = elds16(qd_s[sb][0], aoff ^ (32 * ks));
    if (i + 1 < end) issue(i + 1, sb ^ 1);
    asm volatile("" : "+v"(aoff), "+v"(toff0), "+v"(toff1), "+v"(lane_at));  // (keeps the offsets from being hoisted)
    const char* qt = qd_s[sb][0];
    const char* dt = qd_s[sb][1];
    auto product = [&](const char* xt, const ev8& xa, const ev8& xb, f32x16 (&acc)[NDB]) {  // acc += xt^T [xa | xb]
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int t0 = toff0 ^ (64 * db), t1 = toff1 ^ (64 * db);
        acc[db] = emfma(ecat_tr(lds_read_tr(xt, t0), lds_read_tr(xt, t1)), xa, acc[db]);
        acc[db] = emfma(ecat_tr(lds_read_tr(xt + TILE_BYTES / 4, t0), lds_read_tr(xt + TILE_BYTES / 4, t1)), xb, acc[db]);
      }
    };
    f32x16 p = {}, dp = {};
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) p = emfma(qf[ks], kreg[ks], p);
    __builtin_amdgcn_s_setprio(0);
    // the wave's rows, whose positions ascend: a key is seen from its own position on
    const int t0 = divide(a.div_g, i * BK), rel = i * BK - t0 * a.G;
    const bool masked = (a.causal && t0 + token_in_tile(rel + 32 * qh) + shift < kb * BK + 32 * kh + 31) ||
                        (BIAS && (i + 1) * BK > rows);
    // one head a group: rows stand at consecutive positions, so a lane's 16 entries of the bias table are a fixed pattern
    const int key0 = kb * BK + 32 * kh, pos0 = i * BK + 32 * qh + shift;
    const float* one = nullptr;
    float far = 0.0f;
    if (BIAS && a.G == 1) {
      if (key0 - pos0 - 31 >= a.R) far = tab[bias_row(1, a.R, 0) + a.R];
      else if (key0 + 31 - pos0 <= -a.R) far = tab[bias_row(1, a.R, 0) - a.R];
      else one = tab + bias_row(1, a.R, 0) + key - pos0 - 4 * hi;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r0 = 32 * qh + 8 * g + 4 * hi;
      f32x4 l4 = *reinterpret_cast<const f32x4*>(&st_s[sb][0][r0]);
      if (BIAS && a.G == 1) {
        if (one != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e) l4[e] -= one[-(8 * g + e)];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) l4[e] -= far;
        }
      } else if (BIAS) {
        const int4 p4 = *reinterpret_cast<const int4*>(&pos_s[sb][0][r0]), b4 = *reinterpret_cast<const int4*>(&pos_s[sb][1][r0]);
        const int ps[4] = {p4.x, p4.y, p4.z, p4.w}, gs[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) l4[e] -= tab[gs[e] + min(max(key - ps[e], -a.R), a.R)];
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = i * BK + r0 + e, pos = t0 + token_in_tile(rel + r0 + e) + shift;
          if (row >= rows || (a.causal && key > pos)) l4[e] = INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) p[4 * g + e] = exp2f_fast(fmaf(p[4 * g + e], a.scale_log2, -l4[e]));
    }
    {
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = p[r];
      __builtin_amdgcn_s_setprio(1);
      product(dt, epack8(&x[0]), epack8(&x[8]), acc_v);
    }
    __builtin_amdgcn_sched_barrier(0);  // (dP after dV: raised above it, its operands do not fit the registers)
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) dp = emfma(elds16(dt, aoff ^ (32 * ks)), vreg[ks], dp);
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(&st_s[sb][1][32 * qh + 8 * g + 4 * hi]);
#pragma unroll
      for (int e = 0; e < 4; ++e) p[4 * g + e] = (DS_SCALED ? p[4 * g + e] * ds_mul : p[4 * g + e]) * (dp[4 * g + e] - d4[e]);
    }
    {
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = p[r];
      int change;
      if (DS_SCALED && fit(x, acc_k, change)) ds_mul = ldexpf(ds_mul, change);
      __builtin_amdgcn_s_setprio(1);
      product(qt, epack8(&x[0]), epack8(&x[8]), acc_k);
      __builtin_amdgcn_s_setprio(0);
    }
    dma_wait();
    __syncthreads();
  }

  // the second row half hands its sums over through the staging buffers: [key half][dV | dK][register][lane]
  float* xch = reinterpret_cast<float*>(&qd_s[0][0][0]) + kh * (2 * NDB * 16 * 64);
  if (DS_SCALED) {
    const float back = P_BACK / ds_mul;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc_k[db][r] *= back;
  }
  if (qh == 1) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        xch[(db * 16 + r) * 64 + l] = acc_v[db][r];
        xch[((NDB + db) * 16 + r) * 64 + l] = acc_k[db][r];
      }
  }
  __syncthreads();
  if (qh == 1 || !kvalid) return;
  auto store = [&](f32x16 (&acc)[NDB], int base, float f, e16_t* out) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (acc[db][4 * i + e] + xch[((base + db) * 16 + 4 * i + e) * 64 + l]) * f;
        if (a.ranges > 1) {
          const size_t row = (size_t)range * a.Tk * a.Hk + krow / D;
          *reinterpret_cast<f32x4*>(a.part + (2 * row + (base != 0)) * D + 32 * db + 8 * i + 4 * hi) =
              f32x4{x[0], x[1], x[2], x[3]};
          continue;
        }
        ushort4 o4;
        o4.x = f2e(x[0]); o4.y = f2e(x[1]); o4.z = f2e(x[2]); o4.w = f2e(x[3]);
        *reinterpret_cast<ushort4*>(out + krow + 32 * db + 8 * i + 4 * hi) = o4;
      }
  };
  store(acc_v, 0, P_BACK, a.dv);
  store(acc_k, NDB, a.scale, a.dk);
}

// Tiles of 64 rows x 64 keys; Q and dO stay in registers, K and V are staged. Row statistics are per lane, so P needs no
// reduction. With a bias the LDS (staging, table, four histograms) still leaves two workgroups a CU.
template <int D, bool BIAS>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_bwd_q_kernel(BwdArgs a) {
  constexpr int NKS = D / 16, NDB = D / 32, ROW = D * 2, TILE_BYTES = BK * ROW, NI = D / 32, LPR = D / 8;
  __shared__ __attribute__((aligned(16))) char kv_s[2][2][TILE_BYTES];
  __shared__ float tab[BIAS ? BIAS_TABLE : 1];
  // per wave: dS by (head in group, clamped distance); before the main pass (sum P dP, sum P) of its 32 rows
  __shared__ __attribute__((aligned(8))) float hist[4][BIAS ? BIAS_ROWS : 64];
  const int w = blockIdx.x / a.Hk, hk = blockIdx.x - w * a.Hk, width = 2 * a.R + 1;
  float* dist = BIAS ? a.dist + ((size_t)w * a.Hk + hk) * (a.G * width) : nullptr;
  int b, t;
  Seq s;
  if (!tile_of<BK, false>(a.cu_q, a.cu_k, a.B, a.Tq, a.Tk, a.G, w, s, b, t)) {
    if (BIAS)  // (a tile number without a tile: its sums are read all the same)
      for (int i = threadIdx.x; i < a.G * width; i += 256) dist[i] = 0.0f;
    return;
  }
  const int rows = s.nq * a.G, shift = s.nk - s.nq;
  t = (rows + BK - 1) / BK - 1 - t;  // (under a causal mask the last tiles see the most keys)
  const int tid = threadIdx.x, l = tid & 63, hi = l >> 5, lq = l & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wv & 1, kh = wv >> 1;
  const int r0 = t * BK + 32 * rg, row = r0 + lq;
  const bool valid = row < rows;
  const int tok = divide(a.div_g, row), g = valid ? row - tok * a.G : 0, pos = tok + shift, gb = bias_row(a.G, a.R, g);
  const size_t qrow = ((size_t)(s.q0 + (valid ? tok : 0)) * a.Hk + hk) * a.G + g, at = qrow * D;
  const size_t list = ((size_t)hk * a.Tq + s.q0) * a.G + (valid ? row : 0);
  const int seen = !valid ? 0 : a.causal ? min(max(pos + 1, 0), s.nk) : s.nk;
  // the wave's rows: the first one sees the fewest keys, the last one the most
  const int first = min(r0, rows - 1), last = min(r0 + 31, rows - 1);
  const int low = divide(a.div_g, first) + shift, high = divide(a.div_g, last) + shift;
  const int seen_min = a.causal ? min(max(low + 1, 0), s.nk) : s.nk;
  const int seen_max = r0 >= rows ? 0 : a.causal ? min(max(high + 1, 0), s.nk) : s.nk;
  const int tile_high = divide(a.div_g, min(t * BK + BK, rows) - 1) + shift;
  const int end = ((a.causal ? min(max(tile_high + 1, 0), s.nk) : s.nk) + BK - 1) / BK;

  ev8 qreg[NKS], dreg[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const ev8 z = {};
    qreg[ks] = valid ? *reinterpret_cast<const ev8*>(a.q + at + 16 * ks + 8 * hi) : z;
    dreg[ks] = valid ? *reinterpret_cast<const ev8*>(a.dout + at + 16 * ks + 8 * hi) : z;
  }
  const float lse = valid ? a.lse[qrow] : -INFINITY, ls = lse == -INFINITY ? INFINITY : lse * LOG2E;
  const bool exact = end > 0 && (BIAS || end <= EXACT_CHUNKS);
  float dl = 0.0f;
  if (!exact) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const ev8 z = {};
      const ev8 x = valid ? *reinterpret_cast<const ev8*>(a.out + at + 16 * ks + 8 * hi) : z;
#pragma unroll
      for (int e = 0; e < 8; ++e) dl = fmaf((float)x[e], (float)dreg[ks][e], dl);
    }
    dl = sum_xor32(dl);
  }
  const unsigned stride = (unsigned)a.Hk * ROW;
  unsigned src[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int R = (wv * NI + i) * (64 / LPR) + l / LPR;
    src[i] = (unsigned)R * stride + (unsigned)(((l % LPR) ^ swizzle<D>(R)) * 16);
  }
  const unsigned lds_k = uni(lds_addr(&kv_s[0][0][0]) + (unsigned)wv * (NI * 1024u));
  auto issue = [&](int c, int sb) {
    const size_t base = ((size_t)(s.k0 + c * BK) * a.Hk + hk) * D;
    const unsigned bytes = (unsigned)(min(BK, s.nk - c * BK) - 1) * stride + ROW;
    const srd_t rk = make_srd(a.k + base, bytes), rv = make_srd(a.v + base, bytes);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      dma16_at(rk, lds_k + (unsigned)sb * (2u * TILE_BYTES) + i * 1024, src[i], 0u);
      dma16_at(rv, lds_k + (unsigned)sb * (2u * TILE_BYTES) + TILE_BYTES + i * 1024, src[i], 0u);
    }
  };
  const int koff = kh * (TILE_BYTES / 2) + tile_at<D>(lq, hi);
  int toff0, toff1;
  {
    const int g1 = (l >> 4) & 1, sub = (l & 1) * 8, rowA = 4 * hi + ((l & 15) >> 2);
    toff0 = kh * (TILE_BYTES / 2) + tile_at<D>(rowA, 2 * g1 + ((l & 3) >> 1)) + sub;
    toff1 = kh * (TILE_BYTES / 2) + tile_at<D>(rowA + 8, 2 * g1 + ((l & 3) >> 1)) + sub;
  }
  f32x16 dq[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) dq[db] = f32x16{};
  float far_lo = 0.0f, far_hi = 0.0f;  // dS at distances of -R and below, of R and beyond

  // P (against the statistic ls) and dP of keys key0 .. key0 + 31 (near: by distance, neither all at -R and below nor all at R
  // and beyond)
  auto scores = [&](const ev8 (&kf)[NKS], const char* vt, int key0, float ls, f32x16& x, f32x16& dp, bool& near) {
    x = f32x16{};
    dp = f32x16{};
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) x = emfma(kf[ks], qreg[ks], x);
    const int d0 = key0 + 4 * hi - (valid ? pos : low);  // (a position of the wave's)
    float sc = a.scale_log2, cb = 0.0f;
    near = false;
    if (BIAS) {
      if (key0 - high >= a.R) cb = tab[gb + a.R];
      else if (key0 + 31 - low <= -a.R) cb = tab[gb - a.R];
      else near = true;
    }
    if (near) {
      add_bias(x, sc, tab + gb, d0, a.G, a.R);
      sc = 1.0f;
    }
    if (key0 + 32 > seen_min) {
      const int left = seen - key0 - 4 * hi;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 >= left) x[r] = -INFINITY;
    }
    // (dP's products run under the exponentials)
    if (!BIAS) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) dp = emfma(elds16(vt, koff ^ (32 * ks)), dreg[ks], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = exp2f_fast(fmaf(x[r], sc, cb - ls));
    if (!BIAS) __builtin_amdgcn_s_setprio(0);
  };
  // the chunk's rows of K, read before the next chunk's transfers are issued: S then finds its operands ready
  auto read_k = [&](const char* kt, ev8 (&kf)[NKS]) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) kf[ks] = elds16(kt, koff ^ (32 * ks));
  };
  if (end > 0) issue(0, 0);
  if (BIAS) fill_bias(tab, a.bias, a.buckets, a.num_buckets, a.R, a.G, a.H, hk);
  dma_wait();
  __syncthreads();
  int sb = 0;
  if (exact) {
    float num = 0.0f, den = 0.0f;
    for (int c = 0; c < end; ++c) {
      ev8 kf[NKS];
      read_k(kv_s[sb][0], kf);
      issue(c + 1 < end ? c + 1 : 0, sb ^ 1);  // (after the last chunk the first one again, for the main pass)
      if (c * BK + 32 * kh < seen_max) {
        f32x16 p, dp;
        bool near;
        scores(kf, kv_s[sb][1], c * BK + 32 * kh, ls, p, dp, near);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          num = fmaf(p[r], dp[r], num);
          den += p[r];
        }
      }
      sb ^= 1;
      dma_wait();
      __syncthreads();
    }
    reinterpret_cast<float2*>(hist[wv])[lq] = make_float2(sum_xor32(num), sum_xor32(den));
    __syncthreads();
    const float2 s0 = reinterpret_cast<const float2*>(hist[rg])[lq], s1 = reinterpret_cast<const float2*>(hist[rg + 2])[lq];
    if (s0.y + s1.y > 0.0f) dl = (s0.x + s1.x) / (s0.y + s1.y);
  }
  if (valid && kh == 0 && hi == 0) {
    a.lse2[list] = ls - P_SHIFT;
    a.delta[list] = dl;
  }
  if (BIAS) {
    __syncthreads();
    for (int i = tid; i < 4 * BIAS_ROWS; i += 256) (&hist[0][0])[i] = 0.0f;
    __syncthreads();
  }
  int ds_log2 = DS_LOG2;  // dS and dq are taken times 2^ds_log2
  float ds_ls = ls - (float)DS_LOG2;
  for (int c = 0; c < end; ++c) {
    ev8 kf[NKS];
    read_k(kv_s[sb][0], kf);
    if (c + 1 < end) issue(c + 1, sb ^ 1);
    const char* kt = kv_s[sb][0];
    const char* vt = kv_s[sb][1];
    const int key0 = c * BK + 32 * kh;
    if (key0 < seen_max) {
      f32x16 x, dp;
      bool near;
      scores(kf, vt, key0, ds_ls, x, dp, near);
      const int d0 = key0 + 4 * hi - pos;
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = x[r] * (dp[r] - dl);
      if (BIAS) {
        if (!near) {
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += ds[r];
          if (DS_SCALED) sum = ldexpf(sum, -ds_log2);
          if (key0 - high >= a.R) far_hi += sum;
          else far_lo += sum;
        } else {
          float* h = hist[wv] + g * width + a.R;
          float one[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) one[r] = DS_SCALED ? ldexpf(ds[r], -ds_log2) : ds[r];
          if (a.G == 1) {
            // The run's diagonals, in a 64-lane shift register: row q's dS for key e enters at lane q and moves up a lane
            // a key, so that all of one distance meet; after key 31 lane i holds distance key0 + 31 - (first row) - i. Keys
            // 8 n .. 8 n + 3 are in the low half wave, the next four in the high one, which the swap brings down. (One LDS
            // add for 32 x 32 values: 2303 tokens of 24 heads, D = 64, this kernel 93 us with each added by itself, as
            // below, and 42 so.)
            float v = 0.0f;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              unsigned up[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(one[4 * n + e]), 0u, false, false);
                v = dpp_f<0x138>(v) + __uint_as_float(two[0]);
                up[e] = two[1];
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) v = dpp_f<0x138>(v) + __uint_as_float(up[e]);
            }
            const int d = key0 + 31 - low - l;
            if (d <= -a.R) far_lo += v;
            else if (d >= a.R) far_hi += v;
            else lds_add(h + d, v);
          } else {
            // One key of the run a step: the 32 rows of a half wave stand at different distances or in different heads, so
            // no two lanes of a half add to one entry; the halves go one after the other, and a wave's LDS operations are
            // done in order: the sums have a fixed order without waiting for each.
            h += d0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int e = 8 * (r / 4) + r % 4, d = d0 + e;
              far_lo += d <= -a.R ? one[r] : 0.0f;
              far_hi += d >= a.R && d > -a.R ? one[r] : 0.0f;
              const bool in = valid && d > -a.R && d < a.R;
              if (in && hi == 0) lds_add(h + e, one[r]);
              __builtin_amdgcn_wave_barrier();  // (keeps the compiler from making one instruction of the two)
              if (in && hi == 1) lds_add(h + e, one[r]);
              __builtin_amdgcn_wave_barrier();
            }
          }
        }
      }
      int change;
      if (DS_SCALED && fit(ds, dq, change)) {
        ds_log2 += change;
        ds_ls -= (float)change;
      }
      const ev8 sa = epack8(&ds[0]), sb8 = epack8(&ds[8]);
      if (!BIAS) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int t0 = toff0 ^ (64 * db), t1 = toff1 ^ (64 * db);
        dq[db] = emfma(ecat_tr(lds_read_tr(kt, t0), lds_read_tr(kt, t1)), sa, dq[db]);
        dq[db] = emfma(ecat_tr(lds_read_tr(kt + TILE_BYTES / 4, t0), lds_read_tr(kt + TILE_BYTES / 4, t1)), sb8, dq[db]);
      }
      if (!BIAS) __builtin_amdgcn_s_setprio(0);
    }
    sb ^= 1;
    dma_wait();
    __syncthreads();
  }

  if (BIAS) {  // the far sums of the wave's rows, head by head
    for (int i = 0; i < a.G; ++i) {
      // (a lane of an invalid row holds zeros, or with one head a group sums of other rows)
      const float lo = wave_sum_dpp(g == i ? far_lo : 0.0f), up = wave_sum_dpp(g == i ? far_hi : 0.0f);
      if (l == 0) {
        hist[wv][i * width] += lo;
        hist[wv][i * width + 2 * a.R] += up;
      }
    }
  }
  if (DS_SCALED) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[db][r] = ldexpf(dq[db][r], -ds_log2);
  }
  // the second key half hands its sums over through the staging buffers
  float* xq = reinterpret_cast<float*>(&kv_s[0][0][0]) + rg * (NDB * 16 * 64);
  if (kh == 1) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) xq[(db * 16 + r) * 64 + l] = dq[db][r];
  }
  __syncthreads();
  if (BIAS)
    for (int i = tid; i < a.G * width; i += 256) dist[i] = (hist[0][i] + hist[1][i]) + (hist[2][i] + hist[3][i]);
  if (kh == 1 || !valid) return;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (dq[db][4 * i + e] + xq[(db * 16 + 4 * i + e) * 64 + l]) * a.scale;
      ushort4 q4;
      q4.x = f2e(x[0]); q4.y = f2e(x[1]); q4.z = f2e(x[2]); q4.w = f2e(x[3]);
      *reinterpret_cast<ushort4*>(a.dq + at + 32 * db + 8 * i + 4 * hi) = q4;
    }
}

// dV and dK from the row ranges' sums, in order: four channels a thread. Memory bound: the sums once (ranges * Tk * Hk * 8 D
// bytes), which the rule below weighs as two steps a range.
template <int D>
__global__ __launch_bounds__(256) void kv_sums_kernel(BwdArgs a) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, rows = (size_t)a.Tk * a.Hk, row = i / (D / 2);
  if (row >= rows) return;
  const int c = (int)(i - row * (D / 2)) * 4;  // channels of [dV | dK]
  f32x4 sum = {};
  for (int r = 0; r < a.ranges; ++r) sum += *reinterpret_cast<const f32x4*>(a.part + (r * rows + row) * 2 * D + c);
  ushort4 o4;
  o4.x = f2e(sum[0]); o4.y = f2e(sum[1]); o4.z = f2e(sum[2]); o4.w = f2e(sum[3]);
  *reinterpret_cast<ushort4*>((c < D ? a.dv + row * D + c : a.dk + row * D + c - D)) = o4;
}

// dbias[n][h] = sum over the row tiles and over the distances of bucket n: one workgroup a head. First each of four slices of
// 256 lanes adds every fourth tile, a distance a lane, eight tiles in flight; then a wave adds up a bucket's distances. Latency
// bound: 2303 tokens of 24 heads 4.1 us.
__global__ __launch_bounds__(1024) void bias_sums_kernel(BwdArgs a) {
  __shared__ float sums[4][BIAS_ROWS];
  __shared__ int which[BIAS_ROWS];
  const int h = blockIdx.x, hk = divide(a.div_g, h), g = h - hk * a.G, width = 2 * a.R + 1;
  const int slice = threadIdx.x >> 8, x = threadIdx.x & 255;
  const size_t step = (size_t)a.Hk * a.G * width;
  for (int d = x; d < width; d += 256) {
    const float* p = a.dist + ((size_t)hk * a.G + g) * width + d;
    float sum[8] = {};
    for (int w = slice; w < a.q_tiles; w += 32)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += w + 4 * e < a.q_tiles ? p[(w + 4 * e) * step] : 0.0f;
    sums[slice][d] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
    if (slice == 0) which[d] = min(max(a.buckets[d], 0), a.num_buckets - 1);
  }
  __syncthreads();
  for (int n = threadIdx.x >> 6; n < a.num_buckets; n += 16) {
    float sum = 0.0f;
    for (int d = threadIdx.x & 63; d < width; d += 64)
      if (which[d] == n) sum += (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
    sum = wave_sum_dpp(sum);
    // (a value that fill_bias holds to its limit does not move the scores)
    const size_t at = (size_t)n * a.H + h;
    if ((threadIdx.x & 63) == 0) a.dbias[at] = fabsf(a.bias[at]) > BIAS_MAX ? 0.0f : sum;
  }
}

}  // namespace

}  // namespace es

using namespace es;

// Row ranges of bwd_kv: one to sixteen, by the shortest schedule in steps of one row tile, for sequences of average length. An
// item takes its row tiles and about four steps before and behind them, two more where its sums go through memory. Without a
// mask all items are alike and run in rounds of what the GPU holds; under a causal one they halve on average, start with the
// longest, and end with it or when all work is done. From two rounds of items on the ranges' memory is not worth it. (Whole
// backward, causal, D = 128, us with one range and by this rule: 8192 tokens of 8 heads over one kv head 1793 -> 675, 2000
// tokens 432 -> 91, 4000 tokens of 40 heads over 5 1086 -> 812, 1000 of 64 over 8 253 -> 125.)
static int row_ranges(int B, int Tq, int Tk, int H, int Hk, int D, int causal) {
  const double items = (double)tile_numbers<BK>(B, Tk, 1) * Hk, steps = (double)Tq * (H / Hk) / B / BK;
  const double slots = D == 64 ? 768 : 512;
  int best = 1;
  double least = 0;
  for (int r = 1; r <= 16 && (r == 1 || (steps >= 4.0 * r && items < 2 * slots)); ++r) {
    const double more = r == 1 ? 4 : 6, each = steps / r;
    const double time = causal ? std::max(each + more, items * r / slots * (each / 2 + more))
                               : std::ceil(items * r / slots) * (each + more);
    if (r == 1 || time < 0.97 * least) {
      least = time;
      best = r;
    }
  }
  return best;
}
// lse2 and delta, the distance sums of every (row tile, kv head), the row ranges' sums
struct Offsets {
  size_t dist, part, floats;
};
static Offsets bwd_layout(int B, int Tq, int Tk, int H, int Hk, int D, int R, int with_bias, int causal) {
  Offsets o;
  o.dist = 2 * (size_t)Tq * H;
  o.part = o.dist + (with_bias ? (size_t)tile_numbers<BK>(B, Tq, H / Hk) * H * (2 * R + 1) : 0);
  o.part = (o.part + 3) / 4 * 4;
  const int ranges = row_ranges(B, Tq, Tk, H, Hk, D, causal);
  o.floats = o.part + (ranges > 1 ? (size_t)ranges * Tk * Hk * 2 * D : 0);
  return o;
}

#ifndef ES_ELEM_F16
extern "C" size_t es_packed_bwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D, int R, int with_bias,
                                          int causal) {
  if (B <= 0 || Tq < 0 || Tk < 0 || H <= 0 || Hk <= 0 || H % Hk || R < 0) return 0;
  return bwd_layout(B, Tq, Tk, H, Hk, D, R, with_bias, causal != 0).floats * sizeof(float);
}
#endif

extern "C" int ES_VSA_API(es_packed_bwd)(const void* q, const void* k, const void* v, const void* dout, const void* out,
                                         const float* lse, const int* cu_q, const int* cu_k, const float* bias,
                                         const int* buckets, int num_buckets, int R, void* dq, void* dk, void* dv,
                                         float* dbias, void* workspace, size_t workspace_bytes, int B, int Tq, int Tk, int H,
                                         int Hk, int D, int causal, float scale, hipStream_t stream) {
  if (int st = packed_check(q, k, v, cu_q, cu_k, bias, buckets, num_buckets, R, B, Tq, Tk, H, Hk, D, scale)) return st;
  ES_REQUIRE((Tq == 0 || (dout && out && lse && dq && workspace)) && (Tk == 0 || (dk && dv)), ES_ERR_INVALID,
             "packed: null tensor pointer");
  ES_REQUIRE(aligned16({q, k, v, dout, out, dq, dk, dv, workspace}), ES_ERR_INVALID,
             "packed: tensors must be aligned to 16 bytes");
  ES_REQUIRE((bias != nullptr) == (dbias != nullptr), ES_ERR_INVALID, "packed: dbias goes with bias");
  ES_REQUIRE(workspace_bytes >= es_packed_bwd_workspace(B, Tq, Tk, H, Hk, D, bias ? R : 0, bias != nullptr, causal),
             ES_ERR_INVALID, "packed: workspace too small");
  BwdArgs a = {};
  a.q = (const e16_t*)q;
  a.k = (const e16_t*)k;
  a.v = (const e16_t*)v;
  a.dout = (const e16_t*)dout;
  a.out = (const e16_t*)out;
  a.lse = lse;
  a.bias = bias;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.buckets = buckets;
  a.dq = (e16_t*)dq;
  a.dk = (e16_t*)dk;
  a.dv = (e16_t*)dv;
  a.dbias = dbias;
  a.lse2 = (float*)workspace;
  a.delta = a.lse2 + (size_t)Tq * H;
  const Offsets o = bwd_layout(B, Tq, Tk, H, Hk, D, bias ? R : 0, bias != nullptr, causal != 0);
  a.dist = a.lse2 + o.dist;
  a.part = a.lse2 + o.part;
  a.ranges = row_ranges(B, Tq, Tk, H, Hk, D, causal != 0);
  a.B = B;
  a.Tq = Tq;
  a.Tk = Tk;
  a.H = H;
  a.Hk = Hk;
  a.G = H / Hk;
  a.div_g = fast_div(a.G);
  a.inv_g = 1.0f / (float)a.G;
  a.R = bias ? R : 0;
  a.num_buckets = num_buckets;
  a.causal = causal != 0;
  a.scale = scale;
  a.scale_log2 = scale * LOG2E;
  a.q_tiles = (int)tile_numbers<BK>(B, Tq, a.G);
  a.k_tiles = (int)tile_numbers<BK>(B, Tk, 1);
  ES_REQUIRE((long long)a.q_tiles * Hk < MAX_GRID && (long long)a.k_tiles * Hk * a.ranges < MAX_GRID, ES_ERR_UNSUPPORTED,
             "packed: too many sequences");
  if (Tq > 0) {
    const dim3 grid((unsigned)(a.q_tiles * Hk));
    if (D == 64) {
      if (bias) hipLaunchKernelGGL((packed_bwd_q_kernel<64, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_bwd_q_kernel<64, false>), grid, dim3(256), 0, stream, a);
    } else {
      if (bias) hipLaunchKernelGGL((packed_bwd_q_kernel<128, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_bwd_q_kernel<128, false>), grid, dim3(256), 0, stream, a);
    }
  }
  if (Tk > 0) {
    const dim3 grid((unsigned)(a.k_tiles * Hk * a.ranges));
    if (D == 64) {
      if (bias) hipLaunchKernelGGL((packed_bwd_kv_kernel<64, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_bwd_kv_kernel<64, false>), grid, dim3(256), 0, stream, a);
    } else {
      if (bias) hipLaunchKernelGGL((packed_bwd_kv_kernel<128, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((packed_bwd_kv_kernel<128, false>), grid, dim3(256), 0, stream, a);
    }
    if (a.ranges > 1) {
      const dim3 sums((unsigned)(((long long)Tk * Hk * (D / 2) + 255) / 256));
      if (D == 64) hipLaunchKernelGGL((kv_sums_kernel<64>), sums, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((kv_sums_kernel<128>), sums, dim3(256), 0, stream, a);
    }
  }
  if (bias) {
    if (Tq == 0) a.q_tiles = 0;
    hipLaunchKernelGGL(bias_sums_kernel, dim3((unsigned)H), dim3(1024), 0, stream, a);
  }
  return check_launch("es_packed_bwd");
}
