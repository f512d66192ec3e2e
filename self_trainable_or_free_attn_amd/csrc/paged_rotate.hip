// Norm of every head's query and key row and its rotation by position, in one pass, and the backward of that (gfx950, bf16 / fp16).
//
//   forward   y = R(position) (x r w), r = 1 / sqrt(mean x^2 + eps)
//   backward  g = R(-position) dy, h = g w: dx = r (h - xh mean(h xh)) with xh = x r; dw = sum over rows of g xh
//
// Bound by HBM: every row is read and written once (backward: x and dy read, dx written, xh recomputed). A row takes D / 16 lanes
// (paged.h); a lane takes UNIT heads of a token one behind the other, so that the token's angles are loaded once for them and
// UNIT rows' loads are in flight together.
// Weight gradients: a workgroup keeps to queries or keys, each lane adds up its 16 channels over its rows in registers, the lanes
// of a workgroup are added through LDS in order, and a second launch adds the workgroups' sums: no atomics, the same bits every
// time.
#include "paged.h"

#include <algorithm>
#include <type_traits>

namespace es {

namespace {

constexpr int UNIT = 4;  // heads of a lane group

struct RotateArgs {
  const e16_t *x[2], *dy[2];  // queries, keys
  e16_t* y[2];                // outputs; backward: gradients
  const void* w[2];
  const float* table;
  const int* positions;
  float* sums;  // backward: a workgroup's D sums
  long long stride[2];
  int heads[2], units[2];  // units of UNIT heads of a token
  int blocks[2];           // backward: workgroups of each
  FastDiv div_units, div_unit[2];
  int T, L, R, P, f32;
  float eps;
};

__device__ __forceinline__ int position_of(const RotateArgs& a, int t) {
  const int p = a.positions ? a.positions[t] : a.L == a.T ? t : t % a.L;
  return min(max(p, 0), a.P - 1);
}

template <int D, int PAIRS, bool NORM>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
  constexpr int LPR = D / 16, GROUPS = 256 / LPR;
  const int j = threadIdx.x % LPR;
  const long long u = (long long)blockIdx.x * GROUPS + threadIdx.x / LPR;
  const int units = a.units[0] + a.units[1];
  if (u >= (long long)a.T * units) return;
  const int t = divide(a.div_units, (int)u);
  int part = (int)u - t * units;
  const int which = part >= a.units[0];
  part -= which ? a.units[0] : 0;
  const int head0 = part * UNIT, heads = min(a.heads[which] - head0, UNIT);
  const e16_t* x = a.x[which] + (size_t)t * a.stride[which] + (size_t)head0 * D;
  e16_t* y = a.y[which] + ((size_t)t * a.heads[which] + head0) * D;
  RawRow<D, PAIRS> raw[UNIT];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) raw[i].load(x + min(i, heads - 1) * D, j, a.R);
  Angles<D, PAIRS> angles;
  angles.load(a.table + (size_t)(a.R ? position_of(a, t) : 0) * a.R, j, a.R);
  Weights<D, PAIRS> w;
  if (NORM) w.load(a.w[which], a.f32, j, a.R);
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    if (i >= heads) break;
    float v[8 * RawRow<D, PAIRS>::N];
    raw[i].get(v);
    norm_rotate_row<D, PAIRS, NORM>(v, w, angles, j, a.R, a.eps);
    store8(y + i * D + 8 * j, v);
    store8(y + i * D + 8 * (j + D / 16), v + 8);
  }
}

template <int D, int PAIRS, bool NORM>
__global__ __launch_bounds__(256) void rotate_bwd_kernel(RotateArgs a) {
  constexpr int LPR = D / 16, GROUPS = 256 / LPR;
  const int j = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int which = (int)blockIdx.x >= a.blocks[0], block = blockIdx.x - (which ? a.blocks[0] : 0);
  const long long units = (long long)a.T * a.units[which], step = (long long)a.blocks[which] * GROUPS;
  Weights<D, NEIGHBOURS> w;
  if (NORM) w.load(a.w[which], a.f32, j, a.R);
  float sum[16] = {};
  for (long long u = (long long)block * GROUPS + group; u < units; u += step) {
    const int t = divide(a.div_unit[which], (int)u), head0 = ((int)u - t * a.units[which]) * UNIT;
    const int heads = min(a.heads[which] - head0, UNIT);
    const e16_t* x = a.x[which] + (size_t)t * a.stride[which] + (size_t)head0 * D;
    const size_t at = ((size_t)t * a.heads[which] + head0) * D;
    RawRow<D, PAIRS> dy[UNIT];
    RawRow<D, NEIGHBOURS> raw[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      dy[i].load(a.dy[which] + at + min(i, heads - 1) * D, j, a.R);
      if (NORM) raw[i].load(x + min(i, heads - 1) * D, j, a.R);
    }
    Angles<D, PAIRS> angles;
    angles.load(a.table + (size_t)(a.R ? position_of(a, t) : 0) * a.R, j, a.R);
    const bool second[2] = {j >= a.R / 16, j + D / 16 >= a.R / 16};
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      if (i >= heads) break;
      float g[8 * RawRow<D, PAIRS>::N];
      dy[i].get(g);
      angles.apply(g, g + (PAIRS == PART_HALVES ? 16 : 0), true, second);
      if (NORM) {
        float xh[16], dot = 0.0f;
        raw[i].get(xh);
        const float r = inverse_rms<D>(xh, a.eps);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          xh[e] *= r;
          sum[e] = fmaf(g[e], xh[e], sum[e]);
          g[e] *= w.w[e];
          dot = fmaf(g[e], xh[e], dot);
        }
        dot = lanes_sum<LPR>(dot) * (1.0f / D);
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e] = r * fmaf(-xh[e], dot, g[e]);
      }
      store8(a.y[which] + at + i * D + 8 * j, g);
      store8(a.y[which] + at + i * D + 8 * (j + D / 16), g + 8);
    }
  }
  if (!NORM) return;
  __shared__ float lds[GROUPS][D];
#pragma unroll
  for (int e = 0; e < 16; ++e) lds[group][8 * (j + (e / 8) * (D / 16)) + e % 8] = sum[e];
  __syncthreads();
  if (threadIdx.x < D) {
    float s = 0.0f;
#pragma unroll 8
    for (int i = 0; i < GROUPS; ++i) s += lds[i][threadIdx.x];
    a.sums[(size_t)blockIdx.x * D + threadIdx.x] = s;
  }
}

// dw: grid (D / 16, 2), 16 channels a workgroup, each by 64 lanes' runs of the workgroups' sums (16 lanes each took 15 us for 1024
// sums, these 4)
__global__ __launch_bounds__(1024) void weight_sums_kernel(const float* sums, int blocks_q, int blocks_k, int D, void* dq_weight,
                                                           void* dk_weight, int f32) {
  const int which = blockIdx.y, n = which ? blocks_k : blocks_q;
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
  const float* p = sums + (size_t)(which ? blocks_q : 0) * D + c;
  float s = 0.0f;
#pragma unroll 4
  for (int i = run; i < n; i += 64) s += p[(size_t)i * D];
  __shared__ float lds[64][16];
  lds[run][threadIdx.x & 15] = s;
  for (int m = 32; m >= 1; m >>= 1) {
    __syncthreads();
    if (run < m) lds[run][threadIdx.x & 15] += lds[run + m][threadIdx.x & 15];
  }
  void* out = which ? dk_weight : dq_weight;
  if (run != 0 || out == nullptr) return;
  s = lds[0][threadIdx.x];
  if (f32) reinterpret_cast<float*>(out)[c] = s;
  else reinterpret_cast<e16_t*>(out)[c] = f2e(s);
}

}  // namespace

// Workgroups of the backward: four a CU for queries and keys together, each at least one pass of its lane groups.
static void bwd_blocks(int T, int H, int Hk, int D, int* blocks) {
  const int groups = 256 / (D / 16);
  const long long q = ((long long)T * ((H + UNIT - 1) / UNIT) + groups - 1) / groups;
  const long long k = ((long long)T * ((Hk + UNIT - 1) / UNIT) + groups - 1) / groups;
  const long long most = 1024, all = q + k;
  blocks[0] = (int)(all <= most ? q : std::max<long long>(q > 0, q * most / all));
  blocks[1] = (int)(all <= most ? k : std::max<long long>(k > 0, most - blocks[0]));
}

#ifndef ES_ELEM_F16
extern "C" size_t es_norm_rotate_workspace(int T, int H, int Hk, int D) {
  if (T <= 0 || H < 0 || Hk < 0 || (D != 64 && D != 128)) return 0;
  int blocks[2];
  bwd_blocks(T, H, Hk, D, blocks);
  return (size_t)(blocks[0] + blocks[1]) * D * sizeof(float);
}
#endif

static RotateArgs rotate_args(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* table,
                              const int* positions, void* q_out, void* k_out, int T, int L, int H, int Hk, int R, int P,
                              int weight_f32, double eps, long long q_stride, long long k_stride) {
  RotateArgs a = {};
  a.x[0] = (const e16_t*)q, a.x[1] = (const e16_t*)k;
  a.y[0] = (e16_t*)q_out, a.y[1] = (e16_t*)k_out;
  a.w[0] = q_weight, a.w[1] = k_weight;
  a.table = table;
  a.positions = positions;
  a.stride[0] = q_stride, a.stride[1] = k_stride;
  a.heads[0] = H, a.heads[1] = Hk;
  for (int i = 0; i < 2; ++i) {
    a.units[i] = (a.heads[i] + UNIT - 1) / UNIT;
    a.div_unit[i] = fast_div(a.units[i]);
  }
  a.div_units = fast_div(a.units[0] + a.units[1]);
  a.T = T, a.L = L, a.R = R, a.P = P, a.f32 = weight_f32;
  a.eps = (float)eps;
  return a;
}
static int rotate_sizes(int T, int L, int H, int Hk, int D, long long q_stride, long long k_stride) {
  ES_REQUIRE(L > 0, ES_ERR_INVALID, "rotate: L must be positive");
  ES_REQUIRE(stride_fits(q_stride, H, D, T) && stride_fits(k_stride, Hk, D, T), ES_ERR_INVALID,
             "rotate: row strides must be multiples of 8 that hold a row");
  ES_REQUIRE((long long)T * ((H + 3) / 4 + (Hk + 3) / 4) < (1LL << 30), ES_ERR_UNSUPPORTED, "rotate: too many rows");
  return ES_OK;
}

}  // namespace es

using namespace es;

extern "C" int ES_VSA_API(es_norm_rotate)(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                          const float* table, const int* positions, void* q_out, void* k_out, int T, int L, int H,
                                          int Hk, int D, int R, int P, int halves, int weight_f32, double eps, long long q_stride,
                                          long long k_stride, hipStream_t stream) {
  if (int st = rotate_check(q, k, q_weight, k_weight, table, T, H, Hk, D, R, P, eps)) return st;
  if (T == 0 || H + Hk == 0) return ES_OK;
  if (int st = rotate_sizes(T, L, H, Hk, D, q_stride, k_stride)) return st;
  ES_REQUIRE((H == 0 || q_out) && (Hk == 0 || k_out) && all_aligned16({q_out, k_out}), ES_ERR_INVALID,
             "rotate: outputs must be given and aligned to 16 bytes");
  const RotateArgs a = rotate_args(q, k, q_weight, k_weight, table, positions, q_out, k_out, T, L, H, Hk, R, P, weight_f32, eps,
                                   q_stride, k_stride);
  const long long units = (long long)T * (a.units[0] + a.units[1]), groups = 256 / (D / 16);
  const long long blocks = (units + groups - 1) / groups;
  ES_REQUIRE(blocks < PAGED_GRID, ES_ERR_UNSUPPORTED, "rotate: too many rows");
  for_rotation(D, R, halves, q_weight || k_weight, [&](auto d, auto pairs, auto norm) {
    hipLaunchKernelGGL((rotate_kernel<decltype(d)::value, decltype(pairs)::value, decltype(norm)::value>), dim3((unsigned)blocks),
                       dim3(256), 0, stream, a);
  });
  return check_launch("es_norm_rotate");
}

extern "C" int ES_VSA_API(es_norm_rotate_bwd)(const void* q, const void* k, const void* dq_out, const void* dk_out,
                                              const void* q_weight, const void* k_weight, const float* table,
                                              const int* positions, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                              void* workspace, size_t workspace_bytes, int T, int L, int H, int Hk, int D, int R,
                                              int P, int halves, int weight_f32, double eps, long long q_stride,
                                              long long k_stride, hipStream_t stream) {
  if (int st = rotate_check(q, k, q_weight, k_weight, table, T, H, Hk, D, R, P, eps)) return st;
  const bool norm = q_weight || k_weight;
  ES_REQUIRE(!norm || ((H == 0 || dq_weight) && (Hk == 0 || dk_weight)), ES_ERR_INVALID, "rotate: null gradient of a weight");
  if (H + Hk == 0) return ES_OK;
  if (T > 0) {
    if (int st = rotate_sizes(T, L, H, Hk, D, q_stride, k_stride)) return st;
    ES_REQUIRE((H == 0 || (dq && dq_out)) && (Hk == 0 || (dk && dk_out)) && all_aligned16({dq, dk, dq_out, dk_out, workspace}),
               ES_ERR_INVALID, "rotate: gradients must be given and aligned to 16 bytes");
  }
  RotateArgs a = rotate_args(q, k, q_weight, k_weight, table, positions, dq, dk, T, L > 0 ? L : 1, H, Hk, R, P, weight_f32, eps,
                             q_stride, k_stride);
  a.dy[0] = (const e16_t*)dq_out, a.dy[1] = (const e16_t*)dk_out;
  if (T > 0) bwd_blocks(T, H, Hk, D, a.blocks);  // (no tokens: no sums, gradients of the weights are zeros)
  if (norm) {
    ES_REQUIRE(T == 0 || (workspace && workspace_bytes >= es_norm_rotate_workspace(T, H, Hk, D)), ES_ERR_INVALID,
               "rotate: workspace too small");
    a.sums = (float*)workspace;
  }
  if (T > 0) {
    for_rotation(D, R, halves, norm, [&](auto d, auto pairs, auto with) {
      hipLaunchKernelGGL((rotate_bwd_kernel<decltype(d)::value, decltype(pairs)::value, decltype(with)::value>),
                         dim3((unsigned)(a.blocks[0] + a.blocks[1])), dim3(256), 0, stream, a);
    });
  }
  if (norm)
    hipLaunchKernelGGL(weight_sums_kernel, dim3(D / 16, 2), dim3(1024), 0, stream, a.sums, a.blocks[0], a.blocks[1], D,
                       dq_weight, dk_weight, weight_f32);
  return check_launch("es_norm_rotate_bwd");
}
