// Shared by the kernels of paged caches (paged_*.hip): where a token of a packed batch is held, a head's row over a few lanes, its
// norm and rotation, and the host checks.
//
// A row of D channels is spread over D / 16 lanes of a wave; lane j has the 8-channel chunks j and j + D / 16, so a wave's loads of
// 16 bytes a lane cover whole rows in two pieces, pairs of channels D / 2 apart meet in one lane, and 32 channels (a scale of a
// 4-bit cache) in four neighbouring ones.
#pragma once
#include "../../include/paged_hip.h"
#include "elem.h"
#include "packed_rules.h"

#include <initializer_list>

namespace es {

namespace {

constexpr long long PAGED_GRID = 1LL << 24;  // workgroups of a launch: its threads are counted in 32 bits

// ------------------------------------------------------------------------------------------------ places
struct Places {
  const int *pages, *lens, *cu;
  int B, T, max_pages, num_pages, shift;  // page_size = 1 << shift
  FastDiv div_n;                          // without cu: new tokens of a sequence
};

__device__ __forceinline__ int start_of(const Places& a, int b) {
  if (a.cu == nullptr) return b * (a.T / a.B);
  return b <= 0 ? 0 : min(max(a.cu[b], 0), a.T);
}

// Sequences that end at or before token t (B: t stands behind the last one). With running counts each lane takes one of 64 and the
// answer is searched for among the lanes' values: one load instead of a chain of six. Every lane of the wave calls it.
__device__ __forceinline__ int sequence_of(const Places& a, int t) {
  if (a.cu == nullptr) return divide(a.div_n, t);
  int found = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane_id();
    const int end = b < a.B ? start_of(a, b + 1) : a.T + 1;
    int lo = 0;
#pragma unroll
    for (int step = 32; step >= 1; step >>= 1) lo += __shfl(end, lo + step - 1, 64) <= t ? step : 0;
    lo += __shfl(end, lo, 64) <= t ? 1 : 0;
    found += lo;
    if (!__builtin_amdgcn_ballot_w64(lo == 64)) break;
  }
  return min(found, a.B);
}

// Where token t is held: page < 0: nowhere; position < 0: it has none.
struct Place {
  int position, page, row;
};
__device__ __forceinline__ Place place_of(const Places& a, int t) {
  Place p = {-1, -1, 0};
  const int b = sequence_of(a, t);
  if (b >= a.B || t >= a.T) return p;
  const int len = max(a.lens[b], 0);
  p.position = len - start_of(a, b + 1) + t;
  if (p.position < 0 || p.position >= len) {
    p.position = -1;
    return p;
  }
  const int entry = p.position >> a.shift, page = entry < a.max_pages ? a.pages[(size_t)b * a.max_pages + entry] : -1;
  p.page = page >= 0 && page < a.num_pages ? page : -1;
  p.row = p.position & ((1 << a.shift) - 1);
  return p;
}

// ------------------------------------------------------------------------------------------------ rows
// sums and maxima over the N = 4 or 8 lanes of a row (DPP: quads, then the mirror of eight lanes), the same bits on all of them
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp_f<0xB1>(x);
  x += dpp_f<0x4E>(x);
  if (N == 8) x += dpp_f<0x141>(x);
  return x;
}
template <int CTRL>
__device__ __forceinline__ double dpp_d(double x) {
  const long long b = __builtin_bit_cast(long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (long long)(((unsigned long long)hi << 32) | lo));
}
template <int N>
__device__ __forceinline__ double lanes_sum(double x) {
  x += dpp_d<0xB1>(x);
  x += dpp_d<0x4E>(x);
  if (N == 8) x += dpp_d<0x141>(x);
  return x;
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, dpp_f<0xB1>(x));
  return fmaxf(x, dpp_f<0x4E>(x));
}

__device__ __forceinline__ ev8 load8(const e16_t* p) { return *reinterpret_cast<const ev8*>(p); }
__device__ __forceinline__ void store8(e16_t* p, const float* x) {
  *reinterpret_cast<ev8*>(p) = epack8(x);
}

// how the channels are paired: neighbours, the two halves of a row, the two halves of its first R < D channels
enum Pairs { NEIGHBOURS, HALVES, PART_HALVES };

// Partner chunk of chunk c under PART_HALVES, -1: not rotated; second: the pair's second channel
__device__ __forceinline__ int partner(int c, int half, bool& second) {
  second = c >= half;
  return c < half ? c + half : c < 2 * half ? c - half : -1;
}

// The cosines and sines that a lane needs for its two chunks.
template <int D, int PAIRS>
struct Angles {
  static constexpr int N = PAIRS == PART_HALVES ? 16 : 8;
  float c[N], s[N];
  bool turn[2];  // whether chunk i is rotated

  __device__ __forceinline__ void load(const float* row, int j, int R) {
    const float4* p = reinterpret_cast<const float4*>(row);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = j + i * (D / 16);
      turn[i] = 8 * chunk < R;
      if (PAIRS == HALVES && i == 1) break;
      // pairs of the chunk, two to a float4: four under NEIGHBOURS from 4 chunk on, otherwise eight from 8 (chunk % half) on
      constexpr int M = PAIRS == NEIGHBOURS ? 4 : 8;
      const int at = PAIRS == NEIGHBOURS ? 2 * chunk : 4 * (PAIRS == PART_HALVES && 16 * chunk >= R ? chunk - R / 16 : chunk);
#pragma unroll
      for (int e = 0; e < M; e += 2) {
        const float4 x = turn[i] ? p[at + e / 2] : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
        c[M * i + e] = x.x, s[M * i + e] = x.y, c[M * i + e + 1] = x.z, s[M * i + e + 1] = x.w;
      }
    }
    if (PAIRS == HALVES) turn[1] = turn[0];
  }

  // x[0 .. 7] and x[8 .. 15]: the lane's chunks; y: their partners (PART_HALVES only). back: by the negative angles.
  __device__ __forceinline__ void apply(float* x, const float* y, bool back, const bool* second) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (PAIRS == NEIGHBOURS) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float cc = c[4 * i + e], ss = back ? -s[4 * i + e] : s[4 * i + e];
          const float a = x[8 * i + 2 * e], b = x[8 * i + 2 * e + 1];
          if (turn[i]) x[8 * i + 2 * e] = a * cc - b * ss, x[8 * i + 2 * e + 1] = a * ss + b * cc;
        }
      } else if (PAIRS == HALVES) {
        if (i == 1) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float cc = c[e], ss = back ? -s[e] : s[e], a = x[e], b = x[8 + e];
          x[e] = a * cc - b * ss, x[8 + e] = a * ss + b * cc;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float cc = c[(8 * i + e) % N], ss = back != second[i] ? s[(8 * i + e) % N] : -s[(8 * i + e) % N];
          if (turn[i]) x[8 * i + e] = x[8 * i + e] * cc + y[8 * i + e] * ss;
        }
      }
    }
  }
};

// A lane's 16 (PART_HALVES: also the partners' 16) weights of the norm
template <int D, int PAIRS>
struct Weights {
  static constexpr int N = PAIRS == PART_HALVES ? 32 : 16;
  float w[N];
  __device__ __forceinline__ void load(const void* p, int f32, int j, int R) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      int chunk = j + (i & 1) * (D / 16);
      if (i >= 2) {
        bool second;
        const int other = partner(chunk, R / 16, second);
        chunk = other < 0 ? chunk : other;
      }
      if (f32) {
        const float4* q = reinterpret_cast<const float4*>(p) + 2 * chunk;
        const float4 a = q[0], b = q[1];
        w[8 * i] = a.x, w[8 * i + 1] = a.y, w[8 * i + 2] = a.z, w[8 * i + 3] = a.w;
        w[8 * i + 4] = b.x, w[8 * i + 5] = b.y, w[8 * i + 6] = b.z, w[8 * i + 7] = b.w;
      } else {
        const ev8 v = load8(reinterpret_cast<const e16_t*>(p) + 8 * chunk);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[8 * i + e] = (float)v[e];
      }
    }
  }
};

// A row as it was loaded: the lane's two chunks, under PART_HALVES also their partners.
template <int D, int PAIRS>
struct RawRow {
  static constexpr int N = PAIRS == PART_HALVES ? 4 : 2;
  ev8 v[N];
  __device__ __forceinline__ void load(const e16_t* row, int j, int R) {
    v[0] = load8(row + 8 * j);
    v[1] = load8(row + 8 * (j + D / 16));
    if (PAIRS == PART_HALVES) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int chunk = j + i * (D / 16);
        bool second;
        const int other = partner(chunk, R / 16, second);
        v[2 + i] = load8(row + 8 * (other < 0 ? chunk : other));
      }
    }
  }
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[8 * i + e] = (float)v[i][e];
  }
};

// 1 / sqrt(mean x^2 + eps) of a row
template <int D>
__device__ __forceinline__ float inverse_rms(const float* x, float eps) {
  float sum = x[0] * x[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) sum += x[e] * x[e];
  return rsqrtf(lanes_sum<D / 16>(sum) * (1.0f / D) + eps);
}

// x (16 values of the lane, under PART_HALVES with their partners' behind them), normed and rotated
template <int D, int PAIRS, bool NORM>
__device__ __forceinline__ void norm_rotate_row(float* x, const Weights<D, PAIRS>& w, const Angles<D, PAIRS>& angles, int j, int R,
                                                float eps) {
  if (NORM) {
    const float r = inverse_rms<D>(x, eps);
#pragma unroll
    for (int e = 0; e < Weights<D, PAIRS>::N; ++e) x[e] = x[e] * r * w.w[e];
  }
  const bool second[2] = {j >= R / 16, j + D / 16 >= R / 16};
  angles.apply(x, x + (PAIRS == PART_HALVES ? 16 : 0), false, second);
}

// The same in 64 bits, rounded to float32: a pair at a time, so that few values are held in 64 bits.
template <int D, int PAIRS, bool NORM>
__device__ __forceinline__ void norm_rotate_exact(const RawRow<D, PAIRS>& raw, const Weights<D, PAIRS>& w,
                                                  const Angles<D, PAIRS>& angles, int j, int R, double eps, float* y) {
  double r = 1.0;
  if (NORM) {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const double x = (double)(float)raw.v[e / 8][e % 8];
      sum += x * x;  // (a bf16 value's square has 16 digits, but float32 ends at values of 1.8e19 and 1e-19)
    }
    r = 1.0 / sqrt(lanes_sum<D / 16>(sum) * (1.0 / D) + eps);
  }
  auto value = [&](int e) {
    const double x = (double)(float)raw.v[e / 8][e % 8];
    return NORM ? x * r * (double)w.w[e] : x;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (PAIRS == NEIGHBOURS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 8 * i + 2 * e;
        const double a = value(k), b = value(k + 1), c = angles.c[4 * i + e], s = angles.s[4 * i + e];
        y[k] = (float)(angles.turn[i] ? a * c - b * s : a);
        y[k + 1] = (float)(angles.turn[i] ? a * s + b * c : b);
      }
    } else if (PAIRS == HALVES) {
      if (i == 1) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double a = value(e), b = value(8 + e), c = angles.c[e], s = angles.s[e];
        y[e] = (float)(a * c - b * s);
        y[8 + e] = (float)(a * s + b * c);
      }
    } else {
      const bool second = j + i * (D / 16) >= R / 16;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 8 * i + e, n = k % Angles<D, PAIRS>::N;
        const double a = value(k), b = value((16 + k) % (8 * RawRow<D, PAIRS>::N)), s = second ? angles.s[n] : -angles.s[n];
        y[k] = (float)(angles.turn[i] ? a * (double)angles.c[n] + b * s : a);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ 4 bits
// exponents of the scales: with them every value of a code is a normal number of the token type
#ifdef ES_ELEM_F16
constexpr int SCALE_MIN = -13, SCALE_MAX = 13;
#else
constexpr int SCALE_MIN = -120, SCALE_MAX = 120;
#endif

// The scale of 32 channels whose largest magnitude is `top`, as its float bits >> 23 (= exponent + 127): the smallest power of two
// s with top <= 7 s. (7 and not 6, the largest value: what lies between is off by at most half the step from 4 to 6, and the other
// 31 keep twice the resolution that the next power would leave them.)
__device__ __forceinline__ int scale_of(float top) {
  const unsigned bits = __float_as_uint(top);
  const int e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, SCALE_MIN), SCALE_MAX) + 127;
}
// the codes of 8 values, the first in the lowest bits; to nearest, ties to even
__device__ __forceinline__ unsigned encode8(const float* x, float scale) {
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
}
// 8 codes as token values (exact)
__device__ __forceinline__ ev8 decode8(unsigned c, float scale) {
#ifdef ES_ELEM_F16
#define ES_DECODE2(i) __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, i)
#else
#define ES_DECODE2(i) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, i)
#endif
  const auto p0 = ES_DECODE2(0), p1 = ES_DECODE2(1), p2 = ES_DECODE2(2), p3 = ES_DECODE2(3);
#undef ES_DECODE2
  ev8 r;
  __builtin_memcpy(&r, &p0, 4);
  __builtin_memcpy((char*)&r + 4, &p1, 4);
  __builtin_memcpy((char*)&r + 8, &p2, 4);
  __builtin_memcpy((char*)&r + 12, &p3, 4);
  return r;
}

}  // namespace

// ------------------------------------------------------------------------------------------------ host checks
static inline bool all_aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

// what the entry points that norm and rotate have in common
static inline int rotate_check(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* table, int T,
                               int H, int Hk, int D, int R, int P, double eps) {
  ES_REQUIRE(D == 64 || D == 128, ES_ERR_UNSUPPORTED, "rotate: head dim must be 64 or 128");
  ES_REQUIRE(T >= 0 && H >= 0 && Hk >= 0 && H <= 4096 && Hk <= 4096, ES_ERR_INVALID, "rotate: bad sizes (at most 4096 heads)");
  ES_REQUIRE(T == 0 || ((H == 0 || q) && (Hk == 0 || k)), ES_ERR_INVALID, "rotate: null q / k");
  ES_REQUIRE((H == 0 || Hk == 0 || !q_weight == !k_weight) && (H > 0 || !q_weight) && (Hk > 0 || !k_weight), ES_ERR_INVALID,
             "rotate: both weights or none");
  ES_REQUIRE(R >= 0 && R <= D && R % 16 == 0 && (R == 0) == (table == nullptr), ES_ERR_INVALID,
             "rotate: R must be a multiple of 16 up to the head dim, 0 without a table");
  ES_REQUIRE(R == 0 || P > 0, ES_ERR_INVALID, "rotate: the table has no rows");
  ES_REQUIRE(eps >= 0.0 && eps < 1e30, ES_ERR_INVALID, "rotate: eps must be finite and not negative");
  ES_REQUIRE(all_aligned16({q, k, q_weight, k_weight, table}), ES_ERR_INVALID, "rotate: tensors must be aligned to 16 bytes");
  return ES_OK;
}
// rows of `heads` heads a stride apart do not run into each other
static inline bool stride_fits(long long stride, int heads, int D, int T) {
  return heads == 0 || (stride % 8 == 0 && stride >= (T > 1 ? (long long)heads * D : 0) && stride < (1LL << 40));
}

static inline int places_check(const int* pages, const int* lens, const int* cu, int B, int T, int max_pages, int num_pages,
                               int page_size, int Hk) {
  ES_REQUIRE(B > 0 && T >= 0 && max_pages >= 0 && num_pages >= 0 && Hk > 0, ES_ERR_INVALID, "paged: bad sizes");
  ES_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0, ES_ERR_UNSUPPORTED,
             "paged: the page size must be a power of two from 16 to 4096");
  ES_REQUIRE((long long)max_pages * page_size < (1LL << 30) && (long long)B < (1LL << 24), ES_ERR_UNSUPPORTED,
             "paged: too many pages or sequences");
  ES_REQUIRE(lens && (max_pages == 0 || pages), ES_ERR_INVALID, "paged: null pages / lens");
  ES_REQUIRE(cu || T % B == 0, ES_ERR_INVALID, "paged: without cu the tokens must divide into B equal counts");
  return ES_OK;
}
// (strides: a page's rows a head, in any order of page, head and row)
static inline int cache_check(const void* k, const void* v, int num_pages, int page_size, int Hk, int D, long long page_stride,
                              long long head_stride, long long row_stride) {
  ES_REQUIRE((num_pages == 0 || (k && v)) && all_aligned16({k, v}), ES_ERR_INVALID,
             "paged: the cache must be given and aligned to 16 bytes");
  for (long long s : {page_stride, head_stride, row_stride})
    ES_REQUIRE(s >= 0 && s % 8 == 0 && s < (1LL << 40), ES_ERR_INVALID, "paged: strides of the cache must be multiples of 8");
  ES_REQUIRE(row_stride >= D && row_stride * 2 * 64 < (1LL << 31), ES_ERR_INVALID, "paged: the row stride must hold a row");
  return ES_OK;
}
static inline int cache4_check(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                               int num_pages) {
  ES_REQUIRE((num_pages == 0 || (k_codes && k_scales && v_codes && v_scales)) &&
                 all_aligned16({k_codes, k_scales, v_codes, v_scales}),
             ES_ERR_INVALID, "paged: the cache must be given and aligned to 16 bytes");
  return ES_OK;
}
static inline int log2_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}
static inline Places make_places(const int* pages, const int* lens, const int* cu, int B, int T, int max_pages, int num_pages,
                                 int page_size) {
  return Places{pages, lens, cu, B, T, max_pages, num_pages, log2_of(page_size), fast_div(T / B > 0 ? T / B : 1)};
}

// calls f with the integral constants of the head dim and the pairing, and whether there is a norm
template <class F>
static inline void for_rotation(int D, int R, int halves, bool norm, F f) {
  auto pairs = [&](auto d, auto n) {
    constexpr int dim = decltype(d)::value;
    if (!halves || R == 0) f(d, std::integral_constant<int, NEIGHBOURS>{}, n);
    else if (R == dim) f(d, std::integral_constant<int, HALVES>{}, n);
    else f(d, std::integral_constant<int, PART_HALVES>{}, n);
  };
  auto dims = [&](auto n) {
    if (D == 64) pairs(std::integral_constant<int, 64>{}, n);
    else pairs(std::integral_constant<int, 128>{}, n);
  };
  if (norm) dims(std::true_type{});
  else dims(std::false_type{});
}

}  // namespace es
