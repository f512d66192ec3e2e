// New tokens into a paged cache, and rows of a cache back as tokens (gfx950, bf16 / fp16, caches of 16 or 4 bits).
//
// append: a lane group (paged.h) takes UNIT heads of a token's queries, keys or values. Queries and keys are normed and rotated,
// queries go to a tensor of their own, keys and values to the row of the token's page. One launch does all three, since a step of
// single tokens is bound by launches and by the chain of loads from the running lengths to the page number and the angles.
// 4 bits: a lane's 8 channels are a quarter of the 32 that share a scale. Keys are normed and rotated in 64 bits there: a code then
// follows from the formula alone and not from the order of float32 operations, which moves values that stand next to a border of
// two codes by a whole step. They take one head a lane group: the angles and weights of UNIT heads would be held in 64 bits (171
// registers a lane instead of 106, and 5696 tokens of 40 heads over 8 take 44.7 us instead of 37.9).
#include "paged.h"

#include <type_traits>

namespace es {

namespace {

constexpr int UNIT = 4;  // heads of a lane group

struct AppendArgs {
  const e16_t* x[3];  // queries, keys, values
  const void* w[2];
  const float* table;
  e16_t *q_out, *pages[2];
  uint8_t *codes[2], *scales[2];
  Places places;
  long long stride[3], page_stride, head_stride, row_stride;
  int heads[3], units[3];
  FastDiv div_units;
  int T, Hk, R, P, f32;
  double eps;
};

// 32 channels of a row: this lane's 8 of chunk `chunk` as codes, the scale by the quad's first lane
__device__ __forceinline__ void hold4(const float* x, uint8_t* codes, uint8_t* scales, int chunk, int j) {
  float top = fabsf(x[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
  const int scale = scale_of(quad_max(top));
  *reinterpret_cast<unsigned*>(codes + 4 * chunk) = encode8(x, __uint_as_float((unsigned)scale << 23));
  if (j % 4 == 0) scales[chunk / 4] = (uint8_t)scale;
}

template <int D, int PAIRS, bool NORM, int BITS>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int LPR = D / 16, GROUPS = 256 / LPR;
  const int j = threadIdx.x % LPR;
  const int units = a.units[0] + a.units[1] + a.units[2];
  const long long u = (long long)blockIdx.x * GROUPS + threadIdx.x / LPR, last = (long long)a.T * units - 1;
  const int t = divide(a.div_units, (int)(u < last ? u : last));
  int part = (int)(u < last ? u : last) - t * units;
  const int which = part < a.units[0] ? 0 : part < a.units[0] + a.units[1] ? 1 : 2;
  part -= which == 0 ? 0 : which == 1 ? a.units[0] : a.units[0] + a.units[1];
  const int step = BITS == 4 && which == 1 ? 1 : UNIT, head0 = part * step, heads = min(a.heads[which] - head0, step);
  const e16_t* x = a.x[which] + (size_t)t * a.stride[which] + (size_t)head0 * D;
  RawRow<D, PAIRS> raw[UNIT];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) raw[i].load(x + min(i, heads - 1) * D, j, a.R);
  Weights<D, PAIRS> w;
  if (NORM && which < 2) w.load(a.w[which], a.f32, j, a.R);
  const Place place = place_of(a.places, t);
  if (u > last) return;
  if (place.position < 0 || (which > 0 && place.page < 0)) {
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < UNIT; ++i) {
        if (i >= heads) break;
        e16_t* y = a.q_out + ((size_t)t * a.heads[0] + head0 + i) * D;
        *reinterpret_cast<ev8*>(y + 8 * j) = ev8{};
        *reinterpret_cast<ev8*>(y + 8 * (j + D / 16)) = ev8{};
      }
    }
    return;
  }
  Angles<D, PAIRS> angles;
  if (which < 2) angles.load(a.table + (size_t)(a.R ? min(place.position, a.P - 1) : 0) * a.R, j, a.R);
  auto hold = [&](const float* v, int head) {
    const size_t row = (((size_t)place.page * a.Hk + head) << a.places.shift) + place.row;
    uint8_t* codes = a.codes[which - 1] + row * (D / 2);
    uint8_t* scales = a.scales[which - 1] + row * (D / 32);
    hold4(v, codes, scales, j, j);
    hold4(v + 8, codes, scales, j + D / 16, j);
  };
  if (BITS == 4 && which == 1) {
    float v[16];
    norm_rotate_exact<D, PAIRS, NORM>(raw[0], w, angles, j, a.R, a.eps, v);
    hold(v, head0);
    return;
  }
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    if (i >= heads) break;
    const int head = head0 + i;
    float v[8 * RawRow<D, PAIRS>::N];
    raw[i].get(v);
    if (which < 2) norm_rotate_row<D, PAIRS, NORM>(v, w, angles, j, a.R, (float)a.eps);
    if (BITS == 4 && which > 0) {
      hold(v, head);
      continue;
    }
    e16_t* y = which == 0 ? a.q_out + ((size_t)t * a.heads[0] + head) * D
                          : a.pages[which - 1] + (size_t)place.page * a.page_stride + (size_t)head * a.head_stride +
                                (size_t)place.row * a.row_stride;
    store8(y + 8 * j, v);
    store8(y + 8 * (j + D / 16), v + 8);
  }
}

struct RowsArgs {
  const e16_t* pages[2];
  const uint8_t *codes[2], *scales[2];
  e16_t* out[2];
  Places places;
  long long page_stride, head_stride, row_stride;
  FastDiv div_units;
  int T, Hk, units;  // units of UNIT heads
};

// D / 8 lanes a row; a lane group takes UNIT heads of a token's keys or values (one head a group looked the token's place up as
// often as it moved a row: 5696 tokens of 8 heads from 4 bits 11.0 us, so 7.4)
template <int D, int BITS>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  constexpr int LPR = D / 8;
  const int c = threadIdx.x % LPR, units = 2 * a.units;
  const long long u = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR, last = (long long)a.T * units - 1;
  const int t = divide(a.div_units, (int)(u < last ? u : last));
  int part = (int)(u < last ? u : last) - t * units;
  const int which = part >= a.units, head0 = (part - (which ? a.units : 0)) * UNIT, heads = min(a.Hk - head0, UNIT);
  const Place place = place_of(a.places, t);
  if (u > last) return;
  ev8 x[UNIT] = {};
  if (place.page >= 0) {
    if (BITS == 16) {
      const e16_t* p = a.pages[which] + (size_t)place.page * a.page_stride + (size_t)place.row * a.row_stride + 8 * c;
#pragma unroll
      for (int i = 0; i < UNIT; ++i) x[i] = load8(p + (size_t)(head0 + min(i, heads - 1)) * a.head_stride);
    } else {
      unsigned codes[UNIT], scales[UNIT];
#pragma unroll
      for (int i = 0; i < UNIT; ++i) {
        const size_t row = (((size_t)place.page * a.Hk + head0 + min(i, heads - 1)) << a.places.shift) + place.row;
        codes[i] = *reinterpret_cast<const unsigned*>(a.codes[which] + row * (D / 2) + 4 * c);
        scales[i] = a.scales[which][row * (D / 32) + c / 4];
      }
#pragma unroll
      for (int i = 0; i < UNIT; ++i) x[i] = decode8(codes[i], __uint_as_float(scales[i] << 23));
    }
  }
  e16_t* out = a.out[which] + ((size_t)t * a.Hk + head0) * D + 8 * c;
#pragma unroll
  for (int i = 0; i < UNIT; ++i)
    if (i < heads) *reinterpret_cast<ev8*>(out + i * D) = x[i];
}

}  // namespace

static int append(AppendArgs& a, const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                  const float* table, const int* pages, const int* lens, const int* cu, void* q_out, int B, int T, int max_pages,
                  int num_pages, int page_size, int H, int Hk, int D, int R, int P, int halves, int weight_f32, double eps,
                  long long q_stride, long long k_stride, long long v_stride, int bits, hipStream_t stream) {
  if (int st = rotate_check(q, k, q_weight, k_weight, table, T, H, Hk, D, R, P, eps)) return st;
  if (int st = places_check(pages, lens, cu, B, T, max_pages, num_pages, page_size, Hk)) return st;
  if (T == 0) return ES_OK;
  ES_REQUIRE(v && (H == 0 || q_out) && all_aligned16({v, q_out}), ES_ERR_INVALID,
             "append: v and q_out must be given and aligned to 16 bytes");
  ES_REQUIRE(stride_fits(q_stride, H, D, T) && stride_fits(k_stride, Hk, D, T) && stride_fits(v_stride, Hk, D, T), ES_ERR_INVALID,
             "append: row strides must be multiples of 8 that hold a row");
  a.x[0] = (const e16_t*)q, a.x[1] = (const e16_t*)k, a.x[2] = (const e16_t*)v;
  a.w[0] = q_weight, a.w[1] = k_weight;
  a.table = table;
  a.q_out = (e16_t*)q_out;
  a.places = make_places(pages, lens, cu, B, T, max_pages, num_pages, page_size);
  a.stride[0] = q_stride, a.stride[1] = k_stride, a.stride[2] = v_stride;
  a.heads[0] = H, a.heads[1] = a.heads[2] = Hk;
  for (int i = 0; i < 3; ++i) a.units[i] = bits == 4 && i == 1 ? Hk : (a.heads[i] + UNIT - 1) / UNIT;
  const int units = a.units[0] + a.units[1] + a.units[2];
  a.div_units = fast_div(units);
  a.T = T, a.Hk = Hk, a.R = R, a.P = P, a.f32 = weight_f32;
  a.eps = eps;
  const long long groups = 256 / (D / 16), blocks = ((long long)T * units + groups - 1) / groups;
  ES_REQUIRE((long long)T * units < (1LL << 30) && blocks < PAGED_GRID, ES_ERR_UNSUPPORTED, "append: too many rows");
  for_rotation(D, R, halves, q_weight || k_weight, [&](auto d, auto pairs, auto norm) {
    constexpr int dim = decltype(d)::value, p = decltype(pairs)::value;
    constexpr bool n = decltype(norm)::value;
    if (bits == 16) hipLaunchKernelGGL((append_kernel<dim, p, n, 16>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((append_kernel<dim, p, n, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  });
  return check_launch("es_append_paged");
}

static int paged_rows(RowsArgs& a, const int* pages, const int* lens, const int* cu, void* k, void* v, int B, int T, int max_pages,
                      int num_pages, int page_size, int Hk, int D, int bits, hipStream_t stream) {
  ES_REQUIRE(D == 64 || D == 128, ES_ERR_UNSUPPORTED, "paged rows: head dim must be 64 or 128");
  if (int st = places_check(pages, lens, cu, B, T, max_pages, num_pages, page_size, Hk)) return st;
  if (T == 0) return ES_OK;
  ES_REQUIRE(k && v && all_aligned16({k, v}), ES_ERR_INVALID, "paged rows: outputs must be given and aligned to 16 bytes");
  a.out[0] = (e16_t*)k, a.out[1] = (e16_t*)v;
  a.places = make_places(pages, lens, cu, B, T, max_pages, num_pages, page_size);
  a.T = T, a.Hk = Hk, a.units = (Hk + UNIT - 1) / UNIT;
  a.div_units = fast_div(2 * a.units);
  const long long groups = 256 / (D / 8), blocks = ((long long)T * 2 * a.units + groups - 1) / groups;
  ES_REQUIRE((long long)T * 2 * a.units < (1LL << 30) && blocks < PAGED_GRID, ES_ERR_UNSUPPORTED, "paged rows: too many rows");
  if (D == 64) {
    if (bits == 16) hipLaunchKernelGGL((rows_kernel<64, 16>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rows_kernel<64, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  } else {
    if (bits == 16) hipLaunchKernelGGL((rows_kernel<128, 16>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rows_kernel<128, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  }
  return check_launch("es_paged_rows");
}

}  // namespace es

using namespace es;

extern "C" int ES_VSA_API(es_append_paged)(const void* q, const void* k, const void* v, const void* q_weight,
                                           const void* k_weight, const float* table, const int* pages, const int* lens,
                                           const int* cu, void* q_out, void* k_pages, void* v_pages, int B, int T, int max_pages,
                                           int num_pages, int page_size, int H, int Hk, int D, int R, int P, int halves,
                                           int weight_f32, double eps, long long q_stride, long long k_stride,
                                           long long v_stride, long long page_stride, long long head_stride,
                                           long long row_stride, hipStream_t stream) {
  if (int st = cache_check(k_pages, v_pages, num_pages, page_size, Hk, D, page_stride, head_stride, row_stride)) return st;
  AppendArgs a = {};
  a.pages[0] = (e16_t*)k_pages, a.pages[1] = (e16_t*)v_pages;
  a.page_stride = page_stride, a.head_stride = head_stride, a.row_stride = row_stride;
  return append(a, q, k, v, q_weight, k_weight, table, pages, lens, cu, q_out, B, T, max_pages, num_pages, page_size, H, Hk, D, R,
                P, halves, weight_f32, eps, q_stride, k_stride, v_stride, 16, stream);
}

extern "C" int ES_VSA_API(es_append_paged4)(const void* q, const void* k, const void* v, const void* q_weight,
                                            const void* k_weight, const float* table, const int* pages, const int* lens,
                                            const int* cu, void* q_out, uint8_t* k_codes, uint8_t* k_scales, uint8_t* v_codes,
                                            uint8_t* v_scales, int B, int T, int max_pages, int num_pages, int page_size, int H,
                                            int Hk, int D, int R, int P, int halves, int weight_f32, double eps,
                                            long long q_stride, long long k_stride, long long v_stride, hipStream_t stream) {
  if (int st = cache4_check(k_codes, k_scales, v_codes, v_scales, num_pages)) return st;
  AppendArgs a = {};
  a.codes[0] = k_codes, a.codes[1] = v_codes;
  a.scales[0] = k_scales, a.scales[1] = v_scales;
  return append(a, q, k, v, q_weight, k_weight, table, pages, lens, cu, q_out, B, T, max_pages, num_pages, page_size, H, Hk, D, R,
                P, halves, weight_f32, eps, q_stride, k_stride, v_stride, 4, stream);
}

extern "C" int ES_VSA_API(es_paged_rows)(const void* k_pages, const void* v_pages, const int* pages, const int* lens,
                                         const int* cu, void* k, void* v, int B, int T, int max_pages, int num_pages,
                                         int page_size, int Hk, int D, long long page_stride, long long head_stride,
                                         long long row_stride, hipStream_t stream) {
  if (int st = cache_check(k_pages, v_pages, num_pages, page_size, Hk, D, page_stride, head_stride, row_stride)) return st;
  RowsArgs a = {};
  a.pages[0] = (const e16_t*)k_pages, a.pages[1] = (const e16_t*)v_pages;
  a.page_stride = page_stride, a.head_stride = head_stride, a.row_stride = row_stride;
  return paged_rows(a, pages, lens, cu, k, v, B, T, max_pages, num_pages, page_size, Hk, D, 16, stream);
}

extern "C" int ES_VSA_API(es_paged_rows4)(const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                                          const uint8_t* v_scales, const int* pages, const int* lens, const int* cu, void* k,
                                          void* v, int B, int T, int max_pages, int num_pages, int page_size, int Hk, int D,
                                          hipStream_t stream) {
  if (int st = cache4_check(k_codes, k_scales, v_codes, v_scales, num_pages)) return st;
  RowsArgs a = {};
  a.codes[0] = k_codes, a.codes[1] = v_codes;
  a.scales[0] = k_scales, a.scales[1] = v_scales;
  return paged_rows(a, pages, lens, cu, k, v, B, T, max_pages, num_pages, page_size, Hk, D, 4, stream);
}
