// Forward of attention over packed sequences and over a shared prefix (gfx950, bf16 / fp16): the kernels that give tiles
// (packed_tiles.h) their rows and keys, and when a call cuts its keys into ranges.
#include "packed_tiles.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace es {

namespace {

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
