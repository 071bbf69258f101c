// Sparse paged decode: one query token per row attends, per kv head, to the
// pages that a cheap score selects.
//
// The score reads int8 bounds of each page's keys instead of the keys
// (2 D + 4 bytes per page and kv head instead of 2 * page_size * D):
//   a = max |k|,  s = a / 127,  lo_d = floor(min_t k_td / s),  hi_d = ceil(max_t k_td / s)
// (clamped to +-127).  With the group's query heads quantised alike,
// qi = rint(q / sq), sq = max |q| / 127, the score of a page is
//   s * max_h sum_d max(qi_hd lo_d, qi_hd hi_d),
// up to sq and the quantisation an upper bound of every q.k of the page.
// The sums are integers below 2^24, so the score, hence the selection, does
// not depend on the order of summation.  The first `sink` and the last
// `recent` pages of a row are always taken; the others by falling score
// (ties: lower index) until `select` pages are taken.
//
// Two launches, both bound by what they read from HBM once there are enough
// CTAs, and by latency before that (a row of 5003 tokens: 4.6 us of score and
// 8.8 us of attention, which overlap to 10.7 us).  8 rows of 131072 tokens
// that take 256 of 8192 pages (32 / 8 heads of 128): score 134 MB in 30.5 us
// (4.4 TB/s), selection and attention 134 MB in 38 us (3.5 TB/s, a third of it
// the selection), where dense decode attention reads 4.3 GB.
#include "pl_common.cuh"

namespace pl {

// A page with an inf or NaN key: bounds 0, scale +inf; it scores +inf, so it
// is selected and shows in the output as it does in dense attention.
constexpr int kBoundsThreads = 128;

// ----------------------------------------------------------------- bounds
// One CTA per (page, kv heads); thread = 8 channels (16 bytes) of one head,
// so a token's heads are read side by side and a channel's extremes never
// leave their thread.  One pass over K: 16 loads of a thread are in flight
// and eight CTAs share an SM.  16384 pages of 16 tokens x 8 heads of 128: 98
// us for 571 MB, 5.8 TB/s (89 % of a plain copy's rate); 64 pages 3.6 us,
// which is one round trip to memory and the launch.
template <int D>
__global__ void __launch_bounds__(kBoundsThreads, 8)
    page_bounds_kernel(const bf16* __restrict__ kv, int64_t num_pages, int hkv, int page_size,
                       const int32_t* __restrict__ page_ids, const int32_t* __restrict__ page_len, int n,
                       int8_t* __restrict__ bounds, float* __restrict__ scale, int32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kLanes = D / 8;  // threads of one head: 8 or 16, inside one warp
  const int64_t unit = (int64_t)blockIdx.x * (kBoundsThreads / kLanes) + threadIdx.x / kLanes;
  const int u = threadIdx.x % kLanes;
  const bool live = unit < (int64_t)n * hkv;
  const int i = live ? (int)(unit / hkv) : 0, h = live ? (int)(unit % hkv) : 0;
  const int pg = page_ids[i];
  const bool ok = live && pg >= 0 && pg < num_pages;
  int len = page_size;
  if (page_len != nullptr && live) {
    len = page_len[i];
    if (len < 0 || len > page_size) {
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      len = len < 0 ? 0 : page_size;
    }
  }
  if (live && !ok && !(pg == -1 && len == 0)) set_status(status, PL_ERR_PAGE_OUT_OF_RANGE);
  float lo[8], hi[8];
  bool finite = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
  if (ok) {
    const uint4* src = reinterpret_cast<const uint4*>(kv + ((int64_t)pg * 2 * page_size * hkv + h) * D) + u;
    const int64_t step = (int64_t)hkv * D / 8;
#pragma unroll 16
    for (int t = 0; t < len; ++t) {
      const uint4 v = __ldg(src + t * step);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_bf16x2(w[e]);
        finite = finite && isfinite(f.x) && isfinite(f.y);
        lo[2 * e] = fminf(lo[2 * e], f.x);
        hi[2 * e] = fmaxf(hi[2 * e], f.x);
        lo[2 * e + 1] = fminf(lo[2 * e + 1], f.y);
        hi[2 * e + 1] = fmaxf(hi[2 * e + 1], f.y);
      }
    }
  }
  float a = 0.f;
  if (len > 0 && ok) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
  }
  if (!finite) a = INFINITY;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if (!ok) return;
  const float s = __fmul_rn(a, 1.0f / 127.0f);
  int8_t ql[8], qh[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool zero = !(s > 0.f) || isinf(s) || len == 0;
    ql[e] = zero ? 0 : (int8_t)fminf(fmaxf(floorf(__fdiv_rn(lo[e], s)), -127.f), 127.f);
    qh[e] = zero ? 0 : (int8_t)fminf(fmaxf(ceilf(__fdiv_rn(hi[e], s)), -127.f), 127.f);
  }
  int8_t* dst = bounds + ((int64_t)pg * hkv + h) * 2 * D + u * 8;
  *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(ql);
  *reinterpret_cast<uint2*>(dst + D) = *reinterpret_cast<const uint2*>(qh);
  if (u == 0) scale[(int64_t)pg * hkv + h] = s;
}

// ---------------------------------------------------------- sparse decode
// Two launches.  sparse_score_kernel streams the bounds of all pages and
// leaves an ordered key per (row, kv head, page).  sparse_attend_kernel
// selects and attends: the CTAs of one (row, kv head) form a cluster, each
// finds the selection for itself from the keys (a radix select in shared
// memory), takes its share of the pages, and the partial states meet through
// distributed shared memory.
constexpr int kSparseThreads = 256;
constexpr int kSparseWarps = kSparseThreads / 32;
constexpr int kScorePages = 16;          // pages a warp scores at a time
constexpr int kSparseUnit = 16;          // tokens a warp takes at a time
constexpr int kSparseMaxCluster = 8;
constexpr int kSparseBins = 2048;        // 11 bits of the key per pass
constexpr float kSparseSlack = 8.0f;     // log2 growth of a maximum that is tolerated before the state is rescaled

struct SparseArgs {
  const bf16* q;
  int64_t q_stride_b, q_stride_h;
  const bf16* kv;
  int64_t num_pages, total_pages;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_page_len;
  const int8_t* bounds;
  const float* scale;
  int32_t num_qo_heads, num_kv_heads, group, page_size, select, sink, recent;
  int32_t max_pages;     // no row has more
  int32_t key_stride;    // keys kept per (row, kv head), a multiple of 4
  int32_t splits;        // CTAs per (row, kv head) of the second launch
  float scale_log2;
  bf16* out;
  int64_t o_stride_b, o_stride_h;
  float* out_lse;
  int32_t* selected;     // [batch][hkv][select], ascending, -1 past the last
  uint32_t* keys;        // workspace [batch][hkv][key_stride]: competing pages
  int32_t* status;
};

__device__ __forceinline__ uint32_t order_key(float f) {  // ascending floats -> ascending unsigned
  const uint32_t u = __float_as_uint(f + 0.f);  // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sp_exp2(float x) {  // 2^x on the multi-function unit; x = -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct SparseRow {
  int begin, pages, last;
  __device__ __forceinline__ void load(const SparseArgs& a, int b) {
    begin = a.indptr[b];
    const int end = a.indptr[b + 1];
    const bool ok = begin >= 0 && end >= begin && end <= a.total_pages && end - begin <= a.max_pages;
    if (!ok && threadIdx.x == 0) set_status(a.status, PL_ERR_INVALID_ARGUMENT);
    pages = ok ? end - begin : 0;
    last = a.last_page_len[b];
    last = last < 0 ? 0 : (last > a.page_size ? a.page_size : last);
  }
};

// D(16x8, s32) += A(16x32, s8, row) . B(32x8, s8, col)
__device__ __forceinline__ void mma_s8_16832(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Keys of the pages of row b.  A warp has one kv head and 16 pages a step: a
// matrix product of the pages' bounds (rows) with the group's quantised
// queries (columns; per head min(qi, 0) against lo and max(qi, 0) against hi,
// 2 D bytes).  The product's order along 2 D is free, so a lane's operand is
// what it loads: 16 contiguous bytes of two pages per 64.  The warps of a CTA
// take neighbouring heads of the same pages, whose bounds lie side by side.
// NH: tiles of 8 heads.
//
// The s8 product does 2 D multiplications per page and head in 2 D / 32
// instructions of the warp for 16 pages, so what bounds the kernel is the
// bytes in flight: two steps of 4 KB per warp, 16 warps per SM.
template <int D, int NH>
__global__ void __launch_bounds__(kSparseThreads, 2) sparse_score_kernel(const SparseArgs a) {
  constexpr int kBytes = 2 * D;          // bounds of one page and head
  constexpr int kLd = kBytes / 64;       // 16-byte loads of a lane per page
  __shared__ __align__(16) int8_t qs_all[kSparseWarps][8 * NH][kBytes + 16];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z;
  SparseRow r;
  r.load(a, b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  // heads side by side, and groups of 16 pages when there are fewer heads than warps
  const int hw = min(kSparseWarps, a.num_kv_heads), pw = kSparseWarps / hw;
  const int kvh = (int)blockIdx.y * kSparseWarps + warp % hw;
  // pages that compete; forced ones have no key
  const int count = r.pages - a.recent - a.sink;
  const int step = gridDim.x * pw * kScorePages;
  int p = ((int)blockIdx.x * pw + warp / hw) * kScorePages;
  if (r.pages <= a.select || p >= count || warp >= hw * pw || kvh >= a.num_kv_heads) return;  // no block barrier below

  const int32_t* ids = a.indices + r.begin + a.sink;
  // lane pair (g, t): pages g (even t) and g + 8 (odd t) of a step
  auto page = [&](int at) { return at + g + 8 * (t & 1) < count ? ids[at + g + 8 * (t & 1)] : -1; };
  int pid = page(p);
  // quantise the group's queries: 8 channels a lane and step
  int8_t(*qs)[kBytes + 16] = qs_all[warp];
  constexpr int kMost = 8 * NH * D / 256;
  uint4 qv[kMost];
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int i = (k * 32 + lane) * 8;
    qv[k] = i < a.group * D ? *reinterpret_cast<const uint4*>(a.q + (int64_t)b * a.q_stride_b +
                                                              (int64_t)(kvh * a.group + i / D) * a.q_stride_h + i % D)
                            : make_uint4(0, 0, 0, 0);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&qv[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(w[e]);
      m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
  }
  m = warp_max(m);
  const float sq = __fmul_rn(m, 1.0f / 127.0f), div = sq > 0.f ? sq : 1.f;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int i = (k * 32 + lane) * 8;
    if (k * 256 >= a.group * D) {  // no head's
      *reinterpret_cast<uint2*>(&qs[i / D][i % D]) = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(&qs[i / D][D + i % D]) = make_uint2(0, 0);
      continue;
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&qv[k]);
    int8_t neg[8], pos[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 f = unpack_bf16x2(w[e / 2]);
      const float x = rintf(__fdiv_rn(e % 2 ? f.y : f.x, div));
      const int qi = isfinite(x) ? (int)fminf(fmaxf(x, -127.f), 127.f) : 0;
      neg[e] = (int8_t)min(qi, 0);
      pos[e] = (int8_t)max(qi, 0);
    }
    *reinterpret_cast<uint2*>(&qs[i / D][i % D]) = *reinterpret_cast<uint2*>(neg);
    *reinterpret_cast<uint2*>(&qs[i / D][D + i % D]) = *reinterpret_cast<uint2*>(pos);
  }
  __syncwarp();
  uint2 qb[NH][2 * kLd];  // column g of tile h: the 8 bytes that meet a lane's
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int j = 0; j < 2 * kLd; ++j)
      qb[h][j] = *reinterpret_cast<const uint2*>(&qs[8 * h + g][64 * (j >> 1) + 16 * t + 8 * (j & 1)]);
  uint32_t* keys = a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.key_stride;
  const int8_t* bounds = a.bounds + (int64_t)kvh * kBytes + 16 * t;
  const float* scale = a.scale + kvh;
  // bounds are loaded a step ahead, page ids two
  struct Step {
    uint4 w[2][kLd];
    float sc;  // of this lane's page, NaN: outside the pool
  };
  auto fetch = [&](Step& s, int at, int id) {
    const bool in = id >= 0 && (int64_t)id < a.num_pages;
    if (!in && at + g + 8 * (t & 1) < count && t < 2) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
    const int mine = in ? id : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pg = __shfl_sync(0xffffffffu, mine, (lane & ~3) + i);
      const uint4* src = reinterpret_cast<const uint4*>(bounds + (int64_t)pg * a.num_kv_heads * kBytes);
#pragma unroll
      for (int j = 0; j < kLd; ++j) s.w[i][j] = __ldg(src + 4 * j);
    }
    s.sc = in ? __ldg(scale + (int64_t)mine * a.num_kv_heads) : __int_as_float(0x7fffffff);
  };
  auto score = [&](const Step& s, int at) {
    int c[NH][4];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      c[h][0] = c[h][1] = c[h][2] = c[h][3] = 0;
#pragma unroll
      for (int j = 0; j < kLd; ++j) {
        const uint32_t lo[4] = {s.w[0][j].x, s.w[1][j].x, s.w[0][j].y, s.w[1][j].y};
        const uint32_t hi[4] = {s.w[0][j].z, s.w[1][j].z, s.w[0][j].w, s.w[1][j].w};
        mma_s8_16832(c[h], lo, qb[h][2 * j].x, qb[h][2 * j].y);
        mma_s8_16832(c[h], hi, qb[h][2 * j + 1].x, qb[h][2 * j + 1].y);
      }
    }
    // the maximum over the heads: columns 2 t, 2 t + 1 of pages g and g + 8
    int s0 = INT32_MIN, s1 = INT32_MIN;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (8 * h + 2 * t + i < a.group) {
          s0 = max(s0, c[h][i]);
          s1 = max(s1, c[h][2 + i]);
        }
    s0 = max(s0, __shfl_xor_sync(0xffffffffu, s0, 1));
    s1 = max(s1, __shfl_xor_sync(0xffffffffu, s1, 1));
    s0 = max(s0, __shfl_xor_sync(0xffffffffu, s0, 2));
    s1 = max(s1, __shfl_xor_sync(0xffffffffu, s1, 2));
    const int i = at + g + 8 * (t & 1);
    if (t < 2 && i < count) {
      const float best = (float)((t & 1) ? s1 : s0);
      const bool in = __float_as_int(s.sc) != 0x7fffffff;
      keys[i] = in ? order_key(isinf(s.sc) ? INFINITY : __fmul_rn(best, s.sc)) : 0u;
    }
  };
  Step s0, s1;
  fetch(s0, p, pid);
  pid = page(p + step);
  while (true) {
    if (p + step < count) fetch(s1, p + step, pid);
    pid = page(p + 2 * step);
    score(s0, p);
    p += step;
    if (p >= count) break;
    if (p + step < count) fetch(s0, p + step, pid);
    pid = page(p + 2 * step);
    score(s1, p);
    p += step;
    if (p >= count) break;
  }
}

template <int D>
struct SparseCfg {
  static constexpr int kHalves = D / 64;                       // 64-channel boxes of a tile
  static constexpr int kHalfBytes = kSparseUnit * 128;
  static constexpr int kTile = kHalves * kHalfBytes;           // K (or V) of one unit: 128B-swizzled boxes
  static constexpr int kOPad = D + 4;
  // Tiles (K, V, K, ...) of a warp in flight: with 3 two CTAs fit on an SM.
  static constexpr int kRing = 3;
  static constexpr int kStages = kSparseWarps * kRing * kTile;
  static constexpr int kScratch = kSparseWarps * 16 * kOPad * 4;
  static constexpr int kSelect = (kSparseBins + kSparseBins / 8) * 4;
  // the selection, the tiles in flight and the join of the warps' states use
  // the same bytes one after the other
  static constexpr int kArena = kStages > kScratch ? (kStages > kSelect ? kStages : kSelect)
                                                   : (kScratch > kSelect ? kScratch : kSelect);
  // what the cluster's CTAs send here: float4 chunks [i][CTA], and [CTA][2][16] m, l
  static constexpr int kRecvOff = kArena;
  static constexpr int kRecvMlOff = kRecvOff + (16 * D / 4 + kSparseMaxCluster) * 16;
  static constexpr int kMlOff = kRecvMlOff + kSparseMaxCluster * 32 * 4;  // [2][warps][16]
  static constexpr int kBarOff = kMlOff + 2 * kSparseWarps * 16 * 4;      // [warps][kRing]
  static constexpr int kListOff = kBarOff + kSparseWarps * kRing * 8;
};

// Block-wide exclusive prefix sum of one value per thread; total to all.
__device__ __forceinline__ int sparse_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSparseWarps; ++w) {
    const int u = warp_sums[w];
    before += w < warp ? u : 0;
    total += u;
  }
  return before + inc - v;
}

// Histogram bin b lives at b + b / 8: a thread reads 8 bins in a row
// without bank conflicts.
__device__ __forceinline__ int sparse_bin(int b) { return b + (b >> 3); }

// The selected pages with rank [lo, hi) in index order, into list[0 ..
// hi - lo); all of them to `all` when it is given.  keys: of the competing
// pages [sink, n - recent), 16-byte aligned; n > select.  They are dealt in
// quads of 4 neighbours, quad j of thread t at (j * threads + t) * 4.
// kQuads > 0: held in registers (quads <= kQuads); 0: read from L2 in every
// pass.
template <int kQuads>
__device__ __forceinline__ void sparse_select(const SparseArgs& a, const uint32_t* keys, int n, int* hist, int lo,
                                              int hi, int32_t* list, int32_t* all) {
  __shared__ int warp_sums[kSparseWarps];
  __shared__ uint32_t mm[2 * kSparseWarps];
  __shared__ int found[3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = a.sink, count = n - a.recent - a.sink, want = a.select - a.recent - a.sink;
  const int quads = (count + 4 * kSparseThreads - 1) / (4 * kSparseThreads);
  auto at = [&](int j) { return (j * kSparseThreads + (int)threadIdx.x) * 4; };
  auto quad = [&](int j) {
    return at(j) < count ? *reinterpret_cast<const uint4*>(keys + at(j)) : make_uint4(0, 0, 0, 0);
  };
  uint4 held[kQuads > 0 ? kQuads : 1];
  if constexpr (kQuads > 0) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
      if (j < quads) held[j] = quad(j);
  }
  // f(key, index) for the keys of quad j
  auto four = [&](int j, auto f) {
    uint4 q;
    if constexpr (kQuads > 0)
      q = held[j];
    else
      q = quad(j);
    const int i = at(j);
    if (i < count) f(q.x, i);
    if (i + 1 < count) f(q.y, i + 1);
    if (i + 2 < count) f(q.z, i + 2);
    if (i + 3 < count) f(q.w, i + 3);
  };
  // every(j) for the quads in use
  auto quads_of = [&](auto every) {
    if constexpr (kQuads > 0) {
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
        if (j < quads) every(j);
    } else {
#pragma unroll 1
      for (int j = 0; j < quads; ++j) every(j);
    }
  };
  auto each = [&](auto f) { quads_of([&](int j) { four(j, f); }); };
  uint32_t kmin = 0xffffffffu, kmax = 0;
  each([&](uint32_t k, int) {
    kmin = min(kmin, k);
    kmax = max(kmax, k);
  });
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) {
    mm[warp] = kmin;
    mm[kSparseWarps + warp] = kmax;
  }
  for (int i = threadIdx.x; i < kSparseBins + kSparseBins / 8; i += kSparseThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSparseWarps; ++w) {
    kmin = min(kmin, mm[w]);
    kmax = max(kmax, mm[kSparseWarps + w]);
  }
  // Digits from the highest bit in which the keys differ.  After a pass:
  // taken are the keys whose bits from `shift` on are above `prefix`, and
  // `rest` of those where they equal it.
  int shift = kmin == kmax ? 0 : 32 - __clz(kmin ^ kmax);  // bits below are undecided
  auto upper = [](uint32_t k, int s) { return __funnelshift_rc(k, 0u, s); };  // k >> s, 0 for s = 32
  uint32_t prefix = upper(kmax, shift);  // common to all keys
  int rest = want;
  while (shift > 0 && rest > 0) {
    const int bits = min(11, shift), low = shift - bits;
    each([&](uint32_t k, int) {
      if (upper(k, shift) == prefix) atomicAdd(&hist[sparse_bin((k >> low) & ((1u << bits) - 1))], 1);
    });
    __syncthreads();
    // from the top: the bin in which the count passes `rest`; thread 0 has the highest bins
    constexpr int kPer = kSparseBins / kSparseThreads;
    int h[kPer], sum = 0;
    const int top = (1 << bits) - 1 - threadIdx.x * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      h[j] = top - j >= 0 ? hist[sparse_bin(top - j)] : 0;
      sum += h[j];
    }
    int total;
    int before = sparse_scan(sum, warp_sums, total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (top - j >= 0) hist[sparse_bin(top - j)] = 0;  // for the next pass
      if (before < rest && before + h[j] >= rest) {
        found[0] = top - j;
        found[1] = rest - before;
        found[2] = h[j];
      }
      before += h[j];
    }
    __syncthreads();
    prefix = shift == 32 ? (uint32_t)found[0] : (prefix << bits) | (uint32_t)found[0];
    rest = found[1];
    shift = low;
    if (found[1] == found[2]) break;  // all keys of the bin are taken
  }
  // gather in index order, row of quads after row; counts above and at the
  // prefix in 16 bits each (a row has 4 * threads keys)
  auto bits_of = [&](int j) {  // bit e: key e of the quad is above the prefix; bit 4 + e: at it
    const int i = at(j);
    uint32_t m = 0;
    four(j, [&](uint32_t k, int at_k) {
      const uint32_t u = upper(k, shift);
      m |= (u > prefix ? 1u : u == prefix ? 0x10u : 0u) << (at_k - i);
    });
    return m;
  };
  auto count_of = [](uint32_t m) { return __popc(m & 0xfu) + (__popc(m & 0xf0u) << 16); };
  uint32_t bits[kQuads > 0 ? kQuads : 1];
  int own[kQuads > 0 ? kQuads : 1];  // this thread's count of the row, and the warp's up to it
  int inc[kQuads > 0 ? kQuads : 1];
  auto scan = [&](int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  auto put = [&](int rank, int page) {
    if (rank >= lo && rank < hi) list[rank - lo] = page;
    if (all != nullptr) all[rank] = page;
  };
  auto place = [&](int j, uint32_t m, int gt, int eq) {  // gt, eq: in front of this thread's quad
#pragma unroll 1
    for (uint32_t left = (m | m >> 4) & 0xfu; left != 0; left &= left - 1) {
      const int e = __ffs(left) - 1;
      const bool above = (m >> e) & 1u;
      if (above || eq < rest) put(first + gt + min(eq, rest), first + at(j) + e);
      gt += above ? 1 : 0;
      eq += above ? 0 : 1;
    }
  };
  if constexpr (kQuads > 0) {
    __shared__ int rows[kQuads][kSparseWarps];
    quads_of([&](int j) {
      bits[j] = bits_of(j);
      own[j] = count_of(bits[j]);
      inc[j] = scan(own[j]);
      if (lane == 31) rows[j][warp] = inc[j];
    });
    __syncthreads();
    int gt = 0, eq = 0;  // of the rows before
    quads_of([&](int j) {
      int g = 0, e = 0, ga = 0, ea = 0;
#pragma unroll
      for (int w = 0; w < kSparseWarps; ++w) {
        const int v = rows[j][w];
        g += w < warp ? v & 0xffff : 0;
        e += w < warp ? v >> 16 : 0;
        ga += v & 0xffff;
        ea += v >> 16;
      }
      const int before = inc[j] - own[j];
      if (own[j] != 0) place(j, bits[j], gt + g + (before & 0xffff), eq + e + (before >> 16));
      gt += ga;
      eq += ea;
    });
  } else {
    int gt = 0, eq = 0;
    quads_of([&](int j) {
      bits[0] = bits_of(j);
      int total;
      const int before = sparse_scan(count_of(bits[0]), warp_sums, total);
      if (bits[0] != 0) place(j, bits[0], gt + (before & 0xffff), eq + (before >> 16));
      gt += total & 0xffff;
      eq += total >> 16;
    });
  }
  for (int i = threadIdx.x; i < a.sink; i += kSparseThreads) put(i, i);
  for (int i = threadIdx.x; i < a.recent; i += kSparseThreads) put(a.select - a.recent + i, n - a.recent + i);
  __syncthreads();
}

// D(16x8) += A . B as mma_bf16_16816 with B given as two registers.
__device__ __forceinline__ void mma_bf16_b(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  const uint32_t b[2] = {b0, b1};
  mma_bf16_16816(d, a, b);
}
// Transpose of an 8x8 matrix of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// NH: tiles of 8 query heads (group <= 8 NH).  Tokens are the rows of the
// score product (16 x 8 heads = K . q^T) and channels those of the output
// (O^T = V^T . P), so a group of up to 8 heads wastes no rows; P goes from
// one to the other by an 8x8 transpose in registers.
template <int D, int NH>
__global__ void __launch_bounds__(kSparseThreads, 2) sparse_attend_kernel(const __grid_constant__ CUtensorMap kv_map,
                                                                           const SparseArgs a) {
  using C = SparseCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  float* wml = reinterpret_cast<float*>(smem + C::kMlOff);  // [2][warps][16]
  int32_t* list = reinterpret_cast<int32_t*>(smem + C::kListOff);
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int S = a.splits, PS = a.page_size, group = a.group;
  // q and the tables are read before the wait for the scores' grid, which
  // lets this one start only once they are complete (without that launch
  // this grid follows them directly and waits first)
  const bool scored = a.max_pages > a.select;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&kv_map);
    for (int i = 0; i < kSparseWarps * C::kRing; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  if (S > 1) cluster_arrive_relaxed();  // waited for before the first store into another CTA's memory
  if (!scored) pdl_wait();
  SparseRow r;
  r.load(a, b);
  const int taken = min(r.pages, a.select);
  const int lo = (int)((int64_t)taken * split / S), hi = (int)((int64_t)taken * (split + 1) / S);
  // q as the B operand: head g of tile h, channels 16 kk + 2 t4 (+ 8)
  uint32_t qb[NH][D / 16][2];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    const bool in = 8 * h + g < group;
    const bf16* src = a.q + (int64_t)b * a.q_stride_b + (int64_t)(kvh * group + (in ? 8 * h + g : 0)) * a.q_stride_h;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qb[h][kk][i] = in ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + 8 * i + 2 * t4) : 0u;
  }
  if (scored) pdl_wait();
  pdl_launch_dependents();
  int32_t* all = split == 0 ? a.selected + ((int64_t)b * a.num_kv_heads + kvh) * a.select : nullptr;
  if (r.pages > a.select) {
    const uint32_t* keys = a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.key_stride;
    int* hist = reinterpret_cast<int*>(smem);
    if (r.pages <= 4 * kSparseThreads)
      sparse_select<1>(a, keys, r.pages, hist, lo, hi, list, all);
    else if (r.pages <= 32 * kSparseThreads)
      sparse_select<8>(a, keys, r.pages, hist, lo, hi, list, all);
    else
      sparse_select<0>(a, keys, r.pages, hist, lo, hi, list, all);
  } else {
    if (all != nullptr)
      for (int i = threadIdx.x; i < a.select; i += kSparseThreads) all[i] = i < taken ? i : -1;
  }

  // the selection's use of the ring's bytes, before the copies'
  fence_proxy_async_smem();
  __syncthreads();

  // ---- a warp takes units of 16 tokens: K, V, K, V, ... through its own ring
  const int upp = PS / kSparseUnit;  // units of a page: 1 or 2
  const int ushift = upp == 2 ? 1 : 0;
  const int units = (hi - lo) * upp;
  uint8_t* ring = smem + warp * C::kRing * C::kTile;
  uint64_t* full = bars + warp * C::kRing;
  // page id of a unit (looked at when it is loaded), -1 past the last
  auto nth = [&](int i) { return r.pages <= a.select ? lo + i : list[i]; };  // taken page of the row
  auto page_of = [&](int u) { return u < units ? a.indices[r.begin + nth(u >> ushift)] : -1; };
  auto live_of = [&](int u) {  // its tokens
    if (u >= units) return 0;
    const int len = nth(u >> ushift) == r.pages - 1 ? r.last : PS;
    return min(kSparseUnit, max(0, len - (u & (upp - 1)) * kSparseUnit));
  };
  // Tile into a slot: 16-byte unit c of token t at (c / 8) * kHalfBytes +
  // t * 128 + (((c % 8) ^ (t % 8)) * 16).  One lane; the warp's reads of the
  // slot are over.
  auto load = [&](int slot, int u, int pg, int kv) {
    if (u >= units || lane != 0) return;
    const bool in = pg >= 0 && (int64_t)pg < a.num_pages;
    if (!in) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
    mbar_arrive_expect_tx(&full[slot], C::kTile);
    // out of range: the copy writes zeros
    const int32_t at = in ? 2 * pg + kv : (int32_t)(2 * a.num_pages);
#pragma unroll
    for (int h = 0; h < C::kHalves; ++h)
      tma_load_4d(ring + slot * C::kTile + h * C::kHalfBytes, &kv_map, h * 64, kvh, (u & (upp - 1)) * kSparseUnit, at,
                  &full[slot]);
  };
  float o[NH][D / 16][4];  // O^T: channels 16 j + g (+ 8), heads 8 h + 2 t4 (+ 1)
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[h][j][0] = o[h][j][1] = o[h][j][2] = o[h][j][3] = 0.f;
  float m[NH][2], l[NH][2];
#pragma unroll
  for (int h = 0; h < NH; ++h) m[h][0] = m[h][1] = -INFINITY, l[h][0] = l[h][1] = 0.f;
  const float sl2 = a.scale_log2;
  // unit u, then the two after it; tile n = 2 i + kv of the warp's i-th unit
  // in slot n % 3, phase (n / 3) & 1
  int pg = page_of(warp);
  int pg1 = page_of(warp + kSparseWarps);
  load(0, warp, pg, 0);
  load(1, warp, pg, 1);
  load(2, warp + kSparseWarps, pg1, 0);
  int n = 0;
  bool ok = true;
  for (int u = warp; u < units; u += kSparseWarps, n += 2) {
    const int un = u + kSparseWarps, unn = un + kSparseWarps;
    const int pg2 = page_of(unn), live = live_of(u);
    const int kslot = n % C::kRing, vslot = (n + 1) % C::kRing;
    const uint32_t kt = smem_u32(ring) + kslot * C::kTile, vt = smem_u32(ring) + vslot * C::kTile;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[kslot], (n / C::kRing) & 1));  // K of this unit
    if (!ok) break;
    // ---- scores: tokens g, g + 8 x heads 2 t4, 2 t4 + 1; two chains of products
    float sc[NH][4];
    {
      float s1[NH][4];
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[h][i] = s1[h][i] = 0.f;
      const int tok = (lane & 7) + 8 * ((lane >> 3) & 1), c0 = lane >> 4;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t ka[4];
        const int c = 2 * kk + c0;
        ldsm_x4(kt + (kk / 4) * C::kHalfBytes + tok * 128 + (((c & 7) ^ (tok & 7)) << 4), ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
        for (int h = 0; h < NH; ++h) mma_bf16_b(kk % 2 ? s1[h] : sc[h], ka, qb[h][kk][0], qb[h][kk][1]);
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[h][i] += s1[h][i];
    }
    __syncwarp();
    load(kslot, un, pg1, 1);  // the next V into this K's place
    // ---- online softmax (log2 domain), a column per head
    uint32_t ph[NH][2], pr[NH][2];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const bool in0 = g < live, in1 = g + 8 < live;
      sc[h][0] = in0 ? sc[h][0] * sl2 : -INFINITY;
      sc[h][1] = in0 ? sc[h][1] * sl2 : -INFINITY;
      sc[h][2] = in1 ? sc[h][2] * sl2 : -INFINITY;
      sc[h][3] = in1 ? sc[h][3] * sl2 : -INFINITY;
      // against the running maximum, unless a score exceeds it by 2^8 (or it
      // is the first): then the maximum moves and the state is rescaled
      if (__any_sync(0xffffffffu, fmaxf(sc[h][0], sc[h][2]) > m[h][0] + kSparseSlack ||
                                      fmaxf(sc[h][1], sc[h][3]) > m[h][1] + kSparseSlack)) {
        float al[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(sc[h][i], sc[h][2 + i]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[h][i], mx);
          al[i] = m[h][i] == mn ? 1.f : sp_exp2(m[h][i] - mn);  // m = -inf: 0 times a state of zeros
          m[h][i] = mn;
          l[h][i] *= al[i];
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[h][j][0] *= al[0];
          o[h][j][1] *= al[1];
          o[h][j][2] *= al[0];
          o[h][j][3] *= al[1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float base = m[h][i] == -INFINITY ? 0.f : m[h][i];
        sc[h][i] = sp_exp2(sc[h][i] - base);
        sc[h][2 + i] = sp_exp2(sc[h][2 + i] - base);
        l[h][i] += sc[h][i] + sc[h][2 + i];
      }
      // P as a bf16 pair (value and remainder): O keeps fp32's accuracy, for
      // products that this memory-bound loop has to spare
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // tokens g, g + 8
        const uint32_t hi2 = pack_bf16x2(sc[h][2 * i], sc[h][2 * i + 1]);
        const float2 f = unpack_bf16x2(hi2);
        ph[h][i] = transpose_8x8(hi2);
        pr[h][i] = transpose_8x8(pack_bf16x2(sc[h][2 * i] - f.x, sc[h][2 * i + 1] - f.y));
      }
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&full[vslot], ((n + 1) / C::kRing) & 1));  // V of this unit
    if (!ok) {
      n += 1;  // the next V is under way instead of this K
      break;
    }
    if (live < kSparseUnit) {
      // rows past the last token hold whatever the pool had there, and 0 * NaN is NaN
      for (int idx = lane; idx < (kSparseUnit - live) * C::kHalves * 8; idx += 32) {
        const int t = live + idx / (C::kHalves * 8), hh = (idx / 8) % C::kHalves, c = idx % 8;
        *reinterpret_cast<uint4*>(ring + vslot * C::kTile + hh * C::kHalfBytes + t * 128 + c * 16) =
            make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
    }
    {
      // A = V^T: rows = channels; lanes 8 i .. 8 i + 7 name the token rows of matrix i
      const int tok = (lane & 7) + 8 * (lane >> 4), c0 = (lane >> 3) & 1;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t va[4];
        const int c = 2 * j + c0;
        ldsm_x4_trans(vt + (j / 4) * C::kHalfBytes + tok * 128 + (((c & 7) ^ (tok & 7)) << 4), va[0], va[1], va[2],
                      va[3]);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          mma_bf16_b(o[h][j], va, ph[h][0], ph[h][1]);
          mma_bf16_b(o[h][j], va, pr[h][0], pr[h][1]);
        }
      }
    }
    __syncwarp();
    load(vslot, unn, pg2, 0);  // the K after the next into this V's place
    pg1 = pg2;
  }
  if (!ok) {
    // give up: the copies under way (tiles n .. n + 2, as far as they exist) land first
    if (lane == 0) set_status(a.status, PL_ERR_TIMEOUT);
    const int tiles = 2 * ((units - warp + kSparseWarps - 1) / kSparseWarps);
    for (int i = n; i < min(n + 3, tiles); ++i) (void)mbar_wait(&full[i % C::kRing], (i / C::kRing) & 1);
  }

  // ---- the warps' states meet in shared memory
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[h][i] += __shfl_xor_sync(0xffffffffu, l[h][i], d);
  __syncthreads();  // every warp is done with its buffer
  float* ow = reinterpret_cast<float*>(smem) + warp * 16 * C::kOPad;
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int head = 8 * h + 2 * t4 + i;
      if (head < group)
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          ow[head * C::kOPad + 16 * j + g] = o[h][j][i];
          ow[head * C::kOPad + 16 * j + 8 + g] = o[h][j][2 + i];
        }
      if (g == 0) {
        wml[warp * 16 + head] = m[h][i];
        wml[(kSparseWarps + warp) * 16 + head] = l[h][i];
      }
    }
  __syncthreads();
  auto write = [&](int row, int d, float4 acc, float L, float M) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int head = kvh * group + row;
    bf16* dst = a.out + (int64_t)b * a.o_stride_b + (int64_t)head * a.o_stride_h + d;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    if (d == 0 && a.out_lse != nullptr)
      a.out_lse[(int64_t)b * a.num_qo_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  };
  if (S > 1) cluster_wait();  // every CTA of the cluster runs
  for (int idx = threadIdx.x; idx < group * (D / 4); idx += kSparseThreads) {
    const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSparseWarps; ++w) M = fmaxf(M, wml[w * 16 + row]);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSparseWarps; ++w) {
      const float mw = wml[w * 16 + row];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem) + (w * 16 + row) * C::kOPad + d);
      L += f * wml[(kSparseWarps + w) * 16 + row];
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    if (S == 1) {
      write(row, d, acc, L, M);
    } else {
      // chunk idx is added up by CTA idx % S of the cluster
      const uint32_t at = smem_u32(smem + C::kRecvOff) + ((idx / S) * S + split) * 16;
      dsmem_st_f32x4(dsmem_map(at, idx % S), acc);
      if (d == 0) {
        const uint32_t ml = smem_u32(smem + C::kRecvMlOff) + (split * 32 + row) * 4;
        for (int c = 0; c < S; ++c) {
          dsmem_st_f32(dsmem_map(ml, c), M);
          dsmem_st_f32(dsmem_map(ml + 64, c), L);
        }
      }
    }
  }
  if (S == 1) return;
  cluster_sync_all();  // every CTA's state has arrived; nothing is read remotely after it
  const float4* recv = reinterpret_cast<const float4*>(smem + C::kRecvOff);
  const float* recv_ml = reinterpret_cast<const float*>(smem + C::kRecvMlOff);
  for (int i = threadIdx.x; i * S + split < group * (D / 4); i += kSparseThreads) {
    const int idx = i * S + split;
    const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
    float M = -INFINITY;
    for (int c = 0; c < S; ++c) M = fmaxf(M, recv_ml[c * 32 + row]);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < S; ++c) {
      // without a maximum: a CTA without pages, whose state is 0, or NaN scores,
      // whose sum is NaN
      const float mc = recv_ml[c * 32 + row];
      const float f = mc == -INFINITY ? 1.f : exp2f(mc - M);
      const float4 v = recv[i * S + c];
      L += f * recv_ml[c * 32 + 16 + row];
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    write(row, d, acc, L, M);
  }
}

}  // namespace pl

// =================================================================== host
namespace {

constexpr int kScoreSteps = 4;  // steps of a warp when rows differ in length

int32_t sparse_key_stride(int32_t max_pages) { return (int32_t)(((int64_t)max_pages + 3) & ~int64_t(3)); }

constexpr int kSparseMostListed = 24576;  // selected pages of a row, kept in shared memory

template <int D, int NH>
int32_t launch_attend_nh(const CUtensorMap& map, const pl::SparseArgs& a, int batch, void* stream) {
  auto kern = pl::sparse_attend_kernel<D, NH>;
  // rows that take all their pages need no list
  const int list = a.select < a.max_pages ? 4 * (a.select / a.splits + 2) : 0;
  static_assert(1024 + pl::SparseCfg<D>::kListOff + 4 * (kSparseMostListed + 2) + 16 <= 232448, "the list must fit");
  const int smem = 1024 + pl::SparseCfg<D>::kListOff + ((list + 15) & ~15);
  int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  if (st != PL_OK) return st;
  const dim3 grid(a.splits, a.num_kv_heads, batch);
  if (a.splits == 1) return pl_host::launch_pdl(kern, grid, dim3(pl::kSparseThreads), smem, stream, map, a);
  return pl_host::launch_pdl_cluster(kern, grid, dim3(pl::kSparseThreads), smem, stream, a.splits, map, a);
}

template <int D>
int32_t launch_attend(const CUtensorMap& map, const pl::SparseArgs& a, int batch, void* stream) {
  return a.group <= 8 ? launch_attend_nh<D, 1>(map, a, batch, stream) : launch_attend_nh<D, 2>(map, a, batch, stream);
}

}  // namespace

extern "C" int32_t pl_page_bounds(const void* kv_cache, int64_t num_pages, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t page_size, const int32_t* page_ids, const int32_t* page_len, int32_t n,
                                  int8_t* bounds, float* bound_scale, int32_t* status_dev, void* stream) {
  if (kv_cache == nullptr || bounds == nullptr || bound_scale == nullptr || num_pages <= 0 || num_kv_heads <= 0 ||
      page_size <= 0 || n < 0 || (page_ids == nullptr && n > 0) || (reinterpret_cast<uintptr_t>(kv_cache) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(bounds) & 15) != 0)
    return PL_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return PL_ERR_UNSUPPORTED;
  if (n == 0) return PL_OK;
  const int64_t per = pl::kBoundsThreads / (head_dim / 8);
  const int64_t grid = ((int64_t)n * num_kv_heads + per - 1) / per;
  if (grid > 0x7FFFFFFF) return PL_ERR_INVALID_ARGUMENT;
  auto kern = head_dim == 128 ? pl::page_bounds_kernel<128> : pl::page_bounds_kernel<64>;
  return pl_host::launch_pdl(kern, dim3((int)grid), dim3(pl::kBoundsThreads), 0, stream,
                             static_cast<const pl::bf16*>(kv_cache), num_pages, (int)num_kv_heads, (int)page_size,
                             page_ids, page_len, (int)n, bounds, bound_scale, status_dev);
}

extern "C" int64_t pl_sparse_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t max_pages) {
  if (batch <= 0 || num_kv_heads <= 0 || max_pages <= 0) return 0;
  return (int64_t)batch * num_kv_heads * sparse_key_stride(max_pages) * 4;
}

extern "C" int32_t pl_paged_sparse_decode(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv_cache, int64_t num_pages,
    const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len, int64_t total_pages,
    int32_t max_pages, const int8_t* bounds, const float* bound_scale, int32_t batch, int32_t num_qo_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float sm_scale, int32_t num_select,
    int32_t sink_pages, int32_t recent_pages, void* out, int64_t o_stride_b, int64_t o_stride_h, float* out_lse,
    int32_t* selected, void* workspace, int64_t workspace_bytes, int32_t* status_dev, void* stream) {
  // what has no entries may be null
  if (kv_cache == nullptr || indptr == nullptr || (total_pages > 0 && indices == nullptr) || bounds == nullptr ||
      bound_scale == nullptr || batch < 0 ||
      (batch > 0 && (q == nullptr || last_page_len == nullptr || out == nullptr || selected == nullptr)) ||
      num_pages <= 0 || num_pages > 0x3FFFFFFF || total_pages < 0 || max_pages < 0 || max_pages > 0x7FFFFFF0 || num_kv_heads <= 0 ||
      num_qo_heads <= 0 || num_qo_heads % num_kv_heads != 0 || !(sm_scale > 0.f) || sink_pages < 0 || recent_pages < 1 || num_select < 1 ||
      (int64_t)sink_pages + recent_pages > num_select)
    return PL_ERR_INVALID_ARGUMENT;
  const int group = num_qo_heads / num_kv_heads;
  if ((head_dim != 64 && head_dim != 128) || (page_size != 16 && page_size != 32) || group > 16 ||
      num_kv_heads > 65535 || batch > 65535)
    return PL_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(kv_cache) & 15) != 0 || (reinterpret_cast<uintptr_t>(bounds) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0 ||
      (q_stride_b % 8) != 0 || (q_stride_h % 8) != 0 || (o_stride_b % 8) != 0 || (o_stride_h % 8) != 0)
    return PL_ERR_INVALID_ARGUMENT;
  if (max_pages > num_select && num_select > kSparseMostListed) return PL_ERR_UNSUPPORTED;
  if (batch == 0) return PL_OK;
  if (max_pages > num_select &&
      (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
       workspace_bytes < pl_sparse_workspace_bytes(batch, num_kv_heads, max_pages)))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  pl::SparseArgs a;
  a.q = static_cast<const pl::bf16*>(q);
  a.q_stride_b = q_stride_b;
  a.q_stride_h = q_stride_h;
  a.kv = static_cast<const pl::bf16*>(kv_cache);
  a.num_pages = num_pages;
  a.total_pages = total_pages;
  a.indptr = indptr;
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.bounds = bounds;
  a.scale = bound_scale;
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.page_size = page_size;
  a.select = num_select;
  a.sink = sink_pages;
  a.recent = recent_pages;
  a.max_pages = max_pages;
  a.key_stride = sparse_key_stride(max_pages);
  a.scale_log2 = sm_scale * pl::kLog2e;
  a.out = static_cast<pl::bf16*>(out);
  a.o_stride_b = o_stride_b;
  a.o_stride_h = o_stride_h;
  a.out_lse = out_lse;
  a.selected = selected;
  a.keys = static_cast<uint32_t*>(workspace);
  a.status = status_dev;
  const int sms = pl_host::sm_count();
  if (sms <= 0) return PL_ERR_NO_DEVICE;
  const int64_t items = (int64_t)batch * num_kv_heads;
  CUtensorMap map;
  int32_t st = pl_host::kv_tensor_map_rows(kv_cache, num_pages, num_kv_heads, head_dim, page_size, pl::kSparseUnit, &map);
  if (st != PL_OK) return st;
  if (max_pages > num_select) {
    // as many CTAs as the device holds at once, but no more than there are steps
    const int hw = num_kv_heads < pl::kSparseWarps ? num_kv_heads : pl::kSparseWarps, pw = pl::kSparseWarps / hw;
    const int head_groups = (num_kv_heads + pl::kSparseWarps - 1) / pl::kSparseWarps;
    const int64_t steps = ((int64_t)max_pages + pl::kScorePages * pw - 1) / (pl::kScorePages * pw);
    int64_t chunks = 2 * (int64_t)sms / ((int64_t)batch * head_groups);
    // Rows of unequal length: short pieces, so that the device stays full
    // while the longest is read (24 rows of 500 to 40000 tokens 59.6 -> 51.7
    // us); with rows of equal length every piece would pay for the queries'
    // quantisation again (8 rows of 131072 tokens 72 -> 79 us).
    if (8 * total_pages < 7 * (int64_t)batch * max_pages && chunks < (steps + kScoreSteps - 1) / kScoreSteps)
      chunks = (steps + kScoreSteps - 1) / kScoreSteps;
    chunks = chunks > steps ? steps : (chunks < 1 ? 1 : chunks);
    auto score = head_dim == 128 ? (group <= 8 ? pl::sparse_score_kernel<128, 1> : pl::sparse_score_kernel<128, 2>)
                                 : (group <= 8 ? pl::sparse_score_kernel<64, 1> : pl::sparse_score_kernel<64, 2>);
    st = pl_host::launch_pdl(score, dim3((int)chunks, head_groups, batch), dim3(pl::kSparseThreads), 0, stream, a);
    if (st != PL_OK) return st;
  }
  // CTAs per (row, kv head): two fit on an SM, all at once, and a warp should
  // have a unit.  64 items (8 rows of 131072 tokens, 256 pages each) take 95 us
  // with 2, 72 with 4 and 93 with 8, which no longer all run at once; 192
  // items take 51 us with 1 and 58 with 2.
  const int64_t units = (int64_t)(num_select < max_pages ? num_select : max_pages) * (page_size / pl::kSparseUnit);
  int splits = 1;
  while (splits < pl::kSparseMaxCluster && items * splits * 2 <= 2 * sms && units >= (int64_t)splits * pl::kSparseWarps)
    splits *= 2;
  a.splits = splits;
  return head_dim == 128 ? launch_attend<128>(map, a, batch, stream) : launch_attend<64>(map, a, batch, stream);
}
