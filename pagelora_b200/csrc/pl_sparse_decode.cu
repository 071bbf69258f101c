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
#include "pl_common.cuh"

namespace pl {

// A page with an inf or NaN key: bounds 0, scale +inf; it scores +inf, so it
// is selected and shows in the output as it does in dense attention.
constexpr int kBoundsThreads = 128;

// ----------------------------------------------------------------- bounds
// One CTA per (page, kv heads); thread = 8 channels (16 bytes) of one head.
template <int D>
__global__ void __launch_bounds__(kBoundsThreads)
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
  if (live && !ok) set_status(status, PL_ERR_PAGE_OUT_OF_RANGE);
  int len = page_size;
  if (page_len != nullptr && live) {
    len = page_len[i];
    if (len < 0 || len > page_size) {
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      len = len < 0 ? 0 : page_size;
    }
  }
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
#pragma unroll 8
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
constexpr int kSparseUnit = 16;          // tokens a warp takes at a time
constexpr int kSparseMaxCluster = 8;
constexpr int kSparseKeys = 8192;        // keys held in shared memory; longer rows read them from L2 in every pass
constexpr int kSparseBins = 2048;        // 11 bits of the key per pass

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
  int32_t max_pages;     // keys kept per (row, kv head)
  int32_t splits;        // CTAs per (row, kv head) of the second launch
  float scale_log2;
  bf16* out;
  int64_t o_stride_b, o_stride_h;
  float* out_lse;
  int32_t* selected;     // [batch][hkv][select], ascending, -1 past the last
  uint32_t* keys;        // workspace [batch][hkv][max_pages]
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

// Keys of the pages of (row b, kv head): a matrix product of the group's
// quantised queries (rows; per head min(qi, 0) against lo and max(qi, 0)
// against hi, 2 D bytes) with the bounds of 8 pages a warp and step.  The
// product's order along 2 D is free, so a lane's operand is what it loads:
// 16 contiguous bytes of its page per 64.
template <int D>
__global__ void __launch_bounds__(kSparseThreads) sparse_score_kernel(const SparseArgs a) {
  constexpr int kBytes = 2 * D;          // bounds of one page and head
  constexpr int kLd = kBytes / 64;       // 16-byte loads of a lane per page
  __shared__ __align__(16) int8_t qs[16][kBytes + 16];
  __shared__ float red[kSparseWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int kvh = blockIdx.y, b = blockIdx.z;
  SparseRow r;
  r.load(a, b);
  // pages that compete; forced ones have no key
  const int p_end = r.pages - a.recent;
  const int step = gridDim.x * kSparseWarps * 8;
  if (r.pages <= a.select || a.sink + (int)blockIdx.x * kSparseWarps * 8 >= p_end) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  int p = a.sink + ((int)blockIdx.x * kSparseWarps + warp) * 8;
  int pid = p + g < p_end ? a.indices[r.begin + p + g] : -1;

  // quantise the group's queries; a thread keeps its elements in registers
  constexpr int kMost = 16 * D / kSparseThreads;
  float v[kMost], m = 0.f;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int i = threadIdx.x + k * kSparseThreads;
    v[k] = i < a.group * D
               ? bf2f(a.q[(int64_t)b * a.q_stride_b + (int64_t)(kvh * a.group + i / D) * a.q_stride_h + i % D])
               : 0.f;
    m = fmaxf(m, fabsf(v[k]));
  }
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSparseWarps; ++w) m = fmaxf(m, red[w]);
  const float sq = __fmul_rn(m, 1.0f / 127.0f);
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int i = threadIdx.x + k * kSparseThreads;
    const float x = rintf(__fdiv_rn(v[k], sq > 0.f ? sq : 1.f));
    const int qi = isfinite(x) ? (int)fminf(fmaxf(x, -127.f), 127.f) : 0;
    qs[i / D][i % D] = (int8_t)min(qi, 0);
    qs[i / D][D + i % D] = (int8_t)max(qi, 0);
  }
  __syncthreads();
  uint32_t qa[2 * kLd][4];
#pragma unroll
  for (int j = 0; j < kLd; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = 64 * j + 16 * t + 8 * h;
      const uint2 lo = *reinterpret_cast<const uint2*>(&qs[g][at]);
      const uint2 hi = *reinterpret_cast<const uint2*>(&qs[g + 8][at]);
      qa[2 * j + h][0] = lo.x;
      qa[2 * j + h][1] = hi.x;
      qa[2 * j + h][2] = lo.y;
      qa[2 * j + h][3] = hi.y;
    }
  uint32_t* keys = a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.max_pages;
  for (; p < p_end; p += step) {
    const bool in = pid >= 0 && (int64_t)pid < a.num_pages;
    if (!in && p + g < p_end && t == 0) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
    const int64_t slot = (int64_t)(in ? pid : 0) * a.num_kv_heads + kvh;
    const uint4* src = reinterpret_cast<const uint4*>(a.bounds + slot * kBytes) + t;
    uint4 w[kLd];
#pragma unroll
    for (int j = 0; j < kLd; ++j) w[j] = in ? __ldg(src + 4 * j) : make_uint4(0, 0, 0, 0);
    const float sc = in ? __ldg(a.scale + slot) : 0.f;
    pid = p + step + g < p_end ? a.indices[r.begin + p + step + g] : -1;
    int c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      mma_s8_16832(c, qa[2 * j], w[j].x, w[j].y);
      mma_s8_16832(c, qa[2 * j + 1], w[j].z, w[j].w);
    }
    // rows g and g + 8 of pages 2 t and 2 t + 1: the maximum over the heads
    int s0 = max(g < a.group ? c[0] : INT32_MIN, g + 8 < a.group ? c[2] : INT32_MIN);
    int s1 = max(g < a.group ? c[1] : INT32_MIN, g + 8 < a.group ? c[3] : INT32_MIN);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      s0 = max(s0, __shfl_xor_sync(0xffffffffu, s0, o));
      s1 = max(s1, __shfl_xor_sync(0xffffffffu, s1, o));
    }
    // lane 4 g holds page g's scale; its score sits with t = g / 2
    const int from = g >> 1;
    const int e0 = __shfl_sync(0xffffffffu, s0, from), e1 = __shfl_sync(0xffffffffu, s1, from);
    if (t == 0 && p + g < p_end) {
      const int best = (g & 1) ? e1 : e0;
      keys[p + g] = in ? order_key(isinf(sc) ? INFINITY : __fmul_rn((float)best, sc)) : 0u;
    }
  }
}

template <int D>
struct SparseCfg {
  static constexpr int kRow = 2 * D;                           // bytes of one token's K (or V)
  static constexpr int kTile = kSparseUnit * kRow;             // K (or V) of one unit
  static constexpr int kQRow = 2 * D + 16;                     // padded: conflict-free ldmatrix
  static constexpr int kOPad = D + 4;
  static constexpr int kStages = kSparseWarps * 2 * kTile;     // a warp's unit: K, V
  static constexpr int kScratch = kSparseWarps * 16 * kOPad * 4;
  static constexpr int kSelect = (kSparseKeys + kSparseBins) * 4;
  // the selection, the units in flight and the join of the warps' states use
  // the same bytes one after the other
  static constexpr int kArena = kStages > kScratch ? (kStages > kSelect ? kStages : kSelect)
                                                   : (kScratch > kSelect ? kScratch : kSelect);
  static constexpr int kQOff = kArena;
  static constexpr int kPartOff = kQOff + 16 * kQRow;          // [16][D] fp32: this CTA's state for the cluster
  static constexpr int kMlOff = kPartOff + 16 * D * 4;         // [2][16] of the CTA, then [2][warps][16]
  static constexpr int kListOff = kMlOff + (2 + 2 * kSparseWarps) * 16 * 4;
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

// The selected pages with rank [lo, hi) in index order, into list[0 ..
// hi - lo); all of them to `all` when it is given.  keys[p] for the pages
// [sink, n - recent); n > select.
__device__ __forceinline__ void sparse_select(const SparseArgs& a, const uint32_t* keys, int n, uint8_t* arena, int lo,
                                              int hi, int32_t* list, int32_t* all) {
  __shared__ int warp_sums[kSparseWarps];
  __shared__ uint32_t mm[2 * kSparseWarps];
  __shared__ int found[3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = a.sink, count = n - a.recent - a.sink, want = a.select - a.recent - a.sink;
  uint32_t* held = reinterpret_cast<uint32_t*>(arena);
  int* hist = reinterpret_cast<int*>(arena + kSparseKeys * 4);
  const bool hold = count <= kSparseKeys;
  uint32_t kmin = 0xffffffffu, kmax = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += kSparseThreads) {
    const uint32_t k = __ldcg(keys + first + i);
    if (hold) held[i] = k;
    kmin = min(kmin, k);
    kmax = max(kmax, k);
  }
  auto key = [&](int i) { return hold ? held[i] : __ldcg(keys + first + i); };
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) {
    mm[warp] = kmin;
    mm[kSparseWarps + warp] = kmax;
  }
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
  uint32_t prefix = shift < 32 ? kmax >> shift : 0u;       // common to all keys
  int rest = want;
  while (shift > 0 && rest > 0) {
    const int bits = min(11, shift), low = shift - bits;
    for (int i = threadIdx.x; i < (1 << bits); i += kSparseThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kSparseThreads) {
      const uint32_t k = key(i);
      if (shift == 32 || (k >> shift) == prefix) atomicAdd(&hist[(k >> low) & ((1u << bits) - 1)], 1);
    }
    __syncthreads();
    // from the top: the bin in which the count passes `rest`; thread 0 has the highest bins
    constexpr int kPer = kSparseBins / kSparseThreads;
    int h[kPer], sum = 0;
    const int top = (1 << bits) - 1 - threadIdx.x * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      h[j] = top - j >= 0 ? hist[top - j] : 0;
      sum += h[j];
    }
    int total;
    int before = sparse_scan(sum, warp_sums, total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
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
    const bool exact = found[1] == found[2];
    __syncthreads();
    if (exact) break;  // all keys of the bin are taken
  }
  // Gather in index order: a warp has a contiguous range.
  const int per = (count + kSparseWarps * 32 - 1) / (kSparseWarps * 32) * 32;
  const int i0 = min(count, warp * per), i1 = min(count, i0 + per);
  int n_gt = 0, n_eq = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t k = key(i);
    const uint32_t top = shift == 32 ? 0u : k >> shift;
    n_gt += top > prefix;
    n_eq += top == prefix;
  }
  n_gt = __reduce_add_sync(0xffffffffu, n_gt);
  n_eq = __reduce_add_sync(0xffffffffu, n_eq);
  if (lane == 0) {
    mm[warp] = n_gt;
    mm[kSparseWarps + warp] = n_eq;
  }
  __syncthreads();
  int gt = 0, eq = 0;
  for (int w = 0; w < warp; ++w) {
    gt += mm[w];
    eq += mm[kSparseWarps + w];
  }
  auto put = [&](int rank, int page) {
    if (rank >= lo && rank < hi) list[rank - lo] = page;
    if (all != nullptr) all[rank] = page;
  };
  for (int i = i0; i < i1; i += 32) {
    const uint32_t k = i + lane < i1 ? key(i + lane) : 0u;
    const uint32_t top = shift == 32 ? 0u : k >> shift;
    const bool is_gt = i + lane < i1 && top > prefix, is_eq = i + lane < i1 && top == prefix;
    const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
    const uint32_t below = (1u << lane) - 1;
    const int my_eq = eq + __popc(be & below);
    if (is_gt || (is_eq && my_eq < rest))
      put(first + gt + __popc(bg & below) + min(my_eq, rest), first + i + lane);
    gt += __popc(bg);
    eq += __popc(be);
  }
  for (int i = threadIdx.x; i < a.sink; i += kSparseThreads) put(i, i);
  for (int i = threadIdx.x; i < a.recent; i += kSparseThreads) put(a.select - a.recent + i, n - a.recent + i);
  __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(kSparseThreads, 2) sparse_attend_kernel(const SparseArgs a) {
  using C = SparseCfg<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem + C::kPartOff);
  float* cml = reinterpret_cast<float*>(smem + C::kMlOff);  // [2][16]: the CTA's m, l
  float* wml = cml + 32;                                    // [2][warps][16]
  int32_t* list = reinterpret_cast<int32_t*>(smem + C::kListOff);
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = a.splits, PS = a.page_size, group = a.group;
  // q and the tables are read before the wait for the scores' grid, which
  // lets this one start only once they are complete (without that launch
  // this grid follows them directly and waits first)
  const bool scored = a.max_pages > a.select;
  if (!scored) pdl_wait();
  SparseRow r;
  r.load(a, b);
  const int taken = min(r.pages, a.select);
  const int lo = (int)((int64_t)taken * split / S), hi = (int)((int64_t)taken * (split + 1) / S);
  constexpr int kUnits = D / 8;
  for (int idx = threadIdx.x; idx < 16 * kUnits; idx += kSparseThreads) {
    const int row = idx / kUnits, c = idx % kUnits;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < group)
      v = *reinterpret_cast<const uint4*>(a.q + (int64_t)b * a.q_stride_b +
                                          (int64_t)(kvh * group + row) * a.q_stride_h + c * 8);
    *reinterpret_cast<uint4*>(smem + C::kQOff + row * C::kQRow + c * 16) = v;
  }
  if (scored) pdl_wait();
  pdl_launch_dependents();
  int32_t* all = split == 0 ? a.selected + ((int64_t)b * a.num_kv_heads + kvh) * a.select : nullptr;
  if (r.pages > a.select) {
    sparse_select(a, a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.max_pages, r.pages, smem, lo, hi, list, all);
  } else {
    for (int i = threadIdx.x; i < hi - lo; i += kSparseThreads) list[i] = lo + i;
    if (all != nullptr)
      for (int i = threadIdx.x; i < a.select; i += kSparseThreads) all[i] = i < taken ? i : -1;
    __syncthreads();
  }

  // ---- a warp takes units of 16 tokens: K and V through its own buffer
  const int upp = PS / kSparseUnit;  // units of a page
  const int units = (hi - lo) * upp;
  uint8_t* kt = smem + warp * 2 * C::kTile;
  uint8_t* vt = kt + C::kTile;
  const int64_t token = (int64_t)a.num_kv_heads * D;
  auto page_of = [&](int u) {  // page id of a unit of the list, -1: outside the pool
    if (u >= units) return -1;
    const int pg = a.indices[r.begin + list[u / upp]];
    if (pg < 0 || (int64_t)pg >= a.num_pages) {
      if (lane == 0) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
      return -1;
    }
    return pg;
  };
  auto live_of = [&](int u, int pg) {  // its tokens
    if (u >= units || pg < 0) return 0;
    const int len = list[u / upp] == r.pages - 1 ? r.last : PS;
    return min(kSparseUnit, max(0, len - (u % upp) * kSparseUnit));
  };
  // 16-byte unit c of row t at t * kRow + ((c ^ (t & 7)) * 16); rows past `live` are zero-filled
  auto load = [&](uint8_t* dst, int u, int pg, int live, int kv) {
    const bf16* src = a.kv + (((int64_t)max(pg, 0) * 2 + kv) * PS + (u % upp) * kSparseUnit) * token + (int64_t)kvh * D;
#pragma unroll
    for (int i = 0; i < kSparseUnit * kUnits / 32; ++i) {
      const int idx = i * 32 + lane, t = idx / kUnits, c = idx % kUnits;
      const uint32_t to = smem_u32(dst + t * C::kRow + ((c ^ (t & 7)) << 4));
      const int n = t < live ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src + (n ? t : 0) * token + c * 8), "r"(n)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float sl2 = a.scale_log2;
  const int g = lane >> 2, t4 = lane & 3;
  int pg = page_of(warp), live = live_of(warp, pg);
  int pg_n = page_of(warp + kSparseWarps);
  if (warp < units) {
    load(kt, warp, pg, live, 0);
    load(vt, warp, pg, live, 1);
  }
  for (int u = warp; u < units; u += kSparseWarps) {
    const int un = u + kSparseWarps;
    const int live_n = live_of(un, pg_n);
    asm volatile("cp.async.wait_group 1;" ::: "memory");  // K of this unit
    __syncwarp();
    float sc[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t qa[4], kb[4];
      ldsm_x4(smem_u32(smem + C::kQOff + ((lane & 7) + 8 * ((lane >> 3) & 1)) * C::kQRow + (kk * 16 + 8 * (lane >> 4)) * 2),
              qa[0], qa[1], qa[2], qa[3]);
      const int mi = lane >> 3, tok = (mi >> 1) * 8 + (lane & 7), c = 2 * kk + (mi & 1);
      ldsm_x4(smem_u32(kt + tok * C::kRow + ((c ^ (tok & 7)) << 4)), kb[0], kb[1], kb[2], kb[3]);
      mma_bf16_16816(sc[0], qa, &kb[0]);
      mma_bf16_16816(sc[1], qa, &kb[2]);
    }
    __syncwarp();
    const int pg_nn = page_of(un + kSparseWarps);
    if (un < units)
      load(kt, un, pg_n, live_n, 0);
    else
      asm volatile("cp.async.commit_group;" ::: "memory");
    // ---- online softmax (rows g and g + 8), log2 domain
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = 8 * j + 2 * t4 + c < live;
        sc[j][c] = in ? sc[j][c] * sl2 : -INFINITY;
        sc[j][2 + c] = in ? sc[j][2 + c] * sl2 : -INFINITY;
        mx0 = fmaxf(mx0, sc[j][c]);
        mx1 = fmaxf(mx1, sc[j][2 + c]);
      }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
    const float a0 = m0 == -INFINITY ? 0.f : sp_exp2(m0 - mn0), a1 = m1 == -INFINITY ? 0.f : sp_exp2(m1 - mn1);
    const float b0 = mn0 == -INFINITY ? 0.f : mn0, b1 = mn1 == -INFINITY ? 0.f : mn1;
    m0 = mn0;
    m1 = mn1;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        sc[j][c] = sp_exp2(sc[j][c] - b0);
        sc[j][2 + c] = sp_exp2(sc[j][2 + c] - b1);
        s0 += sc[j][c];
        s1 += sc[j][2 + c];
      }
    l0 = l0 * a0 + s0;
    l1 = l1 * a1 + s1;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      o[j][0] *= a0;
      o[j][1] *= a0;
      o[j][2] *= a1;
      o[j][3] *= a1;
    }
    // P as a bf16 pair (value and remainder): O keeps fp32's accuracy, for
    // products that this memory-bound loop has to spare
    uint32_t ph[4], pl_[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = sc[i >> 1][(i & 1) * 2], y = sc[i >> 1][(i & 1) * 2 + 1];
      ph[i] = pack_bf16x2(x, y);
      const float2 h = unpack_bf16x2(ph[i]);
      pl_[i] = pack_bf16x2(x - h.x, y - h.y);
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");  // V of this unit
    __syncwarp();
#pragma unroll
    for (int dc = 0; dc < D / 8; dc += 2) {
      const int mi = lane >> 3, tok = (mi & 1) * 8 + (lane & 7), c = dc + (mi >> 1);
      uint32_t vb[4];
      ldsm_x4_trans(smem_u32(vt + tok * C::kRow + ((c ^ (tok & 7)) << 4)), vb[0], vb[1], vb[2], vb[3]);
      mma_bf16_16816(o[dc], ph, &vb[0]);
      mma_bf16_16816(o[dc + 1], ph, &vb[2]);
      mma_bf16_16816(o[dc], pl_, &vb[0]);
      mma_bf16_16816(o[dc + 1], pl_, &vb[2]);
    }
    __syncwarp();
    if (un < units)
      load(vt, un, pg_n, live_n, 1);
    else
      asm volatile("cp.async.commit_group;" ::: "memory");
    live = live_n;
    pg_n = pg_nn;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- the warps' states meet in shared memory
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  __syncthreads();  // every warp is done with its buffer
  float* ow = reinterpret_cast<float*>(smem) + warp * 16 * C::kOPad;
#pragma unroll
  for (int j = 0; j < D / 8; ++j) {
    const int d = 8 * j + 2 * t4;
    if (g < group) *reinterpret_cast<float2*>(ow + g * C::kOPad + d) = make_float2(o[j][0], o[j][1]);
    if (g + 8 < group) *reinterpret_cast<float2*>(ow + (g + 8) * C::kOPad + d) = make_float2(o[j][2], o[j][3]);
  }
  if (t4 == 0) {
    wml[warp * 16 + g] = m0;
    wml[warp * 16 + g + 8] = m1;
    wml[(kSparseWarps + warp) * 16 + g] = l0;
    wml[(kSparseWarps + warp) * 16 + g + 8] = l1;
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
      *reinterpret_cast<float4*>(part + row * D + d) = acc;
      if (d == 0) {
        cml[row] = M;
        cml[16 + row] = L;
      }
    }
  }
  if (S == 1) return;
  cluster_sync_all();
  for (int idx = threadIdx.x * S + split; idx < group * (D / 4); idx += kSparseThreads * S) {
    const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
    float mc[kSparseMaxCluster], lc[kSparseMaxCluster];
    float4 v[kSparseMaxCluster];
    float M = -INFINITY;
#pragma unroll
    for (int c = 0; c < kSparseMaxCluster; ++c) {
      mc[c] = -INFINITY;
      if (c >= S) continue;
      mc[c] = dsmem_ld_f32(dsmem_map(smem_u32(cml + row), c));
      lc[c] = dsmem_ld_f32(dsmem_map(smem_u32(cml + 16 + row), c));
      v[c] = dsmem_ld_f32x4(dsmem_map(smem_u32(part + row * D + d), c));
      M = fmaxf(M, mc[c]);
    }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kSparseMaxCluster; ++c) {
      if (mc[c] == -INFINITY) continue;  // a CTA without pages
      const float f = exp2f(mc[c] - M);
      L += f * lc[c];
      acc.x += f * v[c].x;
      acc.y += f * v[c].y;
      acc.z += f * v[c].z;
      acc.w += f * v[c].w;
    }
    write(row, d, acc, L, M);
  }
  cluster_sync_all();  // no CTA leaves while another reads its state
}

}  // namespace pl

// =================================================================== host
namespace {

template <int D>
int32_t launch_attend(const pl::SparseArgs& a, int batch, void* stream) {
  auto kern = pl::sparse_attend_kernel<D>;
  const int list = 4 * ((a.select < a.max_pages ? a.select : a.max_pages) / a.splits + 2);
  const int smem = pl::SparseCfg<D>::kListOff + ((list + 15) & ~15);
  int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  if (st != PL_OK) return st;
  const dim3 grid(a.splits, a.num_kv_heads, batch);
  if (a.splits == 1) return pl_host::launch_pdl(kern, grid, dim3(pl::kSparseThreads), smem, stream, a);
  return pl_host::launch_pdl_cluster(kern, grid, dim3(pl::kSparseThreads), smem, stream, a.splits, a);
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
  return (int64_t)batch * num_kv_heads * max_pages * 4;
}

extern "C" int32_t pl_paged_sparse_decode(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv_cache, int64_t num_pages,
    const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len, int64_t total_pages,
    int32_t max_pages, const int8_t* bounds, const float* bound_scale, int32_t batch, int32_t num_qo_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float sm_scale, int32_t num_select,
    int32_t sink_pages, int32_t recent_pages, void* out, int64_t o_stride_b, int64_t o_stride_h, float* out_lse,
    int32_t* selected, void* workspace, int64_t workspace_bytes, int32_t* status_dev, void* stream) {
  if (q == nullptr || kv_cache == nullptr || indptr == nullptr || indices == nullptr || last_page_len == nullptr ||
      bounds == nullptr || bound_scale == nullptr || out == nullptr || selected == nullptr || batch < 0 ||
      num_pages <= 0 || total_pages < 0 || max_pages < 0 || num_kv_heads <= 0 || num_qo_heads <= 0 ||
      num_qo_heads % num_kv_heads != 0 || !(sm_scale > 0.f) || sink_pages < 0 || recent_pages < 1 || num_select < 1 ||
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
  int32_t st;
  if (max_pages > num_select) {
    // a warp takes 8 pages a step; as many CTAs as fill the device a few
    // times over, but no more than there are steps
    const int64_t steps = (max_pages + 8 * pl::kSparseWarps - 1) / (8 * pl::kSparseWarps);
    int64_t chunks = (8 * (int64_t)sms + items - 1) / items;
    chunks = chunks < 1 ? 1 : (chunks > steps ? steps : chunks);
    auto score = head_dim == 128 ? pl::sparse_score_kernel<128> : pl::sparse_score_kernel<64>;
    st = pl_host::launch_pdl(score, dim3((int)chunks, num_kv_heads, batch), dim3(pl::kSparseThreads), 0, stream, a);
    if (st != PL_OK) return st;
  }
  // CTAs per (row, kv head): two fit on an SM, and a warp should have a unit
  const int64_t units = (int64_t)(num_select < max_pages ? num_select : max_pages) * (page_size / pl::kSparseUnit);
  int splits = 1;
  while (splits < pl::kSparseMaxCluster && items * splits * 2 <= 2 * sms && units >= (int64_t)splits * pl::kSparseWarps)
    splits *= 2;
  a.splits = splits;
  return head_dim == 128 ? launch_attend<128>(a, batch, stream) : launch_attend<64>(a, batch, stream);
}
