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
constexpr int kSparseThreads = 256;
constexpr int kSparseWarps = kSparseThreads / 32;

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
  int32_t max_pages;     // scores kept per (row, kv head)
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

// Scores of all pages of (row b, kv head): one warp per page.
template <int D>
__global__ void __launch_bounds__(kSparseThreads) sparse_score_kernel(const SparseArgs a) {
  __shared__ int8_t qi[16][D];
  __shared__ float red[kSparseWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.y, b = blockIdx.z;
  SparseRow r;
  r.load(a, b);
  if (r.pages <= a.select) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = 0.f;
  for (int i = threadIdx.x; i < a.group * D; i += kSparseThreads) {
    const float v = fabsf(bf2f(a.q[(int64_t)b * a.q_stride_b + (int64_t)(kvh * a.group + i / D) * a.q_stride_h + i % D]));
    m = fmaxf(m, v);
  }
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[0];
  for (int w = 1; w < kSparseWarps; ++w) m = fmaxf(m, red[w]);
  const float sq = __fmul_rn(m, 1.0f / 127.0f);
  for (int i = threadIdx.x; i < a.group * D; i += kSparseThreads) {
    const float v = bf2f(a.q[(int64_t)b * a.q_stride_b + (int64_t)(kvh * a.group + i / D) * a.q_stride_h + i % D]);
    const float x = rintf(__fdiv_rn(v, sq > 0.f ? sq : 1.f));
    qi[i / D][i % D] = isfinite(x) ? (int8_t)fminf(fmaxf(x, -127.f), 127.f) : 0;
  }
  __syncthreads();
  uint32_t* keys = a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.max_pages;
  for (int p = blockIdx.x * kSparseWarps + warp; p < r.pages; p += gridDim.x * kSparseWarps) {
    uint32_t key;
    if (p < a.sink || p >= r.pages - a.recent) {
      key = 0xffffffffu;
    } else {
      const int pg = a.indices[r.begin + p];
      if (pg < 0 || pg >= a.num_pages) {
        if (lane == 0) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
        key = 0;
      } else {
        const int8_t* bd = a.bounds + ((int64_t)pg * a.num_kv_heads + kvh) * 2 * D;
        int best = INT32_MIN;
        for (int g = 0; g < a.group; ++g) {
          int s = 0;
          for (int d = lane; d < D; d += 32) {
            const int x = qi[g][d];
            s += max(x * bd[d], x * bd[D + d]);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          best = max(best, s);
        }
        const float sc = a.scale[(int64_t)pg * a.num_kv_heads + kvh];
        key = order_key(isinf(sc) ? INFINITY : __fmul_rn((float)best, sc));
      }
    }
    if (lane == 0) keys[p] = key;
  }
}

// Selected pages of one (row, kv head): the threshold key bit by bit, then
// the pages above it and the first ones at it, in index order.
__global__ void __launch_bounds__(kSparseThreads) sparse_select_kernel(const SparseArgs a) {
  __shared__ int cnt;
  __shared__ int warp_n[kSparseWarps][2];
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, b = blockIdx.y;
  SparseRow r;
  r.load(a, b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t* sel = a.selected + ((int64_t)b * a.num_kv_heads + kvh) * a.select;
  const int n = r.pages;
  if (n <= a.select) {
    for (int i = threadIdx.x; i < a.select; i += kSparseThreads) sel[i] = i < n ? i : -1;
    return;
  }
  const uint32_t* keys = a.keys + ((int64_t)b * a.num_kv_heads + kvh) * a.max_pages;
  uint32_t t = 0;  // largest t with at least `select` keys >= t
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (threadIdx.x == 0) cnt = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < n; i += kSparseThreads) mine += keys[i] >= c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) atomicAdd(&cnt, mine);
    __syncthreads();
    if (cnt >= a.select) t = c;
    __syncthreads();
  }
  if (threadIdx.x == 0) cnt = 0;
  __syncthreads();
  int above = 0;
  for (int i = threadIdx.x; i < n; i += kSparseThreads) above += keys[i] > t;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
  if (lane == 0) atomicAdd(&cnt, above);
  __syncthreads();
  const int ties = a.select - cnt;
  int at = 0, tie_at = 0;  // taken, and keys at t met, in front of this step
  for (int i0 = 0; i0 < n; i0 += kSparseThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < n ? keys[i] : 0u;
    const bool gt = i < n && k > t, eq = i < n && k == t;
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) {
      warp_n[warp][0] = __popc(bg);
      warp_n[warp][1] = __popc(be);
    }
    __syncthreads();
    int g0 = 0, e0 = tie_at, ga = 0, ea = 0;
    for (int w = 0; w < kSparseWarps; ++w) {
      if (w < warp) {
        g0 += warp_n[w][0];
        e0 += warp_n[w][1];
      }
      ga += warp_n[w][0];
      ea += warp_n[w][1];
    }
    const uint32_t below = (1u << lane) - 1;
    const int eq_rank = e0 + __popc(be & below);
    // position: the keys above t before i, and the taken ties before i
    const int pos = at + g0 + __popc(bg & below) + min(eq_rank, ties) - min(tie_at, ties);
    if (gt || (eq && eq_rank < ties)) sel[pos] = i;
    at += ga + min(tie_at + ea, ties) - min(tie_at, ties);
    tie_at += ea;
  }
}

// Attention over the selected pages: one CTA per (row, kv head), a warp per
// token, channels over the lanes, running (O, m, l) per warp and head.
template <int D>
__global__ void __launch_bounds__(kSparseThreads) sparse_attend_kernel(const SparseArgs a) {
  constexpr int E = D / 32;
  __shared__ float so[kSparseWarps][D];
  __shared__ float sm[kSparseWarps], sl[kSparseWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  SparseRow r;
  r.load(a, b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int PS = a.page_size;
  const int head = kvh * a.group + g;
  const int32_t* sel = a.selected + ((int64_t)b * a.num_kv_heads + kvh) * a.select;
  const int n = min(r.pages, a.select);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf2f(a.q[(int64_t)b * a.q_stride_b + (int64_t)head * a.q_stride_h + lane * E + e]) * a.scale_log2;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int i = warp; i < n * PS; i += kSparseWarps) {
    const int p = sel[i / PS], t = i % PS;
    if (p == r.pages - 1 && t >= r.last) continue;
    const int pg = a.indices[r.begin + p];
    if (pg < 0 || pg >= a.num_pages) {
      if (lane == 0) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
      continue;
    }
    const bf16* k = a.kv + ((((int64_t)pg * 2) * PS + t) * a.num_kv_heads + kvh) * D + lane * E;
    const bf16* v = k + (int64_t)PS * a.num_kv_heads * D;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], bf2f(k[e]), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float w = mn == -INFINITY ? 0.f : exp2f(s - mn), al = m == -INFINITY ? 0.f : exp2f(m - mn);
    l = l * al + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * al + w * bf2f(v[e]);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kSparseThreads) {
    float M = -INFINITY;
    for (int w = 0; w < kSparseWarps; ++w) M = fmaxf(M, sm[w]);
    float L = 0.f, acc = 0.f;
    for (int w = 0; w < kSparseWarps; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M);
      L += f * sl[w];
      acc += f * so[w][d];
    }
    a.out[(int64_t)b * a.o_stride_b + (int64_t)head * a.o_stride_h + d] = f2bf(L == 0.f ? 0.f : acc / L);
    if (d == 0 && a.out_lse != nullptr)
      a.out_lse[(int64_t)b * a.num_qo_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  }
}

}  // namespace pl

// =================================================================== host
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
      sink_pages + recent_pages > num_select)
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
  int32_t st;
  if (max_pages > num_select) {
    const int chunks = (max_pages + 63) / 64;
    auto score = head_dim == 128 ? pl::sparse_score_kernel<128> : pl::sparse_score_kernel<64>;
    st = pl_host::launch_pdl(score, dim3(chunks, num_kv_heads, batch), dim3(pl::kSparseThreads), 0, stream, a);
    if (st != PL_OK) return st;
  }
  st = pl_host::launch_pdl(pl::sparse_select_kernel, dim3(num_kv_heads, batch), dim3(pl::kSparseThreads), 0, stream, a);
  if (st != PL_OK) return st;
  auto attend = head_dim == 128 ? pl::sparse_attend_kernel<128> : pl::sparse_attend_kernel<64>;
  return pl_host::launch_pdl(attend, dim3(num_kv_heads, group, batch), dim3(pl::kSparseThreads), 0, stream, a);
}
