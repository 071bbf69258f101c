// Decode attention cut as one line of work, shared by the windowed, the
// weight-accumulating (pl_window_decode.cu) and the 4-bit (pl_kv4_cache.cu)
// decode kernels.
//
// One query token per row.  A row of `len` cached positions has its token at
// position len - 1; it sees j <= len - 1 with j >= len - window or j < sinks
// (window 0: all).  Work is counted in tiles of 16 positions: an item is a
// (row, block of kv heads), its visible tiles in order, and all items stand
// in one line, rows in order and the blocks of a row behind one another.  The
// line is cut into equal pieces, one per CTA, on the device, since only the
// device knows the rows' lengths: ragged batches load every SM alike, and a
// single row is split over all of them.  Every item also weighs `pad` tiles
// for its fixed cost (query load, join of the warps, output).
//
// A CTA that holds a whole item writes its output; pieces of items leave
// (O unnormalised, max, sum) in the workspace, and line_finish_kernel joins
// them in CTA order.  A CTA has at most two pieces of items it does not hold
// whole: its first (slot 0: it does not begin the item) and its last (slot 1).
// Every sum has a fixed order, nothing in the workspace needs initialisation.
#pragma once

#include "pl_common.cuh"

namespace pl {

constexpr int kTile = 16;               // positions per tile (the tensor cores' M or K)
constexpr float kLineSlack = 8.0f;      // log2 growth of a maximum that is tolerated before O is rescaled

struct LineArgs {
  const bf16* q;
  int64_t q_stride_b, q_stride_h;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_page_len;
  int64_t total_pages;   // entries of indices
  int64_t num_pages;     // pages of the pool
  int32_t batch, num_qo_heads, num_kv_heads, group, page_size;
  int32_t window, sinks;            // window 0: none
  int32_t item_heads, items;        // kv heads per item, items per row
  int32_t ctas, pad, min_tiles;     // CTAs of the grid; fixed cost of an item; smallest piece, in tiles
  float scale_log2;                 // sm_scale * log2(e)
  bf16* out;
  int64_t o_stride_b, o_stride_h;
  float* out_lse;                   // [batch, Hq], natural log, nullable
  float* partial;                   // [ctas][2][item_heads * group][D + 4]
  float* scores;                    // weights only: [total_pages * page_size / 16][Hq][16], log2 domain
  int32_t* status;
};

struct RowSpan {
  int32_t begin;   // first entry in indices
  int32_t len;     // cached positions
  int32_t wlo;     // first position of the window
  int32_t early;   // tiles of sinks in front of the window's first tile
  int32_t first;   // the window's first tile
  int32_t n;       // visible tiles
  __device__ __forceinline__ int tile(int u) const { return u < early ? u : u - early + first; }
};

// Visible tiles of row r; a page table outside `indices` counts as empty.
__device__ __forceinline__ RowSpan row_span(const LineArgs& a, int r, bool report) {
  RowSpan s;
  s.begin = a.indptr[r];
  const int32_t end = a.indptr[r + 1];
  int32_t last = a.last_page_len[r];
  int32_t pages = end - s.begin;
  if (s.begin < 0 || end < s.begin || (int64_t)end > a.total_pages) {
    if (report) set_status(a.status, PL_ERR_INVALID_ARGUMENT);
    pages = 0;
  }
  last = last < 0 ? 0 : (last > a.page_size ? a.page_size : last);
  s.len = pages > 0 ? (pages - 1) * a.page_size + last : 0;
  s.wlo = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
  s.first = s.wlo / kTile;
  const int32_t st = (int32_t)(((int64_t)a.sinks + kTile - 1) / kTile);
  s.early = st < s.first ? st : s.first;
  s.n = s.early + (s.len + kTile - 1) / kTile - s.first;
  return s;
}

// Cost of row r in the line.
__device__ __forceinline__ int64_t row_cost(const LineArgs& a, const RowSpan& s) {
  return s.n > 0 ? (int64_t)a.items * (s.n + a.pad) : 0;
}

struct LineCut {
  int64_t total;   // length of the line
  int64_t ctas;    // pieces in use
  __device__ __forceinline__ int64_t begin(int64_t c) const { return c * total / ctas; }
  __device__ __forceinline__ int64_t holder(int64_t x) const { return ((x + 1) * ctas - 1) / total; }
};

__device__ __forceinline__ LineCut line_cut(const LineArgs& a, int64_t total) {
  LineCut c;
  c.total = total;
  const int64_t most = (total + a.min_tiles - 1) / a.min_tiles;  // pieces of at least min_tiles
  c.ctas = most < a.ctas ? (most > 0 ? most : 1) : a.ctas;
  return c;
}

__device__ __forceinline__ int64_t warp_scan_i64(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Block-wide: the line's cut, and the row that holds this CTA's first position
// (row, row_start).  `sh` is shared scratch of 36 int64.  All threads call.
template <int kThreads>
__device__ __forceinline__ LineCut line_find(const LineArgs& a, int64_t cta, int64_t* sh, int& row,
                                             int64_t& row_start) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int64_t total = 0, cost = 0, incl = 0;
  const bool report = cta == 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int r = base + threadIdx.x;
    cost = r < a.batch ? row_cost(a, row_span(a, r, report)) : 0;
    incl = warp_scan_i64(cost, lane);
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    int64_t before = total;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh[w];
      total += sh[w];
    }
    incl += before;
    __syncthreads();
  }
  const LineCut cut = line_cut(a, total);
  const int64_t at = cut.begin(cta);
  if (threadIdx.x == 0) {
    sh[32] = a.batch;
    sh[33] = 0;
  }
  __syncthreads();
  if (a.batch <= kThreads) {
    if (cost > 0 && incl - cost <= at && at < incl) {
      sh[32] = threadIdx.x;
      sh[33] = incl - cost;
    }
  } else {
    int64_t run = 0;
    for (int base = 0; base < a.batch; base += kThreads) {
      const int r = base + threadIdx.x;
      cost = r < a.batch ? row_cost(a, row_span(a, r, false)) : 0;
      incl = warp_scan_i64(cost, lane);
      if (lane == 31) sh[warp] = incl;
      __syncthreads();
      int64_t before = run;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh[w];
        run += sh[w];
      }
      incl += before;
      if (cost > 0 && incl - cost <= at && at < incl) {
        sh[32] = r;
        sh[33] = incl - cost;
      }
      __syncthreads();
    }
  }
  __syncthreads();
  row = (int)sh[32];
  row_start = sh[33];
  return cut;
}

// The segments of [begin, end) of the line in order: f(row, span, item, lo, hi)
// for tiles lo .. hi of an item; f returns false to stop.
template <typename F>
__device__ __forceinline__ void for_each_segment(const LineArgs& a, int row, int64_t start, int64_t begin, int64_t end,
                                                 F f) {
  for (; row < a.batch && start < end; ++row) {
    const RowSpan s = row_span(a, row, false);
    if (s.n == 0) continue;
    const int64_t per = s.n + a.pad;
    int item = begin > start ? (int)((begin - start) / per) : 0;
    for (; item < a.items; ++item) {
      const int64_t at = start + item * per + a.pad;  // line position of the item's first tile
      if (at >= end) break;
      const int64_t lo = begin > at ? begin - at : 0;
      const int64_t hi = end - at < s.n ? end - at : s.n;
      if (lo < hi && !f(row, s, item, (int)lo, (int)hi)) return;
    }
    start += a.items * per;
  }
}

// 2^x on the multi-function unit; x = -inf gives 0.
__device__ __forceinline__ float line_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Transpose of an 8x8 matrix of 16-bit values held one row of pairs a lane.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Joins the pieces of items that no CTA held whole, in CTA order, and writes
// rows that see nothing (O = 0, LSE = -inf).  One block per (kv head, row);
// the block's threads share the pieces, so that a row cut over all CTAs is
// read with many loads in flight.
template <int D>
__global__ void __launch_bounds__(256) line_finish_kernel(const LineArgs a) {
  constexpr int kThreads = 256, kPiece = D + 4;
  __shared__ int64_t sums[2 * (kThreads / 32)];
  __shared__ __align__(16) float part[kThreads * 4];
  __shared__ float2 part_ml[kThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, row = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int64_t before = 0, total = 0;
  for (int r = threadIdx.x; r < a.batch; r += kThreads) {
    const int64_t c = row_cost(a, row_span(a, r, false));
    total += c;
    if (r < row) before += c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    sums[2 * warp] = total;
    sums[2 * warp + 1] = before;
  }
  __syncthreads();
  total = before = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    total += sums[2 * w];
    before += sums[2 * w + 1];
  }
  const RowSpan s = row_span(a, row, false);
  const int item = kvh / a.item_heads, sub = kvh % a.item_heads;
  int64_t c0 = 0, c1 = -1;
  if (s.n > 0) {
    const LineCut cut = line_cut(a, total);
    const int64_t at = before + (int64_t)item * (s.n + a.pad) + a.pad;
    c0 = cut.holder(at);
    c1 = cut.holder(at + s.n - 1);
    if (c0 == c1) return;  // written by its CTA
  }
  // (M, L, acc) joined with another state; an empty one has m = -inf.
  auto join = [](float& M, float& L, float4& acc, float m, float l, const float4& o) {
    const float top = fmaxf(M, m);
    const float w0 = M == -INFINITY ? 0.f : exp2f(M - top), w1 = m == -INFINITY ? 0.f : exp2f(m - top);
    M = top;
    L = w0 * L + w1 * l;
    acc.x = w0 * acc.x + w1 * o.x;
    acc.y = w0 * acc.y + w1 * o.y;
    acc.z = w0 * acc.z + w1 * o.z;
    acc.w = w0 * acc.w + w1 * o.w;
  };
  // thread = (share of the pieces, head of the group, 4 channels)
  const int per = D / 4;
  const int heads = min(a.group, kThreads / per);
  const int shares = kThreads / (heads * per);
  for (int h0 = 0; h0 < a.group; h0 += heads) {
    const int share = threadIdx.x / (heads * per), hh = threadIdx.x / per % heads, d = 4 * (threadIdx.x % per);
    const int h = h0 + hh;
    const bool on = share < shares && h < a.group;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
      const int head = sub * a.group + h, heads_item = a.item_heads * a.group;
      auto piece = [&](int64_t c) {
        return a.partial + ((c * 2 + (c == c0 ? 1 : 0)) * heads_item + head) * kPiece;
      };
#pragma unroll 4
      for (int64_t c = c0 + share; c <= c1; c += shares) {
        const float* p = piece(c);
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + D));
        const float4 o = __ldcg(reinterpret_cast<const float4*>(p + d));
        join(M, L, acc, ml.x, ml.y, o);
      }
    }
    reinterpret_cast<float4*>(part)[threadIdx.x] = acc;
    part_ml[threadIdx.x] = make_float2(M, L);
    __syncthreads();
    if (on && share == 0) {
      for (int i = 1; i < shares; ++i) {
        const int at = threadIdx.x + i * heads * per;
        join(M, L, acc, part_ml[at].x, part_ml[at].y, reinterpret_cast<const float4*>(part)[at]);
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;  // (a sum of NaN stays NaN)
      const int qh = kvh * a.group + h;
      bf16* dst = a.out + (int64_t)row * a.o_stride_b + (int64_t)qh * a.o_stride_h + d;
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      if (a.out_lse != nullptr && d == 0)
        a.out_lse[(int64_t)row * a.num_qo_heads + qh] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
    __syncthreads();
  }
}

}  // namespace pl

namespace pl_host {

// Bytes of the pieces of a line of `ctas` CTAs.
inline int64_t line_partial_bytes(int ctas, int heads_item, int head_dim) {
  return (int64_t)ctas * 2 * heads_item * (head_dim + 4) * 4;
}

template <int D>
int32_t launch_line_finish(const pl::LineArgs& a, void* stream) {
  return launch_pdl(pl::line_finish_kernel<D>, dim3(a.num_kv_heads, a.batch), dim3(256), 0, stream, a);
}

// Host checks shared by the line decodes; head_dim, group and page size.
inline int32_t line_check(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* cache, int64_t num_pages,
                          const int32_t* indptr, const int32_t* indices, const int32_t* last, int64_t total_pages,
                          int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t ps, float sm_scale,
                          int32_t window, int32_t sinks, const void* out, int64_t o_stride_b, int64_t o_stride_h) {
  if (batch < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || window < 0 || sinks < 0 || total_pages < 0 ||
      num_pages <= 0 || cache == nullptr || !(sm_scale > 0.f))
    return PL_ERR_INVALID_ARGUMENT;
  if ((d != 64 && d != 128) || hq / hkv > 16 || (ps != 16 && ps != 32 && ps != 64 && ps != 128) || batch > 65535 ||
      hkv > 65535 || total_pages * ps > 0x7FFFFFFFll || num_pages * ps > 0x3FFFFFFFll)
    return PL_ERR_UNSUPPORTED;
  if (batch == 0) return PL_OK;
  if (q == nullptr || out == nullptr || indptr == nullptr || last == nullptr || (indices == nullptr && total_pages > 0))
    return PL_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out)) & 15) !=
          0 ||
      q_stride_b % 8 != 0 || q_stride_h % 8 != 0 || o_stride_b % 8 != 0 || o_stride_h % 8 != 0)
    return PL_ERR_INVALID_ARGUMENT;
  return PL_OK;
}

}  // namespace pl_host
