// Operations on the pages of a paged KV cache whose bookkeeping lives on the
// device: rows take new slots, fork, give their pages back, and move their
// kept tokens together.
//
// State: refcount[p] = rows that hold page p (0: free); row r holds
// row_pages[r][0 .. row_num[r]) and its last page last_len[r] tokens.  There
// is no free list: a call that needs N pages takes the N lowest free ids, in
// row order, so its result is a function of the state alone.
//
// The bookkeeping of one call runs in one CTA, or, for a large pool, in one
// thread-block cluster (the pool's counts are read once, spread over the
// warps, and ranked by a prefix sum, across CTAs through distributed shared
// memory).  It checks everything that can be refused before it changes
// anything; a refused call leaves the state as it was and says why in the
// status word.  Moving the data is a second launch over the jobs that the
// first one listed.
//
// The bookkeeping is a chain of dependent reads, barriers and prefix sums and
// is bound by their latency: 6 to 10 us for up to 96 rows, 20 us where 12 rows
// give 24000 kept positions.  The copy is bound by HBM: an eviction that moves
// half of 12 contexts of 4096 tokens in 16 layers takes 519 us for 3.1 GB read
// and written, 6.0 TB/s (91 % of a plain copy's rate), bookkeeping included.
#include "pl_common.cuh"

namespace pl {

constexpr int kPoolThreads = 1024;
constexpr int kPoolWarps = kPoolThreads / 32;
constexpr int kPoolCtas = 8;        // of a cluster
constexpr int kPoolMaxRows = 4096;  // rows of a table (as pl_page_table_build)
constexpr int kPerThread = kPoolMaxRows / kPoolThreads;
// Pools up to this size take one CTA, whose 32 warps read 4096 counts a step;
// past it, that costs more than starting and syncing a cluster does.  A reserve
// and a release of 64 rows, us on one CTA and on a cluster: 4096 pages 10.7,
// 11.4; 16384 pages 13.0, 11.5; 262144 pages 57.8, 15.6.
constexpr int kPoolOneCta = 8192;

struct PoolState {
  int32_t* refcount;
  int32_t num_pages;
  int32_t* row_pages;
  int32_t* row_num;
  int32_t* last_len;
  int32_t rows, cap, page_size;
  int32_t* status;
};

// One page to fill: `tokens` tokens of `page`.  row < 0: they are the first
// tokens of page ~row.  row >= 0: they are the kept tokens
// [index * page_size, ...) of that row.
struct PageJob {
  int32_t page, row, index, tokens;
};

struct PoolSmem {
  int32_t first[kPoolMaxRows + 1];  // exclusive prefix of the pages wanted
  int32_t warp_sum[kPoolWarps];
  int32_t cta_free;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ int pool_warp_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Entries of a thread: `per` consecutive ones, per * kPoolThreads >= n.
__device__ __forceinline__ int pool_per(int n) { return (n + kPoolThreads - 1) / kPoolThreads; }

// Exclusive prefix over the entries (v[i] of entry threadIdx.x * per + i) into
// s.first[0 .. n], and the total in s.first[kPoolMaxRows]; every CTA does the same.
__device__ __forceinline__ void pool_prefix(PoolSmem& s, const int* v, int n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = pool_per(n);
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) sum += i < per ? v[i] : 0;
  const int inc = pool_warp_scan(sum);
  __syncthreads();
  if (lane == 31) s.warp_sum[warp] = inc;
  __syncthreads();
  const int warps = pool_warp_scan(s.warp_sum[lane]);
  int at = (warp > 0 ? __shfl_sync(0xffffffffu, warps, max(warp - 1, 0)) : 0) + inc - sum;
  const int total = __shfl_sync(0xffffffffu, warps, 31);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int e = (int)threadIdx.x * per + i;
    if (i < per && e <= n) s.first[e] = at;
    at += i < per ? v[i] : 0;
  }
  if (threadIdx.x == 0) {
    s.first[n] = total;
    s.first[kPoolMaxRows] = total;
  }
  __syncthreads();
}

// The entry that owns rank k: first[e] <= k < first[e + 1].
__device__ __forceinline__ int pool_owner(const PoolSmem& s, int k, int n) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.first[mid] <= k) lo = mid; else hi = mid;
  }
  return lo;
}

// Whether any thread of the CTA saw `bad` (the CTAs of the cluster look at
// the same state, so their answers agree).
__device__ __forceinline__ bool pool_any(bool bad) { return __syncthreads_or(bad) != 0; }

// Ranks the free pages and calls take(rank, page) for the `need` lowest.
// false: fewer than `need` are free, nothing was called.  Every CTA calls
// it; the counts are read before any CTA goes on past the barrier in here,
// and taken pages' counts are set by `take`.
template <int CTAS, typename Take>
__device__ __forceinline__ bool pool_take(PoolSmem& s, const int32_t* refcount, int num_pages, int need, Take take) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CTAS > 1 ? (int)cluster_rank() : 0;
  auto sync = [] {
    if constexpr (CTAS > 1)
      cluster_sync_all();
    else
      __syncthreads();
  };
  if (need == 0) {  // the same for every CTA; what follows may change counts
    sync();
    return true;
  }
  // contiguous range of every warp, in steps of 128 pages
  const int steps = (num_pages + 127) / 128;
  const int per = (steps + CTAS * kPoolWarps - 1) / (CTAS * kPoolWarps);
  const int p0 = (int)min((int64_t)num_pages, ((int64_t)rank * kPoolWarps + warp) * per * 128);
  const int p1 = (int)min((int64_t)num_pages, (int64_t)p0 + per * 128);
  auto load = [&](int p, int* c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = p + 32 * i + lane < p1 ? __ldcg(refcount + p + 32 * i + lane) : 1;
  };
  int count = 0;
  int head[4] = {1, 1, 1, 1};  // the first step's counts, for the second pass
#pragma unroll 4
  for (int p = p0; p < p1; p += 128) {
    int c[4];
    load(p, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p == p0) head[i] = c[i];
      count += __popc(__ballot_sync(0xffffffffu, c[i] == 0));
    }
  }
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = count;
  __syncthreads();
  const int warps = pool_warp_scan(s.warp_sum[lane]);
  int before = warp > 0 ? __shfl_sync(0xffffffffu, warps, max(warp - 1, 0)) : 0;
  int all = __shfl_sync(0xffffffffu, warps, 31);
  if constexpr (CTAS > 1) {
    if (threadIdx.x == 0) s.cta_free = all;
    cluster_sync_all();
    int v = 0;
    if (lane < CTAS) {
      const uint32_t at = dsmem_map(smem_u32(&s.cta_free), lane);
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    }
    const int ctas = pool_warp_scan(v);
    before += rank > 0 ? __shfl_sync(0xffffffffu, ctas, max(rank - 1, 0)) : 0;
    all = __shfl_sync(0xffffffffu, ctas, 31);
  }
  const bool enough = all >= need;
  if (enough) {
    int k = before;
    for (int p = p0; p < p1 && k < need; p += 128) {
      int c[4];
      if (p == p0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = head[i];
      } else {
        load(p, c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = __ballot_sync(0xffffffffu, c[i] == 0);
        const int mine = k + __popc(b & ((1u << lane) - 1));
        if (c[i] == 0 && mine < need) take(mine, p + 32 * i + lane);
        k += __popc(b);
      }
    }
  }
  sync();  // the remote reads are done, and every taken page is seen by all
  return enough;
}

// ---------------------------------------------------------------- release
__global__ void __launch_bounds__(256) page_release_kernel(const PoolState p, const int32_t* __restrict__ rows, int n) {
  __shared__ int32_t num_s;
  pdl_launch_dependents();
  pdl_wait();
  const int r = rows[blockIdx.x];
  if (r < 0 || r >= p.rows) {
    if (threadIdx.x == 0) set_status(p.status, PL_ERR_INVALID_ARGUMENT);
    return;
  }
  if (threadIdx.x == 0) {
    num_s = atomicExch(&p.row_num[r], 0);  // a row that is listed twice is released once
    p.last_len[r] = 0;
  }
  __syncthreads();
  const int num = min(max(num_s, 0), p.cap);
  for (int i = threadIdx.x; i < num; i += blockDim.x) {
    const int pg = p.row_pages[(int64_t)r * p.cap + i];
    if (pg < 0 || pg >= p.num_pages) {
      set_status(p.status, PL_ERR_PAGE_OUT_OF_RANGE);
    } else if (atomicSub(&p.refcount[pg], 1) <= 0) {
      atomicAdd(&p.refcount[pg], 1);
      set_status(p.status, PL_ERR_REFCOUNT);
    }
  }
}

// One reference less for page pg (of a row's table).
__device__ __forceinline__ void pool_drop(const PoolState& p, int pg) {
  if (pg < 0 || pg >= p.num_pages) {
    set_status(p.status, PL_ERR_PAGE_OUT_OF_RANGE);
  } else if (atomicSub(&p.refcount[pg], 1) <= 0) {
    atomicAdd(&p.refcount[pg], 1);
    set_status(p.status, PL_ERR_REFCOUNT);
  }
}

// ---------------------------------------------------------------- reserve
template <int CTAS>
__global__ void __launch_bounds__(kPoolThreads, 1)
    page_reserve_kernel(const PoolState p, const int32_t* __restrict__ tok_indptr, int total,
                        int32_t* __restrict__ slot_page, int32_t* __restrict__ slot_off,
                        int32_t* __restrict__ positions, int32_t* __restrict__ out_indptr,
                        int32_t* __restrict__ out_indices, int64_t max_indices) {
  __shared__ PoolSmem s;
  __shared__ int32_t csr[kPoolMaxRows + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int rank = CTAS > 1 ? (int)cluster_rank() : 0;
  const int PS = p.page_size;
  const int per = pool_per(p.rows);
  int want[kPerThread], grown[kPerThread];
  bool bad = threadIdx.x == 0 && (tok_indptr[0] != 0 || tok_indptr[p.rows] != total);
  int why = PL_ERR_INVALID_ARGUMENT;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = threadIdx.x * per + i;
    want[i] = grown[i] = 0;
    if (i >= per || r >= p.rows) continue;
    const int n = tok_indptr[r + 1] - tok_indptr[r];
    const int num = p.row_num[r], last = p.last_len[r];
    if (n < 0 || num < 0 || num > p.cap || (num > 0 && (last <= 0 || last > PS))) {
      bad = true;
      continue;
    }
    grown[i] = num;
    if (n == 0) continue;
    const int64_t len = num > 0 ? (int64_t)(num - 1) * PS + last : 0;
    const int64_t g = (len + n + PS - 1) / PS;
    if (g > p.cap) {
      bad = true;
      why = PL_ERR_ROW_CAPACITY;
      continue;
    }
    if (num > 0 && last < PS) {  // the new tokens go into the last page: it has to be the row's own
      const int pg = p.row_pages[(int64_t)r * p.cap + num - 1];
      if (pg < 0 || pg >= p.num_pages) {
        bad = true;
        why = PL_ERR_PAGE_OUT_OF_RANGE;
        continue;
      }
      if (p.refcount[pg] != 1) {
        bad = true;
        why = PL_ERR_PAGE_SHARED;
        continue;
      }
    }
    grown[i] = (int)g;
    want[i] = (int)g - num;
  }
  if (bad) set_status(p.status, why);
  bool refused = pool_any(bad);
  // page table offsets (out_indptr), then the pages wanted
  pool_prefix(s, grown, p.rows);
  for (int i = threadIdx.x; i <= p.rows; i += kPoolThreads) csr[i] = s.first[i];
  __syncthreads();
  if (out_indices != nullptr && csr[p.rows] > max_indices) {
    if (threadIdx.x == 0) set_status(p.status, PL_ERR_WORKSPACE_TOO_SMALL);
    refused = true;
  }
  pool_prefix(s, want, p.rows);
  const int need = refused ? 0 : s.first[kPoolMaxRows];
  const bool enough = pool_take<CTAS>(s, p.refcount, p.num_pages, need, [&](int k, int page) {
    const int r = pool_owner(s, k, p.rows);
    p.row_pages[(int64_t)r * p.cap + p.row_num[r] + (k - s.first[r])] = page;
    p.refcount[page] = 1;
  });
  if (!enough && threadIdx.x == 0) set_status(p.status, PL_ERR_POOL_EXHAUSTED);
  if (refused || !enough) {  // no slots: the appends that follow reject these, whatever the buffers held
    for (int64_t i = rank * kPoolThreads + (int)threadIdx.x; i < total; i += CTAS * kPoolThreads) {
      slot_page[i] = slot_off[i] = -1;
      if (positions != nullptr) positions[i] = 0;
    }
    return;
  }
  // slots of the new tokens and the page table, rows dealt over the warps
  const int lane = threadIdx.x & 31;
  for (int r = rank * kPoolWarps + (threadIdx.x >> 5); r < p.rows; r += CTAS * kPoolWarps) {
    const int num = p.row_num[r], last = p.last_len[r];
    const int t0 = tok_indptr[r], n = tok_indptr[r + 1] - t0;
    const int g = csr[r + 1] - csr[r];
    const int len = num > 0 ? (num - 1) * PS + last : 0;
    const int32_t* pages = p.row_pages + (int64_t)r * p.cap;
    for (int i = lane; i < n; i += 32) {
      const int pos = len + i;
      slot_page[t0 + i] = __ldcg(pages + pos / PS);
      slot_off[t0 + i] = pos % PS;
      if (positions != nullptr) positions[t0 + i] = pos;
    }
    if (out_indices != nullptr)
      for (int i = lane; i < g; i += 32) out_indices[csr[r] + i] = __ldcg(pages + i);
    if (out_indptr != nullptr && lane == 0) {
      out_indptr[r + 1] = csr[r + 1];
      if (r == 0) out_indptr[0] = 0;
    }
    __syncwarp();
    if (n > 0 && lane == 0) {
      p.row_num[r] = g;
      p.last_len[r] = len + n - (g - 1) * PS;
    }
  }
}

// ------------------------------------------------------------------- fork
template <int CTAS>
__global__ void __launch_bounds__(kPoolThreads, 1)
    page_fork_kernel(const PoolState p, const int32_t* __restrict__ src_rows, const int32_t* __restrict__ dst_rows,
                     int n, int32_t* __restrict__ job_count, PageJob* __restrict__ jobs) {
  __shared__ PoolSmem s;
  __shared__ uint32_t taken[kPoolMaxRows / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int rank = CTAS > 1 ? (int)cluster_rank() : 0;
  const int PS = p.page_size;
  if (threadIdx.x < kPoolMaxRows / 32) taken[threadIdx.x] = 0;
  __syncthreads();
  const int per = pool_per(n);
  int want[kPerThread];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int f = threadIdx.x * per + i;
    want[i] = 0;
    if (i >= per || f >= n) continue;
    const int src = src_rows[f], dst = dst_rows[f];
    if (src < 0 || src >= p.rows || dst < 0 || dst >= p.rows || src == dst || p.row_num[dst] != 0) {
      bad = true;
      continue;
    }
    if (atomicOr(&taken[dst >> 5], 1u << (dst & 31)) & (1u << (dst & 31))) bad = true;  // two forks into one row
    const int num = p.row_num[src], last = p.last_len[src];
    if (num < 0 || num > p.cap || (num > 0 && (last <= 0 || last > PS))) {
      bad = true;
      continue;
    }
    want[i] = num > 0 && last < PS ? 1 : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {  // a row that another fork fills is no source
    const int f = threadIdx.x * per + i;
    if (i < per && f < n && src_rows[f] >= 0 && src_rows[f] < p.rows && ((taken[src_rows[f] >> 5] >> (src_rows[f] & 31)) & 1u))
      bad = true;
  }
  if (bad) set_status(p.status, PL_ERR_INVALID_ARGUMENT);
  const bool refused = pool_any(bad);
  pool_prefix(s, want, n);
  const int need = refused ? 0 : s.first[kPoolMaxRows];
  const bool enough = pool_take<CTAS>(s, p.refcount, p.num_pages, need, [&](int k, int page) {
    const int f = pool_owner(s, k, n);
    const int src = src_rows[f], num = p.row_num[src];
    const int old = p.row_pages[(int64_t)src * p.cap + num - 1];
    const bool ok = old >= 0 && old < p.num_pages;
    if (!ok) set_status(p.status, PL_ERR_PAGE_OUT_OF_RANGE);
    p.row_pages[(int64_t)dst_rows[f] * p.cap + num - 1] = page;
    p.refcount[page] = 1;
    jobs[k] = PageJob{page, ~(ok ? old : 0), 0, ok ? p.last_len[src] : 0};
  });
  if (!enough && threadIdx.x == 0) set_status(p.status, PL_ERR_POOL_EXHAUSTED);
  const bool done = !refused && enough;
  if (rank == 0 && threadIdx.x == 0) *job_count = done ? need : 0;
  if (!done) return;
  const int lane = threadIdx.x & 31;
  for (int f = rank * kPoolWarps + (threadIdx.x >> 5); f < n; f += CTAS * kPoolWarps) {
    const int src = src_rows[f], dst = dst_rows[f];
    const int num = p.row_num[src], last = p.last_len[src];
    const int shared = num - (num > 0 && last < PS ? 1 : 0);
    for (int i = lane; i < shared; i += 32) {
      const int pg = p.row_pages[(int64_t)src * p.cap + i];
      p.row_pages[(int64_t)dst * p.cap + i] = pg;
      if (pg >= 0 && pg < p.num_pages)
        atomicAdd(&p.refcount[pg], 1);
      else
        set_status(p.status, PL_ERR_PAGE_OUT_OF_RANGE);
    }
    if (lane == 0) {
      p.row_num[dst] = num;
      p.last_len[dst] = num > 0 ? last : 0;
    }
  }
}

// ---------------------------------------------------------------- compact
// Row r keeps its tokens [0, keep_from) and the positions keep[r][0 ..
// keep_count).  `stays` leading tokens keep their place; whole pages of them
// stay, the tokens after those go to new pages (their old ones may belong to
// other rows too) and the old pages are given back.  When nothing moves the
// row is cut in place, unless its new partial last page is shared.
struct CompactRow {
  int full, want, len, held;  // pages that stay, new pages, new length, old pages that are kept
};

__device__ __forceinline__ bool compact_row(const PoolState& p, int r, const int32_t* keep_from, const int32_t* keep,
                                            int64_t keep_stride, const int32_t* keep_count, int max_keep,
                                            CompactRow& c, int& why) {
  const int PS = p.page_size;
  const int num = p.row_num[r], last = p.last_len[r];
  const int kf = keep_from[r], k = keep_count[r];
  c = CompactRow{0, 0, 0, 0};
  why = PL_ERR_INVALID_ARGUMENT;
  if (num < 0 || num > p.cap || (num > 0 && (last <= 0 || last > PS))) return false;
  const int64_t old = num > 0 ? (int64_t)(num - 1) * PS + last : 0;
  if (kf < 0 || k < 0 || k > max_keep || (int64_t)kf + k > old) return false;
  // keep ascends, so keep[i] == kf + i holds up to some i: search with 8
  // probes a step (their loads overlap)
  const int32_t* kr = keep + (int64_t)r * keep_stride;
  int lo = 0, hi = k;
  while (lo < hi) {
    const int gap = (hi - lo + 8) / 9;
    int v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = lo + (j + 1) * gap - 1;
      v[j] = at < hi ? kr[at] - at : INT32_MAX;
    }
    int held = 0;  // leading probes that keep their place
#pragma unroll
    for (int j = 0; j < 8; ++j) held += held == j && v[j] == kf;
    if (held < 8) hi = min(hi, lo + (held + 1) * gap - 1);
    lo += held * gap;
  }
  const int stays = kf + lo;
  c.len = kf + k;
  c.full = stays / PS;
  const int rest = c.len - c.full * PS;
  bool cut = lo == k;
  if (cut && rest > 0) {
    const int pg = p.row_pages[(int64_t)r * p.cap + c.full];
    if (pg < 0 || pg >= p.num_pages) {
      why = PL_ERR_PAGE_OUT_OF_RANGE;
      return false;
    }
    cut = p.refcount[pg] == 1;
  }
  c.want = cut ? 0 : (rest + PS - 1) / PS;
  c.held = c.full + (cut && rest > 0 ? 1 : 0);
  return true;
}

template <int CTAS>
__global__ void __launch_bounds__(kPoolThreads, 1)
    page_compact_kernel(const PoolState p, const int32_t* __restrict__ keep_from, const int32_t* __restrict__ keep,
                        int64_t keep_stride, const int32_t* __restrict__ keep_count, int max_keep,
                        int32_t* __restrict__ job_count, int32_t* __restrict__ old_pages, int2* __restrict__ src_range,
                        PageJob* __restrict__ jobs) {
  __shared__ PoolSmem s;
  __shared__ uint32_t full_s[kPoolMaxRows];  // pages that stay; top bit: one old page more is kept (a cut)
  pdl_launch_dependents();
  pdl_wait();
  const int rank = CTAS > 1 ? (int)cluster_rank() : 0;
  const int PS = p.page_size;
  const int per = pool_per(p.rows);
  int want[kPerThread];
  bool bad = false;
  int why = PL_OK;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = threadIdx.x * per + i;
    want[i] = 0;
    if (i >= per || r >= p.rows) continue;
    CompactRow c;
    int w;
    if (!compact_row(p, r, keep_from, keep, keep_stride, keep_count, max_keep, c, w)) {
      bad = true;
      why = w;
    }
    want[i] = c.want;
    full_s[r] = (uint32_t)c.full | (c.held > c.full ? 0x80000000u : 0u);
  }
  if (bad) set_status(p.status, why);
  const bool refused = pool_any(bad);
  pool_prefix(s, want, p.rows);
  const int need = refused ? 0 : s.first[kPoolMaxRows];
  const bool enough = pool_take<CTAS>(s, p.refcount, p.num_pages, need, [&](int k, int page) {
    const int r = pool_owner(s, k, p.rows), index = (int)(full_s[r] & 0x7fffffffu) + (k - s.first[r]);
    const int len = keep_from[r] + keep_count[r];
    jobs[k] = PageJob{page, r, index, min(PS, len - index * PS)};
    p.refcount[page] = 1;
  });
  if (!enough && threadIdx.x == 0) set_status(p.status, PL_ERR_POOL_EXHAUSTED);
  const bool done = !refused && enough;
  if (rank == 0 && threadIdx.x == 0) *job_count = done ? need : 0;
  if (!done) return;
  // the old pages: noted for the copy, given back
  const int lane = threadIdx.x & 31;
  for (int r = rank * kPoolWarps + (threadIdx.x >> 5); r < p.rows; r += CTAS * kPoolWarps) {
    const int num = p.row_num[r], len = keep_from[r] + keep_count[r];
    const int moved = s.first[r + 1] - s.first[r];
    const int full = (int)(full_s[r] & 0x7fffffffu), held = full + (int)(full_s[r] >> 31);
    int32_t* pages = p.row_pages + (int64_t)r * p.cap;
    for (int i = full + lane; i < num; i += 32) {
      const int pg = pages[i];
      if (moved > 0) old_pages[(int64_t)r * p.cap + i] = pg;
      if (i >= held) pool_drop(p, pg);
    }
    __syncwarp();
    for (int i = lane; i < moved; i += 32) pages[full + i] = __ldcg(&jobs[s.first[r] + i].page);
    // positions that a moved token may come from
    if (lane == 0) src_range[r] = make_int2(full * PS, num > 0 ? (num - 1) * PS + p.last_len[r] : 0);
    __syncwarp();
    if (lane == 0) {
      const int pn = (len + PS - 1) / PS;
      p.row_num[r] = pn;
      p.last_len[r] = len - (pn > 0 ? pn - 1 : 0) * PS;
    }
  }
}

// ------------------------------------------------------------------- copy
// Fills the listed pages in every layer.  One CTA takes (job, slice of the
// 2 * layers K and V halves); the source slot of each of the page's tokens
// is looked up once, a thread's places (16-byte units of the page) are
// worked out once, and then it has kCopyDepth loads in flight per half.
struct CopyArgs {
  char* pool;
  int64_t layer_stride;  // bytes
  int32_t layers, page_size, num_pages;
  int32_t token_units;   // 16-byte units of one token's K (or V) in one layer
  const int32_t* job_count;
  const PageJob* jobs;
  const int32_t* old_pages;
  const int2* src_range;  // per row: [first, past the last) position that a moved token may come from
  int32_t cap;
  const int32_t* keep_from;
  const int32_t* keep;
  int64_t keep_stride;
  int32_t* status;
};

// 768 threads an SM with 4 loads each: the eviction above takes 519 us, with 8
// loads 543, with 2 or 4 CTAs an SM 544 and 531.
constexpr int kCopyThreads = 256;
constexpr int kCopyDepth = 4;
constexpr int kCopyCtasPerSm = 3;

__global__ void __launch_bounds__(kCopyThreads, kCopyCtasPerSm) page_copy_kernel(const CopyArgs a) {
  __shared__ int32_t src_slot[128];
  pdl_wait();
  pdl_launch_dependents();
  const int jobs = *a.job_count;
  if (jobs == 0) return;
  const int PS = a.page_size, halves = 2 * a.layers;
  // halves of a slice: one round of the CTAs when there are few, else at
  // least two, in runs of at most 8 (jobs of unequal length even out)
  const int64_t all = (int64_t)jobs * halves;
  const int64_t share = all <= 2 * (int64_t)gridDim.x ? (all + gridDim.x - 1) / gridDim.x : all / (2 * (int64_t)gridDim.x);
  const int slice = (int)min((int64_t)8, max((int64_t)1, share));
  const int slices = (halves + slice - 1) / slice;
  const int64_t half = (int64_t)PS * a.token_units;  // 16-byte units
  for (int64_t u = blockIdx.x; u < (int64_t)jobs * slices; u += gridDim.x) {
    const PageJob job = a.jobs[u / slices];
    const int h0 = (int)(u % slices) * slice, h1 = min(halves, h0 + slice);
    __syncthreads();
    for (int t = threadIdx.x; t < job.tokens; t += kCopyThreads) {
      int slot = -1;
      if (job.row < 0) {
        slot = ~job.row * PS + t;
      } else {
        const int i = job.index * PS + t, kf = a.keep_from[job.row];
        const int pos = i < kf ? i : a.keep[(int64_t)job.row * a.keep_stride + i - kf];
        const int2 in = a.src_range[job.row];
        const int pg = pos >= in.x && pos < in.y ? a.old_pages[(int64_t)job.row * a.cap + pos / PS] : -1;
        if (pg >= 0 && pg < a.num_pages)
          slot = pg * PS + pos % PS;
        else
          set_status(a.status, PL_ERR_INVALID_ARGUMENT);
      }
      src_slot[t] = slot;
    }
    __syncthreads();
    const int units = job.tokens * a.token_units;
    for (int at = threadIdx.x; at < units; at += kCopyThreads * kCopyDepth) {
      int64_t from[kCopyDepth];  // unit in a layer's half-0 plane, -1: none
      int64_t to = (int64_t)job.page * 2 * half + at;
#pragma unroll
      for (int i = 0; i < kCopyDepth; ++i) {
        const int x = at + i * kCopyThreads, t = x / a.token_units, c = x - t * a.token_units;
        const int slot = x < units ? src_slot[t] : -1;
        const int pg = slot / PS;
        from[i] = slot < 0 ? -1 : (int64_t)pg * 2 * half + (int64_t)(slot - pg * PS) * a.token_units + c;
      }
      for (int h = h0; h < h1; ++h) {
        uint4* plane = reinterpret_cast<uint4*>(a.pool + (int64_t)(h >> 1) * a.layer_stride) + (h & 1) * half;
        uint4 v[kCopyDepth];
#pragma unroll
        for (int i = 0; i < kCopyDepth; ++i)
          if (from[i] >= 0) v[i] = __ldcs(plane + from[i]);
#pragma unroll
        for (int i = 0; i < kCopyDepth; ++i)
          if (from[i] >= 0) __stcs(plane + to + i * kCopyThreads, v[i]);
      }
    }
  }
}

}  // namespace pl

// =================================================================== host
namespace {

int64_t align16(int64_t v) { return (v + 15) & ~int64_t(15); }

int32_t pool_state(int32_t* refcount, int64_t num_pages, int32_t* row_pages, int32_t* row_num, int32_t* last_len,
                   int32_t rows, int32_t cap, int32_t page_size, int32_t* status, pl::PoolState* out) {
  if (refcount == nullptr || row_pages == nullptr || row_num == nullptr || last_len == nullptr || num_pages <= 0 ||
      rows < 0 || cap <= 0 || page_size <= 0)
    return PL_ERR_INVALID_ARGUMENT;
  // slots (page * page_size + offset) and row lengths are 32-bit
  if (rows > pl::kPoolMaxRows || num_pages * page_size > 0x7FFFFFFFll || (int64_t)cap * page_size > 0x7FFFFFFFll ||
      page_size > 128 || (int64_t)rows * cap > 0x7FFFFFFFll)
    return PL_ERR_UNSUPPORTED;
  *out = pl::PoolState{refcount, (int32_t)num_pages, row_pages, row_num, last_len, rows, cap, page_size, status};
  return PL_OK;
}

int32_t copy_args(void* pool, int64_t layer_stride_bytes, int32_t layers, int64_t token_bytes, const pl::PoolState& p,
                  pl::CopyArgs* out) {
  if (pool == nullptr || layers <= 0 || token_bytes <= 0 || layer_stride_bytes < 0) return PL_ERR_INVALID_ARGUMENT;
  if (token_bytes % 16 != 0 || token_bytes > (1 << 24) || layers > (1 << 16)) return PL_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(pool) & 15) != 0 || layer_stride_bytes % 16 != 0) return PL_ERR_INVALID_ARGUMENT;
  out->pool = static_cast<char*>(pool);
  out->layer_stride = layer_stride_bytes;
  out->layers = layers;
  out->page_size = p.page_size;
  out->num_pages = p.num_pages;
  out->token_units = (int32_t)(token_bytes / 16);
  out->old_pages = nullptr;
  out->src_range = nullptr;
  out->cap = p.cap;
  out->keep_from = out->keep = nullptr;
  out->keep_stride = 0;
  out->status = p.status;
  return PL_OK;
}

int32_t launch_copy(const pl::CopyArgs& a, int64_t max_jobs, void* stream) {
  const int sms = pl_host::sm_count();
  if (sms <= 0) return PL_ERR_NO_DEVICE;
  const int64_t units = max_jobs * 2 * a.layers, most = (int64_t)sms * pl::kCopyCtasPerSm;
  return pl_host::launch_pdl(pl::page_copy_kernel, dim3((int)(units < most ? units : most)), dim3(pl::kCopyThreads), 0,
                             stream, a);
}

// A bookkeeping kernel on one CTA or, for a large pool, one cluster.
template <typename K1, typename K8, typename... Args>
int32_t launch_pool(K1 one, K8 cluster, const pl::PoolState& p, void* stream, Args... args) {
  if (p.num_pages <= pl::kPoolOneCta)
    return pl_host::launch_pdl(one, dim3(1), dim3(pl::kPoolThreads), 0, stream, p, args...);
  return pl_host::launch_pdl_cluster(cluster, dim3(pl::kPoolCtas), dim3(pl::kPoolThreads), 0, stream, pl::kPoolCtas, p,
                                     args...);
}

}  // namespace

extern "C" int32_t pl_page_release(int32_t *refcount, int64_t num_pages, int32_t *row_pages, int32_t *row_num_pages,
                                   int32_t *last_page_len, int32_t num_rows, int32_t row_capacity,
                                   const int32_t *rows, int32_t num_released, int32_t *status_dev, void *stream) {
  pl::PoolState p;
  int32_t st = pool_state(refcount, num_pages, row_pages, row_num_pages, last_page_len, num_rows, row_capacity, 1,
                          status_dev, &p);
  if (st != PL_OK) return st;
  if (num_released < 0 || (rows == nullptr && num_released > 0)) return PL_ERR_INVALID_ARGUMENT;
  if (num_released == 0) return PL_OK;
  return pl_host::launch_pdl(pl::page_release_kernel, dim3(num_released), dim3(256), 0, stream, p, rows,
                             (int)num_released);
}

extern "C" int32_t pl_page_reserve(int32_t *refcount, int64_t num_pages, int32_t *row_pages, int32_t *row_num_pages,
                                   int32_t *last_page_len, int32_t num_rows, int32_t row_capacity, int32_t page_size,
                                   const int32_t *tok_indptr, int32_t total_tokens, int32_t *slot_page,
                                   int32_t *slot_offset, int32_t *positions_out, int32_t *out_indptr,
                                   int32_t *out_indices, int64_t max_indices, int32_t *status_dev, void *stream) {
  pl::PoolState p;
  int32_t st = pool_state(refcount, num_pages, row_pages, row_num_pages, last_page_len, num_rows, row_capacity,
                          page_size, status_dev, &p);
  if (st != PL_OK) return st;
  if (tok_indptr == nullptr || total_tokens < 0 || max_indices < 0 ||
      (total_tokens > 0 && (slot_page == nullptr || slot_offset == nullptr)))
    return PL_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return total_tokens == 0 ? PL_OK : PL_ERR_INVALID_ARGUMENT;
  return launch_pool(pl::page_reserve_kernel<1>, pl::page_reserve_kernel<pl::kPoolCtas>, p, stream, tok_indptr,
                     (int)total_tokens, slot_page, slot_offset, positions_out, out_indptr, out_indices, max_indices);
}

extern "C" int64_t pl_page_fork_workspace_bytes(int32_t num_forks) {
  return num_forks < 0 ? 0 : 16 + (int64_t)num_forks * (int64_t)sizeof(pl::PageJob);
}

extern "C" int32_t pl_page_fork(void *pool, int64_t layer_stride_bytes, int32_t num_layers, int64_t token_bytes,
                                int32_t *refcount, int64_t num_pages, int32_t *row_pages, int32_t *row_num_pages,
                                int32_t *last_page_len, int32_t num_rows, int32_t row_capacity, int32_t page_size,
                                const int32_t *src_rows, const int32_t *dst_rows, int32_t num_forks, void *workspace,
                                int64_t workspace_bytes, int32_t *status_dev, void *stream) {
  pl::PoolState p;
  int32_t st = pool_state(refcount, num_pages, row_pages, row_num_pages, last_page_len, num_rows, row_capacity,
                          page_size, status_dev, &p);
  if (st != PL_OK) return st;
  pl::CopyArgs c;
  st = copy_args(pool, layer_stride_bytes, num_layers, token_bytes, p, &c);
  if (st != PL_OK) return st;
  if (num_forks < 0 || num_forks > num_rows || (num_forks > 0 && (src_rows == nullptr || dst_rows == nullptr)))
    return PL_ERR_INVALID_ARGUMENT;
  if (num_forks == 0) return PL_OK;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < pl_page_fork_workspace_bytes(num_forks))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  int32_t* count = static_cast<int32_t*>(workspace);
  pl::PageJob* jobs = reinterpret_cast<pl::PageJob*>(count + 4);
  st = launch_pool(pl::page_fork_kernel<1>, pl::page_fork_kernel<pl::kPoolCtas>, p, stream, src_rows, dst_rows,
                   (int)num_forks, count, jobs);
  if (st != PL_OK) return st;
  c.job_count = count;
  c.jobs = jobs;
  return launch_copy(c, num_forks, stream);
}

extern "C" int64_t pl_cache_compact_workspace_bytes(int32_t num_rows, int32_t row_capacity) {
  if (num_rows < 0 || row_capacity < 0) return 0;
  const int64_t n = (int64_t)num_rows * row_capacity;
  return 16 + align16(8 * (int64_t)num_rows) + align16(4 * n) + n * (int64_t)sizeof(pl::PageJob);
}

extern "C" int32_t pl_cache_compact(void *pool, int64_t layer_stride_bytes, int32_t num_layers, int64_t token_bytes,
                                    int32_t *refcount, int64_t num_pages, int32_t *row_pages, int32_t *row_num_pages,
                                    int32_t *last_page_len, int32_t num_rows, int32_t row_capacity, int32_t page_size,
                                    const int32_t *keep_from, const int32_t *keep, int64_t keep_stride,
                                    const int32_t *keep_count, int32_t max_keep, void *workspace,
                                    int64_t workspace_bytes, int32_t *status_dev, void *stream) {
  pl::PoolState p;
  int32_t st = pool_state(refcount, num_pages, row_pages, row_num_pages, last_page_len, num_rows, row_capacity,
                          page_size, status_dev, &p);
  if (st != PL_OK) return st;
  pl::CopyArgs c;
  st = copy_args(pool, layer_stride_bytes, num_layers, token_bytes, p, &c);
  if (st != PL_OK) return st;
  if (keep_from == nullptr || keep_count == nullptr || max_keep < 0 || keep_stride < max_keep ||
      (keep == nullptr && max_keep > 0))
    return PL_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return PL_OK;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < pl_cache_compact_workspace_bytes(num_rows, row_capacity))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  int32_t* count = static_cast<int32_t*>(workspace);
  int2* src_range = reinterpret_cast<int2*>(count + 4);
  int32_t* old_pages = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(src_range) + align16(8 * (int64_t)num_rows));
  const int64_t n = (int64_t)num_rows * row_capacity;
  pl::PageJob* jobs = reinterpret_cast<pl::PageJob*>(reinterpret_cast<char*>(old_pages) + align16(4 * n));
  st = launch_pool(pl::page_compact_kernel<1>, pl::page_compact_kernel<pl::kPoolCtas>, p, stream, keep_from, keep,
                   keep_stride, keep_count, (int)max_keep, count, old_pages, src_range, jobs);
  if (st != PL_OK) return st;
  c.job_count = count;
  c.jobs = jobs;
  c.old_pages = old_pages;
  c.src_range = src_range;
  c.keep_from = keep_from;
  c.keep = keep;
  c.keep_stride = keep_stride;
  return launch_copy(c, n, stream);
}
