// Attention for a tree of drafted tokens over the paged KV cache, with the
// tree's ancestor mask and the greedy acceptance of a path.
//
// Request b has n_b query tokens (its drafted tree); their K/V are the last
// n_b of its kv_len_b cached positions.  Token i sees the whole context
// (positions below kv_len_b - n_b) and the drafted tokens whose bit is set
// in its mask row:
//   o_i = sum_t p_t v_t / l,  p_t = 2^(s_t - m),  s_t = q_i.k_t * sm_scale * log2(e)
// over the seen positions t; lse_i = ln 2 * (m + log2 l).  A row that sees
// nothing gives o = 0 and lse = -inf.
//
// A work item is (request, kv head, row tile): 128 * NT tensor-core rows,
// row R = token * group + head of the group, so all rows that read one K/V
// tile (128 positions) sit in one CTA.  The items' tiles form one line
// (request, kv head, row tile, position) that is cut into equal pieces, one
// per CTA (one CTA per SM), so ragged contexts fill the device; a CTA takes
// the one or few item segments of its piece in turn.  A segment that covers
// its item writes the output; the others leave (O, m, l) in the workspace
// and tree_merge_kernel joins them.  Per CTA:
//   8 * NT warps  softmax, two threads per row (half of the tile's positions
//                 each): scores from TMEM, mask, online softmax (log2
//                 domain), P into the scores' TMEM columns as the A operand;
//   K, V          a TMA producer each, K_0, V_0, K_1, ... through one ring;
//   MMA           one lane issues tcgen05.mma: S = Q.K^T into TMEM, O += P.V.
// P is rounded to bf16, as the tensor core's operand (each p by at most 2^-8
// of itself).  One row tile: O is divided by the sum of the rounded values, so
// that a row of few positions is nearly exact (of one: exact) and the error
// of a long one stays about that of the output's own rounding; lse takes the
// sum of the fp32 values.  Two row tiles have no registers for a second sum
// (8 requests of 64 tokens at 32768 positions 750 -> 790 us) and divide by
// that one.  P as two bf16 values, rounded and remainder, would leave the
// output's rounding alone and takes 5 to 18 % more time (16 requests of 20
// tokens 209 -> 225 us, the 8 above 745 -> 880).
// The maximum that p and the sums are relative to may lag by 2^8, so O is
// rescaled in TMEM only when a row's maximum grows past that, which is rare.
// It lies within 2 of a maximum whatever the scores' size (kTreeNearMax).
// Waits are bounded: on expiry the kernel records PL_ERR_TIMEOUT, drains its
// copies and returns.
//
// Few rows read the cache once and are bound by HBM: 16 requests of 20 tokens
// at 8000 positions (32 / 8 heads of 128) take 210 us in two layers, 5.0 TB/s;
// 89 us of a layer are this kernel, where a plain copy of the bytes takes 81.
// Many rows are bound by the chain maximum -> its exchange -> exponentials ->
// P.V -> next scores of each of two row tiles in turn: 8 requests of 64 tokens
// at 32768 positions take 737 us in two layers, 747 TFLOP/s (660 us before the
// power limit lowers the clock from 1.8 to 1.6 GHz).  The prefill kernel, which
// does not wait for the maximum, does the same products at 998 TFLOP/s.
#include "pl_common.cuh"

namespace pl {

constexpr int kTreeM = 128;              // rows of one tile
constexpr int kTreeN = 128;              // positions of one K/V tile
constexpr float kTreeSlack = 8.0f;       // log2 growth of a row's maximum that is tolerated before O is rescaled
// The two threads of a row tell each other their maxima in bf16, one word in
// all, which shared memory has room for.  Below this size that is off by at
// most 2; from here on the row takes the fp32 maxima, in three more barriers.
constexpr float kTreeNearMax = 1024.0f;
// From this size on the fp32 product score * scale is itself off by more than
// 2 from the exact one that a fused multiply-add takes: the scores are scaled
// before the maximum is subtracted, so that the highest gives p = 1.
constexpr float kTreeScaledMax = 67108864.0f;
// What a warp that gave up tells in place of its maximum (a NaN that no
// rounding gives): its partner does not go on to the fp32 exchange.
constexpr uint16_t kTreeGaveUp = 0xffff;
// Places on the line that an item takes beside its tiles: its look-up, first
// scores, masked tiles and epilogue take a CTA about 6300 cycles, a tile 2340.
// us with 0, 1, 2, 3, 4 places: 12 requests of 5-33 tokens at 300-4100
// positions, 32 kv heads, two layers 213, 197, 187, 185, 186; 32 of 1-40
// tokens at 100-9000, 8 kv heads 184, 154, 158, 145, 143-159; 24 of 40-90
// tokens 337, 308, 278, 251, 245; requests of equal length do not change.
constexpr int kTreeItemCost = 3;
// Places of the line: positions on it, and sums of two, are 32-bit.
constexpr uint32_t kTreeMostPlaces = 1u << 30;
constexpr int kTreeMaxTokens = 1024;     // drafted tokens of one request (tree_mask / tree_accept)

struct TreeArgs {
  const bf16* q;
  const bf16* kv;  // the pool the tensor map covers (read for inf / NaN elements of V only)
  int64_t q_stride_t, q_stride_h;
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_last;
  const uint32_t* mask;  // [total_q][words]
  int64_t mask_stride;
  int64_t num_pages, total_pages;
  int32_t words, batch, total_q, num_qo_heads, num_kv_heads, group, page_size, min_split, ctas;
  float scale_log2;
  bf16* out;
  int64_t out_stride_t, out_stride_h;
  float* lse;      // optional [total_q, Hq], natural log
  float* part_o;   // [2 * ctas][128 * NT][D]
  float* part_ml;  // [2 * ctas][3][128 * NT]: m, l, the sum of the rounded p
  int32_t* status;
};

// Segments between the V producer, which looks them up, and the softmax
// warps: the ring of K/V tiles keeps the producer at most 3 tiles, hence 4
// segments, ahead.
constexpr int kTreeSegs = 8;
// One segment of an item: K/V tiles [j0, j1).
struct TreeSeg {
  int q0, n, kv_begin, n_pages, kv_len, kvh, rt, j0, j1, whole;
};

template <int D, int NT>
struct TreeCfg {
  static constexpr int kSoftmaxThreads = 256 * NT;  // two per row
  // Softmax warps first, then the K producer, the MMA and the V producer
  // warp; an idle warp completes the last warpgroup where registers are
  // dealt anew.
  static constexpr int kProducerWarp = 8 * NT, kMmaWarp = 8 * NT + 1, kProducer2Warp = 8 * NT + 2;  // K, -, V
  static constexpr int kThreads = NT == 2 ? 640 : 96 + kSoftmaxThreads;
  // NT = 2: 20 warps are launched with 96 registers a thread (5 warps per
  // scheduler); the softmax threads (4 warpgroups) take 104, the rest 64:
  // 512 * 104 + 128 * 64 = 640 * 96.  The host takes one row tile when the
  // kernel does not start with 96.
  static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 64;
  static constexpr int kRows = kTreeM * NT;
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = kTreeM * 128;
  static constexpr int kQBytes = kChunks * kChunkBytes;
  static constexpr int kKVBytes = kChunks * kChunkBytes;
  static constexpr int kSlots = 7 - NT;  // fills the shared memory at D = 128
  static constexpr int kQOff = 0;
  static constexpr int kSlotOff = kQOff + NT * kQBytes;
  // Words shared by a row's two threads.  One row tile: two sets in turn,
  // since a thread may be a tile ahead of its partner's read.
  static constexpr int kPairSets = NT == 1 ? 2 : 1;
  static constexpr int kPairOff = kSlotOff + kSlots * kKVBytes;  // [sets][NT][128]
  static constexpr int kBarOff = kPairOff + kPairSets * kRows * 4;
  static constexpr int kNumBars = 2 * kSlots + 8 + 1 + kTreeSegs;  // full empty | s[2] p[2] o[2] q[2] | fin | seg[]
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;  // tmem slot, flags, range, any_bad, segments
  static constexpr int kSmemBytes = 1024 + kMiscOff + 64 + kTreeSegs * (int)sizeof(TreeSeg);
  // Scores take 128 columns at 128 * buf (P in their place), O_x at 256 +
  // 128 x.  One row tile: its scores alternate between two buffers, so that
  // the next tile's are computed during this one's softmax.
  static constexpr int kTmemCols = 512;
  __host__ __device__ static constexpr int buf(int x, int t) { return NT == 1 ? (t & 1) : x; }
  __host__ __device__ static constexpr int phase(int t) { return NT == 1 ? (t >> 1) & 1 : t & 1; }
  static_assert(kSmemBytes <= 232448, "tree tiles exceed the shared-memory limit");
};

// Byte offset of 16-byte unit `u` of row `r` in a 128B-swizzled K-major chunk.
__device__ __forceinline__ uint32_t tr_swz(int r, int u) { return r * 128 + ((u ^ (r & 7)) << 4); }
// 2^x on the multi-function unit (PTX ex2.approx, flush-to-zero); x = -inf gives 0.
__device__ __forceinline__ float tr_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sizes of one request: query tokens, cached tokens, row tiles, K/V tiles.
struct TreeReq {
  int q0, n, kv_begin, n_pages, kv_len, rts, ntiles;
  __device__ __forceinline__ void load(const TreeArgs& a, int b, int rows) {
    q0 = a.qo_indptr[b];
    const int q1 = a.qo_indptr[b + 1];
    const bool ok = q0 >= 0 && q1 >= q0 && q1 <= a.total_q;
    n = ok ? q1 - q0 : 0;
    // a table that leaves [0, total_pages), or has 2^31 positions, counts as
    // empty (and is reported)
    kv_begin = a.kv_indptr[b];
    const int kv_end = a.kv_indptr[b + 1];
    n_pages = kv_begin >= 0 && kv_end >= kv_begin && kv_end <= a.total_pages ? kv_end - kv_begin : 0;
    if ((int64_t)n_pages * a.page_size > 0x7FFFFFFF) n_pages = 0;
    int last = a.kv_last[b];
    last = last < 0 ? 0 : (last > a.page_size ? a.page_size : last);
    kv_len = n_pages > 0 ? (n_pages - 1) * a.page_size + last : 0;
    rts = (int)(((int64_t)n * a.group + rows - 1) / rows);
    ntiles = max(1, (kv_len + kTreeN - 1) / kTreeN);  // an empty context still writes its zero rows
  }
  // length of an item on the line: its tiles and what it costs besides
  __device__ __forceinline__ int span() const { return ntiles + kTreeItemCost; }
  // of the request (kTreeMostPlaces bounds the total of all requests)
  __device__ __forceinline__ int work(int hkv) const { return rts * hkv * span(); }
  // the same, or kTreeMostPlaces + 1 where it is more than that
  __device__ __forceinline__ uint32_t places(int hkv) const {
    return (uint32_t)min((int64_t)rts * hkv * span(), (int64_t)kTreeMostPlaces + 1);
  }
};

// Inclusive prefix sum over a warp.
__device__ __forceinline__ int tree_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Sums of places stay at kTreeMostPlaces + 1 from there on.
__device__ __forceinline__ uint32_t tree_add(uint32_t a, uint32_t b) { return min(a + b, kTreeMostPlaces + 1); }
__device__ __forceinline__ uint32_t tree_add_warp(uint32_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = tree_add(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Length of the line (one warp), 0 when it has more than kTreeMostPlaces (more
// than hours of work, or a qo_indptr that goes back and names tokens often).
__device__ __forceinline__ int tree_total(const TreeArgs& a, int rows) {
  uint32_t t = 0;
  for (int b = threadIdx.x & 31; b < a.batch; b += 32) {
    TreeReq r;
    r.load(a, b, rows);
    t = tree_add(t, r.places(a.num_kv_heads));
  }
  t = tree_add_warp(t);
  if (t <= kTreeMostPlaces) return (int)t;
  if (blockIdx.x == 0) set_status(a.status, PL_ERR_UNSUPPORTED);
  return 0;
}

// Its part of a CTA.
__device__ __forceinline__ int tree_share(int total, int ctas) { return max(1, (total + ctas - 1) / ctas); }

// The requests that hold places w0 and w1 of the line (batch: past the end)
// and where they begin.  A cut in front of an item's second tile, or inside an
// item of at most min_split tiles, moves to the item's start, so short items
// are never split (and never merged).  One warp.
struct TreeAt {
  int b, base, w;
};
__device__ __forceinline__ void tree_locate(const TreeArgs& a, int rows, TreeAt& at0, TreeAt& at1) {
  const int lane = threadIdx.x & 31;
  TreeAt* at[2] = {&at0, &at1};
  int base = 0;
  at0.b = at1.b = a.batch;
  for (int b0 = 0; b0 < a.batch && at1.b == a.batch; b0 += 32) {
    TreeReq r;
    int n = 0;
    r.ntiles = 1;  // lanes past the batch
    if (b0 + lane < a.batch) {
      r.load(a, b0 + lane, rows);
      n = r.work(a.num_kv_heads);
    }
    const int inc = base + tree_scan(n);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t hit = __ballot_sync(0xffffffffu, n > 0 && at[i]->w < inc);
      if (at[i]->b < a.batch || hit == 0) continue;
      const int l = __ffs(hit) - 1;
      at[i]->b = b0 + l;
      at[i]->base = __shfl_sync(0xffffffffu, inc - n, l);
      const int nt = __shfl_sync(0xffffffffu, r.ntiles, l);
      const int off = (at[i]->w - at[i]->base) % (nt + kTreeItemCost);
      if (nt <= a.min_split || off <= kTreeItemCost) at[i]->w -= off;
    }
    base = __shfl_sync(0xffffffffu, inc, 31);
  }
}

// Walks the item segments of the range [w, w_end) of the line.
struct TreeIter {
  int b, w, w_end, base;  // base: where request b begins
  __device__ __forceinline__ bool more() const { return w < w_end; }
  __device__ __forceinline__ bool next(const TreeArgs& a, int rows, TreeSeg& s) {
    if (w >= w_end) return false;
    TreeReq r;
    r.load(a, b, rows);
    while (w - base >= r.work(a.num_kv_heads)) {
      base += r.work(a.num_kv_heads);
      ++b;
      r.load(a, b, rows);
    }
    const int item = (w - base) / r.span();
    const int off = w - base - item * r.span();
    const int end = min(off + (w_end - w), r.span());
    s.q0 = r.q0;
    s.n = r.n;
    s.kv_begin = r.kv_begin;
    s.n_pages = r.n_pages;
    s.kv_len = r.kv_len;
    s.j0 = max(0, off - kTreeItemCost);
    s.j1 = end - kTreeItemCost;
    s.rt = item % r.rts;
    s.kvh = item / r.rts;
    s.whole = s.j0 == 0 && s.j1 == r.ntiles;
    w += end - off;
    return true;
  }
};

// Bits of a mask row from bit `off` on (off >= 0), zero past the row's words.
__device__ __forceinline__ uint32_t tree_bits(const uint32_t* row, int words, int off) {
  const int i = off >> 5, s = off & 31;
  const uint32_t lo = i < words ? row[i] : 0u;
  const uint32_t hi = i + 1 < words ? row[i + 1] : 0u;
  return __funnelshift_r(lo, hi, s);
}

// Wait for a phase of `bar`; false when it ran out or the CTA gave up (looked
// at only while polling, so a wait that is met costs one poll).
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int32_t* flags) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long c0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0 && (flags[0] != 0 || clock64() - c0 > kWaitTimeoutCycles)) return false;
  }
}
// Wait of a whole warp: one lane polls (many pollers of one barrier slow all
// shared-memory traffic).
__device__ __forceinline__ bool tree_warp_wait(uint64_t* bar, uint32_t parity, volatile int32_t* flags) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = tree_wait(bar, parity, flags);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// Arrival of a whole warp: its tensor-memory and shared-memory accesses are
// ordered before the one lane's arrive.
__device__ __forceinline__ void tree_warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

template <int D, int NT>
__global__ void __launch_bounds__(TreeCfg<D, NT>::kThreads, 1)
    paged_tree_kernel(const __grid_constant__ CUtensorMap kv_map, const TreeArgs a) {
  using C = TreeCfg<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* full = bars;
  uint64_t* empty = bars + C::kSlots;
  uint64_t* sready = bars + 2 * C::kSlots;  // [2] scores of a tile in buffer [i]
  uint64_t* pready = sready + 2;            // [2] P in buffer [i] (8 warps)
  uint64_t* odone = sready + 4;             // [2] P.V of a tile from buffer [i] (two row tiles: P_x.V of a segment) complete
  uint64_t* qready = sready + 6;            // [2] Q_x of a segment staged (8 warps)
  uint64_t* fin = sready + 8;
  uint64_t* dready = sready + 9;            // [kTreeSegs] segment looked up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
  volatile int32_t* flags = reinterpret_cast<volatile int32_t*>(smem + C::kMiscOff + 16);  // abort, K and V tiles issued
  volatile int32_t* range = reinterpret_cast<volatile int32_t*>(smem + C::kMiscOff + 32);  // b, w, w_end, base
  uint32_t* any_bad = reinterpret_cast<uint32_t*>(smem + C::kMiscOff + 48);  // a drafted V held inf or NaN
  TreeSeg* segs = reinterpret_cast<TreeSeg*>(smem + C::kMiscOff + 64);       // [kTreeSegs], j0 < 0: the end

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sready[x], 1);
      mbar_init(&pready[x], 8);
      mbar_init(&odone[x], 1);
      mbar_init(&qready[x], 8);
    }
    mbar_init(fin, 1);
    for (int i = 0; i < kTreeSegs; ++i) mbar_init(&dready[i], 1);
    flags[0] = flags[1] = flags[2] = 0;
    any_bad[0] = 0;
    fence_barrier_init();
  }
  if (warp == C::kProducerWarp) {
    if (lane == 0) prefetch_tensormap(&kv_map);
    pdl_wait();
    const int total = tree_total(a, C::kRows), share = tree_share(total, a.ctas);
    TreeAt at0, at1;
    at0.w = (int)min((int64_t)total, (int64_t)blockIdx.x * share);
    at1.w = min(total, at0.w + share);
    tree_locate(a, C::kRows, at0, at1);
    if (lane == 0) {
      range[0] = at0.b;
      range[1] = at0.w;
      range[2] = at1.w;
      range[3] = at0.base;
    }
  } else if (warp == C::kMmaWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // after this wait a dependent grid may read the same tables: it is not
  // released before every CTA has seen them complete
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x == 0 && warp == C::kProducerWarp)  // arguments that no launch can check on the host
    for (int b = lane; b < a.batch; b += 32) {
      TreeReq r;
      r.load(a, b, C::kRows);
      if (r.n != a.qo_indptr[b + 1] - r.q0 || r.n_pages != a.kv_indptr[b + 1] - r.kv_begin || r.n > 32 * a.words ||
          r.n > r.kv_len)
        set_status(a.status, PL_ERR_INVALID_ARGUMENT);
    }
  const uint32_t tmem = *tmem_slot;
  TreeIter it{range[0], range[1], range[2], range[3]};  // may be empty: nothing is loaded then
  const int PS = a.page_size;

  if (warp == C::kProducerWarp || warp == C::kProducer2Warp) {
    if constexpr (NT == 2) reg_dealloc<C::kOtherRegs>();
    // ------------------------------------------------------------ producers
    // One warp brings the K tiles, one the V tiles (ring item 2 t + kv): a
    // page's box costs ~65 cycles of issue, 32 boxes a tile at 16-token
    // pages, which one warp alone could not issue as fast as they arrive.
    const int kv = warp == C::kProducerWarp ? 0 : 1;
    const int ppt = kTreeN / PS;
    const int boxes = ppt * C::kChunks;  // <= 16
    const int p = lane / C::kChunks, hh = lane % C::kChunks;
    int t = 0;
    bool go = true;
    TreeSeg sg;
    for (int seg = 0;; ++seg) {
      // the end is published after a timeout too: the softmax warps rely on it
      const bool some = go && it.next(a, C::kRows, sg);
      if (kv == 1 && lane == 0) {
        segs[seg % kTreeSegs] = sg;
        if (!some) segs[seg % kTreeSegs].j0 = -1;
        mbar_arrive(&dready[seg % kTreeSegs]);
      }
      if (!some) break;
      // This lane's page of tile j (-1: past the row's pages), read two tiles ahead.
      auto page = [&](int j) {
        return lane < boxes && j < sg.j1 && j * ppt + p < sg.n_pages ? a.kv_indices[sg.kv_begin + j * ppt + p] : -1;
      };
      int32_t pid = page(sg.j0), pid1 = page(sg.j0 + 1);
      for (int j = sg.j0; j < sg.j1; ++j, ++t) {
        const int32_t pid2 = page(j + 2);
        const int i = 2 * t + kv, s = i % C::kSlots;
        if (i >= C::kSlots && !tree_warp_wait(&empty[s], ((i / C::kSlots) - 1) & 1, flags)) {
          if (lane == 0) set_status(a.status, PL_ERR_TIMEOUT);
          flags[0] = 1;
          go = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[s], C::kKVBytes);
        __syncwarp();
        if (lane < boxes) {
          const bool in = pid >= 0 && (int64_t)pid < a.num_pages;
          if (!in && j * ppt + p < sg.n_pages) set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
          uint8_t* dst = smem + C::kSlotOff + s * C::kKVBytes + hh * C::kChunkBytes + p * PS * 128;
          // out of range: the copy writes zeros
          tma_load_4d(dst, &kv_map, hh * 64, sg.kvh, 0, in ? 2 * pid + kv : (int32_t)(2 * a.num_pages), &full[s]);
        }
        pid = pid1;
        pid1 = pid2;
      }
    }
    if (lane == 0) flags[1 + kv] = t;
  } else if (warp == C::kMmaWarp) {
    if constexpr (NT == 2) reg_dealloc<C::kOtherRegs>();
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(kTreeM, kTreeN);
      constexpr uint32_t idesc_o = umma_idesc_bf16(kTreeM, D) | (1u << 16);  // B (V) MN-major
      auto wait_item = [&](int item) -> bool {
        return tree_wait(&full[item % C::kSlots], (item / C::kSlots) & 1, flags);
      };
      auto issue_s = [&](int x, int t) {
        const uint32_t qb = smem_u32(smem + C::kQOff + x * C::kQBytes);
        const uint32_t kb = smem_u32(smem + C::kSlotOff + ((2 * t) % C::kSlots) * C::kKVBytes);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem + (uint32_t)(C::buf(x, t) * kTreeN), umma_desc_k_sw128(qb + c * C::kChunkBytes + 32 * k),
                      umma_desc_k_sw128(kb + c * C::kChunkBytes + 32 * k), idesc_s, (c | k) ? 1u : 0u);
        umma_commit(&sready[C::buf(x, t)]);
      };
      auto issue_pv = [&](int x, int t, bool first) {
        const uint32_t vb = smem_u32(smem + C::kSlotOff + ((2 * t + 1) % C::kSlots) * C::kKVBytes);
#pragma unroll
        for (int kk = 0; kk < kTreeN / 16; ++kk)
          // P of positions 0..63 starts at S_x's first column, of 64..127 at its 64th
          umma_bf16_ts(tmem + (uint32_t)(256 + x * 128),
                       tmem + (uint32_t)(C::buf(x, t) * kTreeN + (kk >> 2) * 64 + (kk & 3) * 8),
                       umma_desc_mn_sw128(vb + kk * 16 * 128, C::kChunkBytes, 1024), idesc_o,
                       (!first || kk > 0) ? 1u : 0u);
      };
      // One run over all tiles of the CTA: the first scores of a segment are
      // issued while the last tile of the segment before is worked on.
      bool ok = true;
      TreeSeg sg;
      int seg = 0, j = 0;
      bool more = it.next(a, C::kRows, sg);
      if (more) {
        j = sg.j0;
        for (int x = 0; x < NT; ++x) ok = ok && tree_wait(&qready[x], 0, flags);
        ok = ok && wait_item(0);
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < NT; ++x) issue_s(x, 0);
          umma_commit(&empty[0]);
        }
      }
      for (int t = 0; ok && more; ++t) {
        const bool last = j + 1 == sg.j1;  // tile of the segment
        more = !last || it.more();         // tiles in this CTA
        // K of the next tile and V of this one are waited for in front of
        // P, whose arrival starts the products
        if (more) ok = wait_item(2 * t + 2);
        if (NT == 1 && more) {  // the next scores are computed during this tile's softmax
          if (last) ok = ok && tree_wait(&qready[0], (seg + 1) & 1, flags);
          if (!ok) break;
          tc_fence_after();
          issue_s(0, t + 1);
          umma_commit(&empty[(2 * t + 2) % C::kSlots]);
        }
        ok = ok && wait_item(2 * t + 1);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          ok = ok && tree_wait(&pready[C::buf(x, t)], C::phase(t), flags);
          if (!ok) break;
          tc_fence_after();
          issue_pv(x, t, j == sg.j0);
          if (NT == 1 || last) umma_commit(&odone[NT == 1 ? t & 1 : x]);
          if (x == NT - 1) umma_commit(&empty[(2 * t + 1) % C::kSlots]);
          if (NT == 2 && more) {
            if (last) {
              ok = tree_wait(&qready[x], (seg + 1) & 1, flags);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(x, t + 1);
            if (x == NT - 1) umma_commit(&empty[(2 * t + 2) % C::kSlots]);
          }
        }
        ++j;
        if (last && more) {
          (void)it.next(a, C::kRows, sg);
          ++seg;
          j = sg.j0;
        }
      }
      if (!ok) {
        set_status(a.status, PL_ERR_TIMEOUT);
        flags[0] = 1;
      }
      umma_commit(fin);
      if (!mbar_wait(fin, 0)) set_status(a.status, PL_ERR_TIMEOUT);
    }
  } else if (warp > C::kProducer2Warp) {
    if constexpr (NT == 2) reg_dealloc<C::kOtherRegs>();
  } else {
    if constexpr (NT == 2) reg_alloc<C::kSoftmaxRegs>();
    // -------------------------------------------------- softmax / epilogue
    // Per row tile two groups of four warps; group `half` has the positions
    // 64 half .. 64 half + 63 of every K/V tile, so a row's two threads share
    // its running maximum (through shared memory) and keep a sum each.  A
    // warp whose wait ran out does no further work but still meets the one
    // named barrier of every tile and says so there (kTreeGaveUp), so that no
    // other warp is left in one.
    const int x = warp / 8;
    const int half = (warp / 4) & 1;
    const int quad = warp & 3;
    const int m = 32 * quad + lane;  // row of the tile == TMEM lane
    const uint32_t row_tmem = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t o_tmem = row_tmem + (uint32_t)(256 + x * 128 + half * (D / 2));
    const uint32_t pair_bar = 1 + x * 4 + quad;
    uint32_t* pair0 = reinterpret_cast<uint32_t*>(smem + C::kPairOff) + x * kTreeM + m;
    const float sl2 = a.scale_log2;
    bool ok = true;
    int t = 0;
    // First tile of segment `seg`, -1 past the last.  The producer publishes
    // every segment or, when it gives up, the end, each within a bounded
    // time; all warps wait for that, so they see the same segments.
    auto seg_start = [&](int seg) {
      if (lane == 0)
        for (int i = 0; i < 8 && !mbar_wait(&dready[seg % kTreeSegs], (seg / kTreeSegs) & 1); ++i) {}
      __syncwarp();
      return *const_cast<volatile int*>(&segs[seg % kTreeSegs].j0);
    };
    // this thread's half of its q row of segment `seg` (rows outside are zero)
    auto stage_q = [&](int seg) {
      const volatile TreeSeg& sg = segs[seg % kTreeSegs];
      const int row = sg.rt * C::kRows + x * kTreeM + m, tok = row / a.group;
      const bool row_ok = tok < sg.n;
      const int head = sg.kvh * a.group + row % a.group;
      const bf16* src = a.q + (int64_t)(sg.q0 + tok) * a.q_stride_t + (int64_t)head * a.q_stride_h;
      uint8_t* qs = smem + C::kQOff + x * C::kQBytes;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int u = half * (D / 16) + i;
        const uint4 v = row_ok ? __ldg(reinterpret_cast<const uint4*>(src) + u) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(qs + (u >> 3) * C::kChunkBytes + tr_swz(m, u & 7)) = v;
      }
      fence_proxy_async_smem();
      tree_warp_arrive(&qready[x]);
    };
    if (seg_start(0) >= 0) stage_q(0);
    for (int seg = 0;; ++seg) {
      const int j0 = seg_start(seg);
      if (j0 < 0) break;
      const volatile TreeSeg& sg = segs[seg % kTreeSegs];
      // this thread's row of the request, computed where it is needed
      auto row_of = [&]() { return sg.rt * C::kRows + x * kTreeM + m; };
      // else: rows past the request's, nothing to compute
      const bool warp_ok = (sg.rt * C::kRows + x * kTreeM + 32 * quad) / a.group < sg.n;
      float m_run = -INFINITY, l_run = 0.f, n_run = 0.f;  // sums of p, of p as rounded
      const int j1 = sg.j1;
      // V rows past the last token hold whatever the pool had there, and a
      // drafted token's V may hold inf or NaN that a row which masks the
      // token must not meet (0 * NaN is NaN): the former are cleared, the
      // latter's inf / NaN elements replaced by zero and noted, for the rows
      // that do see them (epilogue).  Tile 0's warps without rows do it, or
      // all of them when each has rows.
      const int quads = min(4, (sg.n * a.group - sg.rt * C::kRows + 31) / 32);
      auto clean_v = [&](int j, int t) {
        const int item = 2 * t + 1;
        if (!tree_warp_wait(&full[item % C::kSlots], (item / C::kSlots) & 1, flags)) return;
        uint8_t* vt = smem + C::kSlotOff + (item % C::kSlots) * C::kKVBytes;
        const int kv_len = sg.kv_len, ctx = kv_len - sg.n;
        const int r0 = max(ctx - j * kTreeN, 0), r_live = min(kTreeN, kv_len - j * kTreeN), units = C::kChunks * 8;
        const int per = quads == 4 ? 4 : 4 - quads;  // warps of each half that do it
        const int at0 = (half * per + (quads == 4 ? quad : quad - quads)) * 32 + lane;
        for (int idx = at0; idx < (kTreeN - r0) * units; idx += 64 * per) {
          const int r = r0 + idx / units, hh = (idx / 8) % C::kChunks, u = idx % 8;
          uint4* at = reinterpret_cast<uint4*>(vt + hh * C::kChunkBytes + r * 128 + u * 16);
          if (r >= r_live) {
            *at = make_uint4(0, 0, 0, 0);
          } else {
            uint4 e = *at;
            uint32_t* w = reinterpret_cast<uint32_t*>(&e);
            bool hit = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((w[k] & 0x7f80u) == 0x7f80u) { w[k] &= 0xffff0000u; hit = true; }
              if ((w[k] & 0x7f800000u) == 0x7f800000u) { w[k] &= 0x0000ffffu; hit = true; }
            }
            if (hit) {
              *at = e;
              atomicOr(any_bad, 1u);
            }
          }
        }
        fence_proxy_async_smem();
      };
      const int first_masked = (sg.kv_len - sg.n) / kTreeN;  // tiles from here on reach the drafted tokens
      for (int j = j0; j < j1; ++j, ++t) {
        const int sb = C::buf(x, t);
        const uint32_t s_tmem = row_tmem + (uint32_t)(sb * kTreeN + 64 * half);
        ok = ok && tree_warp_wait(&sready[sb], C::phase(t), flags);
        // the segment's last scores are there: q makes room for the next one's
        if (ok && j == j1 - 1 && seg_start(seg + 1) >= 0) stage_q(seg + 1);
        bf16* pair_max = reinterpret_cast<bf16*>(pair0 + (C::kPairSets == 2 ? (t & 1) * C::kRows : 0));  // [half]
        const bool masked = j >= first_masked;  // uniform over the CTA
        if (!warp_ok) {
          if (ok && masked && x == 0) clean_v(j, t);
          if (ok) tree_warp_arrive(&pready[sb]);
          continue;
        }
        if (!ok) {
          pair_max[half] = __ushort_as_bfloat16(kTreeGaveUp);
          named_barrier(pair_bar, 64);
          continue;
        }
        tc_fence_after();
        float v[64];
        tmem_ld64(s_tmem, v);
        if (masked) {
          const int kv_len = sg.kv_len, ctx = kv_len - sg.n;  // drafted token i sits at position ctx + i
          const int tok = row_of() / a.group;
          const bool row_ok = tok < sg.n;
          const uint32_t* mrow = a.mask + (int64_t)(sg.q0 + (row_ok ? tok : 0)) * a.mask_stride;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int pos = j * kTreeN + 64 * half + 32 * c;
            const int rel = pos - ctx;  // drafted index of the column group's first position
            uint32_t w = 0;
            if (row_ok) {
              if (rel >= 0)
                w = tree_bits(mrow, a.words, rel);
              else if (rel > -32)
                w = (0xffffffffu >> (32 + rel)) | (tree_bits(mrow, a.words, 0) << (-rel));
              else
                w = 0xffffffffu;
            }
            const int live = kv_len - pos;
            w = live >= 32 ? w : (live <= 0 ? 0u : w & (0xffffffffu >> (32 - live)));
#pragma unroll
            for (int i = 0; i < 32; ++i) v[32 * c + i] = ((w >> i) & 1u) ? v[32 * c + i] : -INFINITY;
          }
        }
        float mx[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(v[k], v[k + 4]);
#pragma unroll
        for (int i = 8; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
        // both threads of the row take the larger of the two maxima, as
        // rounded to bf16: a common reference within 2 of the maximum serves
        const bf16 mine = f2bf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2);
        pair_max[half] = mine;
        named_barrier(pair_bar, 64);
        const uint16_t theirs = *reinterpret_cast<volatile uint16_t*>(&pair_max[half ^ 1]);
        float tmax = fmaxf(bf2f(mine), bf2f(__ushort_as_bfloat16(theirs)));
        float sl = sl2;
        const bool large = fabsf(tmax) >= kTreeNearMax && tmax != -INFINITY && theirs != kTreeGaveUp;
        // (the votes of a row's two warps agree: tmax and m_run are the same)
        if (__builtin_expect(__any_sync(0xffffffffu, tmax > m_run + kTreeSlack || m_run == -INFINITY || large), 0)) {
          if (__builtin_expect(__any_sync(0xffffffffu, large), 0)) {
            volatile float* word = reinterpret_cast<float*>(pair_max);
            float top = v[0];
#pragma unroll
            for (int i = 1; i < 64; ++i) top = fmaxf(top, v[i]);
            top *= sl2;
            named_barrier(pair_bar, 64);  // both have read the rounded maxima
            if (half == 1) *word = top;
            named_barrier(pair_bar, 64);
            if (half == 0) *word = tmax = fmaxf(top, *word);
            named_barrier(pair_bar, 64);
            if (half == 1) tmax = *word;
            if (__any_sync(0xffffffffu, fabsf(tmax) >= kTreeScaledMax && tmax != -INFINITY)) {
#pragma unroll
              for (int i = 0; i < 64; ++i) v[i] *= sl2;
              sl = 1.f;
            }
          }
          const float m_new = fmaxf(m_run, tmax);
          const bool rescale = m_run != -INFINITY && m_new > m_run + kTreeSlack;
          const float alpha = rescale ? tr_exp2(m_run - m_new) : 1.f;
          if (__any_sync(0xffffffffu, rescale)) {
            // O_x of the tiles before has to be complete (two row tiles: it
            // is, S was issued after it)
            if (NT == 1 && !tree_warp_wait(&odone[sb ^ 1], ((t - 1) >> 1) & 1, flags)) ok = false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[16];
              tmem_ld16(o_tmem + 16 * c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16_wait(o_tmem + 16 * c, o);
            }
            l_run *= alpha;
            if constexpr (NT == 1) n_run *= alpha;
          }
          if (rescale || m_run == -INFINITY) m_run = m_new;
        }
        const float nb = m_run == -INFINITY ? 0.f : -m_run;
        const float2 sl2_2 = make_float2(sl, sl), nb_2 = make_float2(nb, nb);
        float2 sm[2], sn[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) sm[k] = sn[k] = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 e = fma_f32x2(make_float2(v[32 * c + i], v[32 * c + i + 1]), sl2_2, nb_2);
            e.x = tr_exp2(e.x);
            e.y = tr_exp2(e.y);
            sm[(i >> 1) & 1] = add_f32x2(sm[(i >> 1) & 1], e);
            pk[i / 2] = pack_bf16x2(e.x, e.y);
            if constexpr (NT == 1) sn[(i >> 1) & 1] = add_f32x2(sn[(i >> 1) & 1], unpack_bf16x2(pk[i / 2]));
          }
          tmem_st16_u32(s_tmem + 16 * c, pk);
        }
        sm[0] = add_f32x2(sm[0], sm[1]);
        l_run += sm[0].x + sm[0].y;
        if constexpr (NT == 1) {
          sn[0] = add_f32x2(sn[0], sn[1]);
          n_run += sn[0].x + sn[0].y;
        }
        tmem_st_wait();
        if (masked && x == 0 && quads == 4) clean_v(j, t);
        tc_fence_before();
        tree_warp_arrive(&pready[sb]);
      }
      // ---- epilogue of the segment: each thread of a row has half of its channels
      ok = ok && tree_warp_wait(&odone[NT == 1 ? (t - 1) & 1 : x], (NT == 1 ? (t - 1) >> 1 : seg) & 1, flags);
      if (!ok) {
        if (lane == 0) set_status(a.status, PL_ERR_TIMEOUT);
        flags[0] = 1;
      }
      if (!warp_ok) continue;
      tc_fence_after();
      // (the partner's read of the last maxima lies behind its P, hence behind O)
      float* pair_sum = reinterpret_cast<float*>(pair0);
      // half 0 gets the row's l, both halves its n
      if constexpr (NT == 2) n_run = l_run;
      if (half == 1) *pair_sum = l_run;
      named_barrier(pair_bar, 64);
      if (half == 0) l_run += *const_cast<volatile float*>(pair_sum);
      named_barrier(pair_bar, 64);
      if (half == 1) *pair_sum = n_run;
      named_barrier(pair_bar, 64);
      if (half == 0) *pair_sum = n_run += *const_cast<volatile float*>(pair_sum);
      named_barrier(pair_bar, 64);
      n_run = *const_cast<volatile float*>(pair_sum);
      named_barrier(pair_bar, 64);  // read: the next segment's maxima may go there
      if (!ok) continue;
      const int row = row_of(), tok = row / a.group;
      const bool row_ok = tok < sg.n;
      const int head = sg.kvh * a.group + row % a.group;
      const int ctx = sg.kv_len - sg.n, n = sg.n;
      const bool whole = sg.whole != 0;
      // any_bad is final: every P of the segment was waited for by its P.V
      const bool check_bad = *const_cast<volatile uint32_t*>(any_bad) != 0 && j1 * kTreeN > ctx;
      const float inv = n_run == 0.f ? 0.f : 1.f / n_run;
      const int slot = 2 * (int)blockIdx.x + (j0 > 0 ? 0 : 1);
      bf16* dst = a.out + (int64_t)(sg.q0 + tok) * a.out_stride_t + (int64_t)head * a.out_stride_h + half * (D / 2);
      float* pdst = a.part_o + ((int64_t)slot * C::kRows + x * kTreeM + m) * D + half * (D / 2);
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        float v[32];
        tmem_ld32(o_tmem + 32 * c, v);
        if (check_bad && row_ok) {
          // the inf / NaN elements of the seen drafted tokens of this segment
          const uint32_t* mrow = a.mask + (int64_t)(sg.q0 + tok) * a.mask_stride;
          const int64_t tstride = (int64_t)a.num_kv_heads * D;
          for (int jj = max(0, max(-ctx, j0 * kTreeN - ctx)); jj < n && ctx + jj < j1 * kTreeN; ++jj) {
            if (!(tree_bits(mrow, a.words, jj) & 1u)) continue;
            const int pos = ctx + jj;
            const int32_t pid = a.kv_indices[sg.kv_begin + pos / PS];
            if (pid < 0 || (int64_t)pid >= a.num_pages) continue;
            const bf16* vrow = a.kv + (((int64_t)pid * 2 + 1) * PS + pos % PS) * tstride + (int64_t)sg.kvh * D +
                               half * (D / 2) + 32 * c;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e = bf2f(vrow[i]);
              if (!isfinite(e)) v[i] += e;
            }
          }
        }
        if (row_ok) {
          if (whole) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) pk[i / 2] = pack_bf16x2(v[i] * inv, v[i + 1] * inv);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              reinterpret_cast<uint4*>(dst + 32 * c)[u] =
                  make_uint4(pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]);
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              reinterpret_cast<float4*>(pdst + 32 * c)[u] = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
          }
        }
      }
      if (row_ok && half == 0) {
        if (whole) {
          if (a.lse != nullptr)
            a.lse[(int64_t)(sg.q0 + tok) * a.num_qo_heads + head] =
                l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
        } else {
          float* ml = a.part_ml + (int64_t)slot * 3 * C::kRows + x * kTreeM + m;
          ml[0] = m_run;
          ml[C::kRows] = l_run;
          ml[2 * C::kRows] = n_run;
        }
      }
      tc_fence_before();  // O was read: the next segment's first P.V (issued after its P arrives) may overwrite it
    }
  }

  // ------------------------------------------------------------ teardown
  __syncthreads();
  if (threadIdx.x == 0) {
    // copies that were issued but not waited for (after a timeout) land before the exit
    auto issued = [&](int i) { return (i >> 1) < flags[1 + (i & 1)]; };
    const int most = 2 * max((int)flags[1], (int)flags[2]);
    for (int i = max(0, most - 2 * C::kSlots); i < most; ++i)
      if (issued(i) && !issued(i + C::kSlots)) (void)mbar_wait(&full[i % C::kSlots], (i / C::kSlots) & 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the partial states of the items that several CTAs shared: one warp
// per (query token, head), the states weighted by 2^(m - max m).  A state that
// saw nothing has the sum 0 and is left out; one whose scores are all NaN also
// has no maximum (m = -inf), but a sum of NaN, which reaches the row.  The tables
// are read before the wait for the attention's grid (which lets this one
// start only once they are complete).
constexpr int kMergeThreads = 128;
template <int D>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeArgs a, int rows) {
  const int lane = threadIdx.x & 31;
  const int tok_g = blockIdx.x;
  // the request of this token, where it begins on the line, and the line's length
  int q0 = 0, rts = 0, nt = 0, base = 0, total = 0;
  uint32_t places = 0;
  bool found = false;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    TreeReq r;
    r.n = r.rts = r.ntiles = r.q0 = 0;  // lanes past the batch
    if (b0 + lane < a.batch) r.load(a, b0 + lane, rows);
    const int w = r.work(a.num_kv_heads), inc = total + tree_scan(w);
    const uint32_t hit = __ballot_sync(0xffffffffu, r.q0 <= tok_g && tok_g < r.q0 + r.n);
    if (hit != 0 && !found) {
      const int l = __ffs(hit) - 1;
      found = true;
      q0 = __shfl_sync(0xffffffffu, r.q0, l);
      rts = __shfl_sync(0xffffffffu, r.rts, l);
      nt = __shfl_sync(0xffffffffu, r.ntiles, l);
      base = __shfl_sync(0xffffffffu, inc - w, l);
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
    places = tree_add(places, tree_add_warp(r.places(a.num_kv_heads)));
  }
  if (places > kTreeMostPlaces) found = false;  // refused: there is nothing to join
  const int share = tree_share(total, a.ctas);
  const int head = blockIdx.y * (kMergeThreads / 32) + threadIdx.x / 32;
  const int row = (tok_g - q0) * a.group + head % a.group;
  const int w = base + ((head / a.group) * rts + row / rows) * (nt + kTreeItemCost);
  const int m = row % rows;
  const int ca = (w + kTreeItemCost) / share, cb = (w + kTreeItemCost + nt - 1) / share;
  pdl_wait();
  pdl_launch_dependents();
  if (!found || nt <= a.min_split || head >= a.num_qo_heads || ca == cb) return;  // not split
  auto slot = [&](int c) { return (int64_t)(2 * c + (c == ca ? 1 : 0)); };
  constexpr int E = D / 32;
  float acc[E], L = 0.f, N = 0.f, M = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int c0 = ca; c0 <= cb; c0 += 32) {
    // a lane per state: its maximum and sum; then all lanes add the states up
    float mc = -INFINITY, lc = 0.f, nc = 0.f;
    if (c0 + lane <= cb) {
      const float* ml = a.part_ml + slot(c0 + lane) * 3 * rows + m;
      mc = ml[0];
      lc = ml[rows];
      nc = ml[2 * rows];
    }
    const float m_new = fmaxf(M, warp_max(mc));
    const float old = M == -INFINITY ? 0.f : exp2f(M - m_new);
    const bool any = lc != 0.f;
    const float wt = mc == -INFINITY ? 1.f : exp2f(mc - m_new);
    L = L * old + warp_sum(any ? wt * lc : 0.f);
    N = N * old + warp_sum(any ? wt * nc : 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= old;
    M = m_new;
    const int n = min(32, cb - c0 + 1);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float* o = a.part_o + (slot(c0 + i) * rows + m) * D + lane * E;
      float v[E];
      if constexpr (E == 4) {
        const float4 f = *reinterpret_cast<const float4*>(o);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(o);
        v[0] = f.x; v[1] = f.y;
      }
      const float wi = __shfl_sync(0xffffffffu, wt, i);
      const bool saw = __shfl_sync(0xffffffffu, any ? 1 : 0, i) != 0;  // else the state holds no values
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += saw ? wi * v[e] : 0.f;
    }
  }
  const float inv = N == 0.f ? 0.f : 1.f / N;
  bf16* dst = a.out + (int64_t)tok_g * a.out_stride_t + (int64_t)head * a.out_stride_h + lane * E;
  if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[(int64_t)tok_g * a.num_qo_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// --------------------------------------------------------------- the tree
// Ancestor-or-self bits of every drafted token: thread (token, word) walks
// the parent chain in shared memory and keeps the bits of its word.
__global__ void __launch_bounds__(256)
    tree_mask_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ qo_indptr,
                     const int32_t* __restrict__ base_pos, int total_q, int words, uint32_t* __restrict__ mask,
                     int64_t mask_stride, int32_t* __restrict__ depth, int32_t* __restrict__ positions,
                     int32_t* status) {
  __shared__ int16_t par[kTreeMaxTokens];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int q0 = qo_indptr[b], q1 = qo_indptr[b + 1];
  const int n = q1 - q0;
  if (q0 < 0 || n < 0 || q1 > total_q || n > kTreeMaxTokens || n > 32 * words) {
    if (threadIdx.x == 0) set_status(status, PL_ERR_INVALID_ARGUMENT);
    return;
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int p = parents[q0 + i];
    if (p < -1 || p >= i) {  // not in topological order: the token stands alone
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      p = -1;
    }
    par[i] = (int16_t)p;
  }
  __syncthreads();
  for (int idx = blockIdx.y * blockDim.x + threadIdx.x; idx < n * words; idx += gridDim.y * blockDim.x) {
    const int i = idx / words, w = idx % words;
    uint32_t bits = 0;
    int d = -1;
    for (int j = i; j >= 0; j = par[j], ++d)
      if ((j >> 5) == w) bits |= 1u << (j & 31);
    mask[(int64_t)(q0 + i) * mask_stride + w] = bits;
    if (w == 0) {
      if (depth != nullptr) depth[q0 + i] = d;
      if (positions != nullptr) positions[q0 + i] = (base_pos != nullptr ? base_pos[b] : 0) + d;
    }
  }
}

// Greedy acceptance: a drafted token is taken when it and all its ancestors
// are what the model chose after their parents; the deepest taken token
// (lowest index among equals) ends the kept path.
__global__ void __launch_bounds__(128)
    tree_accept_kernel(const int32_t* __restrict__ parents, const int64_t* __restrict__ tokens,
                       const int64_t* __restrict__ targets, const int32_t* __restrict__ qo_indptr,
                       const int32_t* __restrict__ base_pos, int total_q, int max_keep, int32_t* __restrict__ keep,
                       int64_t keep_stride, int32_t* __restrict__ keep_count, int64_t* __restrict__ next_token,
                       int32_t* status) {
  __shared__ int16_t par[kTreeMaxTokens];
  __shared__ uint8_t good[kTreeMaxTokens];
  __shared__ int best_s;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int q0 = qo_indptr[b], q1 = qo_indptr[b + 1];
  const int n = q1 - q0;
  if (q0 < 0 || n < 0 || q1 > total_q || n > kTreeMaxTokens) {
    if (threadIdx.x == 0) {
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      keep_count[b] = 0;
      next_token[b] = -1;
    }
    return;
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int p = parents[q0 + i];
    bool ok = true;
    if (p < -1 || p >= i) {  // not in topological order: never taken
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      p = -1;
      ok = false;
    }
    par[i] = (int16_t)p;
    good[i] = ok && (p < 0 || tokens[q0 + i] == targets[q0 + p]);
  }
  if (threadIdx.x == 0) best_s = 0;
  __syncthreads();
  // key: depth + 1 of a taken token, then the lower index
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int d = 0, j = i;
    while (j >= 0 && good[j]) {
      ++d;
      j = par[j];
    }
    if (j < 0) atomicMax(&best_s, d * kTreeMaxTokens + (kTreeMaxTokens - 1 - i));
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int key = best_s;
    int count = key / kTreeMaxTokens;
    const int best = kTreeMaxTokens - 1 - key % kTreeMaxTokens;
    if (count > max_keep) {
      set_status(status, PL_ERR_INVALID_ARGUMENT);
      count = 0;
    }
    next_token[b] = count > 0 ? targets[q0 + best] : -1;
    keep_count[b] = count;
    int j = best;
    for (int i = count - 1; i >= 0; --i, j = par[j]) keep[(int64_t)b * keep_stride + i] = base_pos[b] + j;
    best_s = count;
  }
  __syncthreads();
  for (int i = best_s + threadIdx.x; i < max_keep; i += blockDim.x) keep[(int64_t)b * keep_stride + i] = -1;
}

}  // namespace pl

// =================================================================== host
namespace {

// Two row tiles per CTA read a K/V tile once for both, with scores that are
// not computed ahead: taken when the mean request fills an even number of row
// tiles, so that no tile is empty.  16 requests at 8000 positions (32 / 8
// heads of 128), us with one and with two tiles per CTA: 128 rows of a kv
// head 114, 162; 132 rows 189, 165; 256 rows 205, 192; 384 rows 309, 354.
bool tree_two_tiles(int total_q, int batch, int group) {
  const int64_t tile_rows = (int64_t)batch * pl::kTreeM;
  return (((int64_t)total_q * group + tile_rows - 1) / tile_rows) % 2 == 0;
}

// Items of up to this many tiles stay whole, and when all pages together make
// no more, the merge launch is left out.  8 tokens at 600 positions (5 tiles)
// take 15.2 us whole and 15.7 us split; 16 tiles gain 5 us from the split.
constexpr int kTreeMinSplit = 6;

// Whether the kernel for two row tiles starts with the registers that its
// warps' shares add up to.  A compiler that gives it another count leaves the
// wide calls to the form with one row tile, which takes the same arguments.
template <int D>
bool tree_split_adds_up() {
  static const bool ok = [] {
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, pl::paged_tree_kernel<D, 2>) == cudaSuccess &&
           (f.numRegs + 7) / 8 * 8 == pl::TreeCfg<D, 2>::kLaunchRegs;
  }();
  return ok;
}

template <int D, int NT>
int32_t launch_tree(const CUtensorMap& map, const pl::TreeArgs& a, bool merge, void* stream) {
  using C = pl::TreeCfg<D, NT>;
  auto kern = pl::paged_tree_kernel<D, NT>;
  int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (st != PL_OK) return st;
  st = pl_host::launch_pdl(kern, dim3(a.ctas), dim3(C::kThreads), C::kSmemBytes, stream, map, a);
  if (st != PL_OK || !merge) return st;
  constexpr int warps = pl::kMergeThreads / 32;
  return pl_host::launch_pdl(pl::tree_merge_kernel<D>, dim3(a.total_q, (a.num_qo_heads + warps - 1) / warps),
                             dim3(pl::kMergeThreads), 0, stream, a, (int)C::kRows);
}

}  // namespace

extern "C" int64_t pl_tree_workspace_bytes(int32_t batch, int32_t total_q, int32_t num_qo_heads, int32_t num_kv_heads,
                                           int32_t head_dim) {
  if (batch <= 0 || total_q <= 0 || num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads != 0 ||
      head_dim <= 0)
    return 0;
  const int sms = pl_host::sm_count();
  const int64_t rows = pl::kTreeM * (tree_two_tiles(total_q, batch, num_qo_heads / num_kv_heads) ? 2 : 1);
  return 2 * (int64_t)(sms > 0 ? sms : 148) * rows * (head_dim + 3) * 4;
}

extern "C" int32_t pl_paged_tree_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv_cache, int64_t num_pages,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len,
    int64_t total_pages, const int32_t* tree_mask, int64_t mask_stride, int32_t mask_words, int32_t batch,
    int32_t total_q, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float sm_scale,
    void* out, int64_t out_stride_t, int64_t out_stride_h, float* out_lse, void* workspace, int64_t workspace_bytes,
    int32_t* status_dev, void* stream) {
  // what has no entries may be null
  if (kv_cache == nullptr || qo_indptr == nullptr || kv_indptr == nullptr || kv_last_page_len == nullptr ||
      (total_pages > 0 && kv_indices == nullptr) ||
      (total_q > 0 && (q == nullptr || tree_mask == nullptr || out == nullptr)) || batch < 0 || total_q < 0 ||
      num_pages <= 0 || num_pages > 0x3FFFFFFF || total_pages < 0 || mask_words <= 0 || mask_stride < mask_words ||
      num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads != 0 || !(sm_scale > 0.f))
    return PL_ERR_INVALID_ARGUMENT;
  const int group = num_qo_heads / num_kv_heads;
  if (group > pl::kTreeM || (head_dim != 64 && head_dim != 128) ||
      (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) || num_kv_heads > 65535)
    return PL_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(kv_cache) & 15) != 0 || (reinterpret_cast<uintptr_t>(q) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(out) & 15) != 0 || (q_stride_t % 8) != 0 || (q_stride_h % 8) != 0 ||
      (out_stride_t % 8) != 0 || (out_stride_h % 8) != 0)
    return PL_ERR_INVALID_ARGUMENT;
  if (batch == 0 || total_q == 0) return PL_OK;
  // no request has more than total_pages pages: below kTreeMinSplit tiles nothing is split
  const bool merge = total_pages * page_size > (int64_t)kTreeMinSplit * pl::kTreeN;
  if (merge && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
                workspace_bytes < pl_tree_workspace_bytes(batch, total_q, num_qo_heads, num_kv_heads, head_dim)))
    return PL_ERR_WORKSPACE_TOO_SMALL;

  CUtensorMap map;
  int32_t st = pl_host::kv_tensor_map(kv_cache, num_pages, num_kv_heads, head_dim, page_size, &map);
  if (st != PL_OK) return st;
  const int sms = pl_host::sm_count();
  if (sms <= 0) return PL_ERR_NO_DEVICE;

  const bool two = tree_two_tiles(total_q, batch, group) &&
                   (head_dim == 128 ? tree_split_adds_up<128>() : tree_split_adds_up<64>());
  pl::TreeArgs a;
  a.q = static_cast<const pl::bf16*>(q);
  a.kv = static_cast<const pl::bf16*>(kv_cache);
  a.q_stride_t = q_stride_t;
  a.q_stride_h = q_stride_h;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.kv_last = kv_last_page_len;
  a.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  a.mask_stride = mask_stride;
  a.num_pages = num_pages;
  a.total_pages = total_pages;
  a.words = mask_words;
  a.batch = batch;
  a.total_q = total_q;
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.page_size = page_size;
  a.min_split = kTreeMinSplit;
  a.ctas = sms;
  a.scale_log2 = sm_scale * pl::kLog2e;
  a.out = static_cast<pl::bf16*>(out);
  a.out_stride_t = out_stride_t;
  a.out_stride_h = out_stride_h;
  a.lse = out_lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = workspace == nullptr ? nullptr : a.part_o + 2 * (int64_t)sms * pl::kTreeM * (two ? 2 : 1) * head_dim;
  a.status = status_dev;
  if (head_dim == 128) return two ? launch_tree<128, 2>(map, a, merge, stream) : launch_tree<128, 1>(map, a, merge, stream);
  return two ? launch_tree<64, 2>(map, a, merge, stream) : launch_tree<64, 1>(map, a, merge, stream);
}

extern "C" int32_t pl_tree_mask(const int32_t* parents, const int32_t* qo_indptr, const int32_t* base_positions,
                                int32_t batch, int32_t total_q, int32_t mask_words, int32_t* mask, int64_t mask_stride,
                                int32_t* depth, int32_t* positions, int32_t* status_dev, void* stream) {
  if (qo_indptr == nullptr || (total_q > 0 && (parents == nullptr || mask == nullptr)) || batch < 0 ||
      total_q < 0 || mask_words <= 0 ||
      mask_stride < mask_words)
    return PL_ERR_INVALID_ARGUMENT;
  if (batch == 0 || total_q == 0) return PL_OK;
  const int64_t per = ((int64_t)total_q * mask_words + 255) / 256;
  const int gy = (int)(per < 1 ? 1 : (per > 16 ? 16 : per));
  return pl_host::launch_pdl(pl::tree_mask_kernel, dim3(batch, gy), dim3(256), 0, stream, parents, qo_indptr,
                             base_positions, (int)total_q, (int)mask_words, reinterpret_cast<uint32_t*>(mask),
                             mask_stride, depth, positions, status_dev);
}

extern "C" int32_t pl_tree_accept(const int32_t* parents, const int64_t* tokens, const int64_t* targets,
                                  const int32_t* qo_indptr, const int32_t* base_positions, int32_t batch,
                                  int32_t total_q, int32_t max_keep, int32_t* keep, int64_t keep_stride,
                                  int32_t* keep_count, int64_t* next_token, int32_t* status_dev, void* stream) {
  if ((total_q > 0 && (parents == nullptr || tokens == nullptr || targets == nullptr)) || qo_indptr == nullptr ||
      base_positions == nullptr || keep == nullptr || keep_count == nullptr || next_token == nullptr || batch < 0 ||
      total_q < 0 || max_keep <= 0 || keep_stride < max_keep)
    return PL_ERR_INVALID_ARGUMENT;
  if (batch == 0) return PL_OK;
  return pl_host::launch_pdl(pl::tree_accept_kernel, dim3(batch), dim3(128), 0, stream, parents, tokens, targets,
                             qo_indptr, base_positions, (int)total_q, (int)max_keep, keep, keep_stride, keep_count,
                             next_token, status_dev);
}
