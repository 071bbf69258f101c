// Decode attention of one token per row over the bf16 paged cache, cut as one
// line of work (pl_line_decode.cuh): with a sliding window and sinks
// (pl_paged_window_decode), or over the whole context with the attention
// weight of every cached token accumulated (pl_paged_decode_weights).
//
// A CTA walks its piece of the line tile by tile (16 positions of one kv
// head): warp 0 brings K and warp 1 V by TMA (16 positions x 64 channels a
// box, 128B-swizzled, 32 KB an instruction) through a ring that runs on across
// items.  (A warp's instruction takes about 0.4 us beside 0.7 for 32 KB of
// rows: one warp for both, 64 KB at a time, 140 us for 48 windows of 4096
// positions, 32 KB at a time 171.)  Tile i belongs to consumer warp i % 8.
// Positions are the
// rows of S^T = K.Q^T (mma m16n8k16: eight query heads side by side, so a
// group of up to 8 wastes no row) and channels the rows of O^T = V^T.P^T; P
// goes from the one's result layout to the other's operand layout by an 8x8
// transpose in registers.  Exponentials are taken against a reference that
// moves only when a score exceeds it by 2^8, which one vote per tile decides.
// The eight warps' states are joined in shared memory at an item's end.
//
// Bound by HBM: 512 bytes of K and V per position and kv head at head_dim 128
// for 16 x 8 tensor-core columns.  P enters the tensor core as bf16 (at most
// 2^-8 relative a term, as the output's own rounding; over many terms it
// averages out); maxima, sums and O are fp32.
#include <mutex>

#include "pl_line_decode.cuh"

namespace pl {

constexpr int kLineWarps = 8;                          // consumer warps
constexpr int kLineThreads = 32 * (2 + kLineWarps);
constexpr int kLineAccum = 256;                        // positions per block of the accumulation

template <int D, int NT>
struct LineCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = kTile * 128;             // one box
  static constexpr int kTileBytes = kHalves * kHalfBytes;    // K (or V) of a tile
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kBatch = 8 * (128 / D);               // tiles per producer instruction: 32 KB of K or of V
  // Three batches make the ring (48 windows: 126 us, two 130); two where the
  // join of two column blocks takes the room.
  static constexpr int kStages = (NT == 1 ? 3 : 2) * kBatch;  // a multiple of kLineWarps
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPiece = D + 4;                       // floats of a head's piece in the workspace
  static constexpr int kJoinOff = kStages * kStageBytes;     // [warps][kHeads][D], swizzled
  static constexpr int kMlOff = kJoinOff + kLineWarps * kHeads * D * 4;  // [warps][kHeads] (m, l)
  static constexpr int kBarOff = kMlOff + kLineWarps * kHeads * 8;
  static constexpr int kOkOff = kBarOff + 2 * kStages * 8;   // [stages] the tile's page exists
  static constexpr int kFindOff = (kOkOff + kStages * 4 + 15) & ~15;  // 36 int64
  static constexpr int kFlagOff = kFindOff + 36 * 8;
  static constexpr int kSmemBytes = kFlagOff + 16 + 1024;
  static_assert(kStages % kLineWarps == 0, "a stage belongs to one warp");
  static_assert(kSmemBytes <= 232448, "the ring exceeds the shared-memory limit");
};

__device__ __forceinline__ uint32_t line_swz(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

template <int D, int NT, bool kWeights>
__global__ void __launch_bounds__(kLineThreads, 1)
    line_decode_kernel(const __grid_constant__ CUtensorMap kv_map, const LineArgs a) {
  using C = LineCfg<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + C::kStages;
  int32_t* page_ok = reinterpret_cast<int32_t*>(smem + C::kOkOff);
  volatile int32_t* flags = reinterpret_cast<volatile int32_t*>(smem + C::kFlagOff);  // [0] abort, [1] its copy
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 2);  // K's and V's copies
      mbar_init(&empty[s], 1);
    }
    flags[0] = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 64) prefetch_tensormap(&kv_map);
  pdl_launch_dependents();
  pdl_wait();  // q, the page table and the cache come from upstream kernels
  int row0;
  int64_t row_start;
  const LineCut cut =
      line_find<kLineThreads>(a, blockIdx.x, reinterpret_cast<int64_t*>(smem + C::kFindOff), row0, row_start);
  if ((int64_t)blockIdx.x >= cut.ctas) return;  // fewer pieces than CTAs: nothing was started
  const int64_t begin = cut.begin(blockIdx.x), end = cut.begin((int64_t)blockIdx.x + 1);

  if (warp < 2) {
    // ----------------------------------------------------------- producers
    const int kv = warp, hh = lane % C::kHalves;
    int i0 = 0;  // tiles of this CTA so far
    for_each_segment(a, row0, row_start, begin, end, [&](int, const RowSpan& sp, int kvh, int lo, int hi) {
      const int n = hi - lo;
      // page ids of 32 tiles a load, one load ahead: its latency would else bound every batch
      auto entry = [&](int u) { return u < n ? a.indices[sp.begin + sp.tile(lo + u) * kTile / a.page_size] : -1; };
      int32_t now = entry(lane), next = entry(32 + lane);
      for (int u0 = 0; u0 < n; u0 += C::kBatch) {
        if (u0 != 0 && u0 % 32 == 0) {
          now = next;
          next = entry(u0 + 32 + lane);
        }
        const int u = u0 + lane / C::kHalves;
        const bool on = lane < C::kBatch * C::kHalves && u < n;
        const int i = i0 + u, s = i % C::kStages;
        const int32_t pid = __shfl_sync(0xffffffffu, now, u % 32);
        bool ok = true;
        if (on && i >= C::kStages) ok = mbar_wait(&empty[s], ((i / C::kStages) - 1) & 1);
        if (__any_sync(0xffffffffu, !ok || flags[0] != 0)) {
          if (__any_sync(0xffffffffu, !ok) && lane == 0) set_status(a.status, PL_ERR_TIMEOUT);
          flags[0] = 1;
          // the copies in flight land (bounded) before the CTA ends
          const int issued = i0 + u0;
          if (lane == 0)
            for (int j = issued > C::kStages ? issued - C::kStages : 0; j < issued; ++j)
              (void)mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1);
          return false;
        }
        const bool valid = on && pid >= 0 && (int64_t)pid < a.num_pages;
        if (on && hh == 0) {
          if (kv == 0) page_ok[s] = valid;
          if (valid) {
            mbar_arrive_expect_tx(&full[s], C::kTileBytes);
          } else {
            set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
            mbar_arrive(&full[s]);
          }
        }
        __syncwarp();
        if (valid)
          tma_load_4d(smem + s * C::kStageBytes + kv * C::kTileBytes + hh * C::kHalfBytes, &kv_map, hh * 64, kvh,
                      sp.tile(lo + u) * kTile % a.page_size, 2 * pid + kv, &full[s]);
      }
      i0 += n;
      return true;
    });
  } else {
    // ----------------------------------------------------------- consumers
    const int cw = warp - 2, ctid = threadIdx.x - 64;
    const int g = lane >> 2, t = lane & 3;
    float* join = reinterpret_cast<float*>(smem + C::kJoinOff);
    float2* ml = reinterpret_cast<float2*>(smem + C::kMlOff);
    const float sl2 = a.scale_log2;
    int i0 = 0;
    for_each_segment(a, row0, row_start, begin, end, [&](int row, const RowSpan& sp, int kvh, int lo, int hi) {
      // Q as the tensor core's B operand: head g of each block of eight
      uint32_t qb[NT][D / 16][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = 8 * nt + g;
        const bf16* src = a.q + (int64_t)row * a.q_stride_b + (int64_t)(kvh * a.group + h) * a.q_stride_h + 2 * t;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qb[nt][kk][0] = h < a.group ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * kk)) : 0u;
          qb[nt][kk][1] = h < a.group ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * kk + 8)) : 0u;
        }
      }
      float o[NT][D / 16][4];
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
      const int n = hi - lo;
      // tile i of the CTA belongs to warp i % kLineWarps (a stage always to the same one)
      for (int u = (cw - i0 % kLineWarps + kLineWarps) % kLineWarps; u < n; u += kLineWarps) {
        const int i = i0 + u, s = i % C::kStages;
        bool ok = mbar_wait(&full[s], (i / C::kStages) & 1);
        if (__any_sync(0xffffffffu, !ok || flags[0] != 0)) {
          if (!ok) set_status(a.status, PL_ERR_TIMEOUT);
          flags[0] = 1;
          break;
        }
        const int tile = sp.tile(lo + u), base = tile * kTile;
        const uint8_t* kt = smem + s * C::kStageBytes;
        uint8_t* vt = smem + s * C::kStageBytes + C::kTileBytes;
        const bool here = page_ok[s] != 0;
        auto sees = [&](int pos) { return here && pos < sp.len && (pos >= sp.wlo || pos < a.sinks); };
        const bool see0 = sees(base + g), see1 = sees(base + g + 8);
        if (base + kTile > sp.len || (base < sp.wlo && base + kTile > a.sinks) || !here) {
          // hidden positions: p is 0, but 0 x NaN is NaN, so their V rows are cleared
          for (int idx = lane; idx < kTile * 8 * C::kHalves; idx += 32) {
            const int r = idx / (8 * C::kHalves), c = idx % (8 * C::kHalves);
            if (!sees(base + r))
              *reinterpret_cast<uint4*>(vt + (c / 8) * C::kHalfBytes + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        // ---- S^T = K . Q^T: 16 positions x 8 heads, two chains
        float sc[NT][4], sd[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[nt][c] = sd[nt][c] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int r = (lane & 7) + 8 * ((lane >> 3) & 1), c = 2 * kk + (lane >> 4);
          uint32_t ka[4];
          ldsm_x4(smem_u32(kt + (c >> 3) * C::kHalfBytes + line_swz(r, c & 7)), ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816((kk & 1) ? sd[nt] : sc[nt], ka, qb[nt][kk]);
        }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float v = (sc[nt][c] + sd[nt][c]) * sl2;
            sc[nt][c] = (c < 2 ? see0 : see1) ? v : -INFINITY;
            grow |= sc[nt][c] > m[nt][c & 1] + kLineSlack;
          }
        if constexpr (kWeights) {
          float* dst = a.scores + ((int64_t)(sp.begin) * (a.page_size / kTile) + tile) * a.num_qo_heads * kTile +
                       kvh * a.group * kTile;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int h = 8 * nt + 2 * t + (c & 1);
              if (h < a.group) dst[h * kTile + g + 8 * (c >> 1)] = sc[nt][c];
            }
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(sc[nt][e], sc[nt][2 + e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              top = fmaxf(top, m[nt][e]);
              const float keep = m[nt][e] == -INFINITY ? 0.f : line_exp2(m[nt][e] - top);  // 0 x NaN stays NaN
              m[nt][e] = top;
              l[nt][e] *= keep;
#pragma unroll
              for (int j = 0; j < D / 16; ++j) {
                o[nt][j][e] *= keep;
                o[nt][j][2 + e] *= keep;
              }
            }
        }
        // ---- P, its sums, and P^T as the B operand
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float n0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], n1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
          const float p0 = line_exp2(sc[nt][0] - n0), p1 = line_exp2(sc[nt][1] - n1);
          const float p2 = line_exp2(sc[nt][2] - n0), p3 = line_exp2(sc[nt][3] - n1);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pb[nt][0] = movmatrix_trans(pack_bf16x2(p0, p1));
          pb[nt][1] = movmatrix_trans(pack_bf16x2(p2, p3));
        }
        // ---- O^T += V^T . P^T
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const int r = (lane & 7) + 8 * (lane >> 4), c = 2 * j + ((lane >> 3) & 1);
          uint32_t va[4];
          ldsm_x4_trans(smem_u32(vt + (c >> 3) * C::kHalfBytes + line_swz(r, c & 7)), va[0], va[1], va[2], va[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][j], va, pb[nt]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      i0 += n;

      // ---- join the warps' states (a warp without tiles has m = -inf, l = 0)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
      // channel d of head h at d ^ 8 (h / 2 % 4): the lanes of a store differ in bank
      float* mine = join + cw * C::kHeads * D;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            mine[(8 * nt + 2 * t + (c & 1)) * D + ((16 * j + g + 8 * (c >> 1)) ^ (8 * t))] = o[nt][j][c];
        if (g == 0) {
          ml[cw * C::kHeads + 8 * nt + 2 * t] = make_float2(m[nt][0], l[nt][0]);
          ml[cw * C::kHeads + 8 * nt + 2 * t + 1] = make_float2(m[nt][1], l[nt][1]);
        }
      }
      named_barrier(1, 32 * kLineWarps);
      const bool whole = lo == 0 && hi == sp.n;
      float* piece = a.partial + ((int64_t)blockIdx.x * 2 + (lo == 0 ? 1 : 0)) * a.group * C::kPiece;
      for (int idx = ctid; idx < a.group * (D / 4); idx += 32 * kLineWarps) {
        const int h = idx / (D / 4), d = 4 * (idx % (D / 4));
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kLineWarps; ++w) M = fmaxf(M, ml[w * C::kHeads + h].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kLineWarps; ++w) {
          const float2 x = ml[w * C::kHeads + h];
          const float wt = x.x == -INFINITY ? 0.f : exp2f(x.x - M);  // 0 x NaN stays NaN: a query of NaN
          const float4 v = *reinterpret_cast<const float4*>(join + (w * C::kHeads + h) * D + (d ^ (8 * (h / 2 % 4))));
          L += wt * x.y;
          acc.x += wt * v.x;
          acc.y += wt * v.y;
          acc.z += wt * v.z;
          acc.w += wt * v.w;
        }
        if (flags[0] != 0) continue;
        if (whole) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          const int head = kvh * a.group + h;
          bf16* dst = a.out + (int64_t)row * a.o_stride_b + (int64_t)head * a.o_stride_h + d;
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          if (a.out_lse != nullptr && d == 0)
            a.out_lse[(int64_t)row * a.num_qo_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        } else {
          *reinterpret_cast<float4*>(piece + h * C::kPiece + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(piece + h * C::kPiece + D) = make_float2(M, L);
        }
      }
      if (ctid == 0) flags[1] = flags[0];  // one decision for all warps
      named_barrier(1, 32 * kLineWarps);   // the scratch is read before the next item's states come
      return flags[1] == 0;
    });
  }
}

// weight[row][pos] += sum over the query heads of 2^(score - lse), from the
// scores and log sums that the decode left.  One block takes 256 positions of
// the page table's line; each thread one position, heads in order.
__global__ void __launch_bounds__(kLineAccum)
    weight_add_kernel(const LineArgs a, const float* lse, float* weight, int64_t weight_stride, int32_t capacity) {
  extern __shared__ float lse2[];  // [Hq] of the row at hand
  pdl_launch_dependents();
  pdl_wait();
  const int per = a.page_size / kTile;                       // tiles per entry
  const int64_t tiles = a.total_pages * per;
  const int64_t t0 = (int64_t)blockIdx.x * (kLineAccum / kTile);
  const int64_t t1 = t0 + kLineAccum / kTile < tiles ? t0 + kLineAccum / kTile : tiles;
  // first row whose pages end behind this block's first tile
  __shared__ int first_row;
  if (threadIdx.x == 0) first_row = a.batch;
  __syncthreads();
  for (int r = threadIdx.x; r < a.batch; r += kLineAccum)
    if ((int64_t)a.indptr[r + 1] * per > t0 && (r == 0 || (int64_t)a.indptr[r] * per <= t0)) atomicMin(&first_row, r);
  __syncthreads();
  const int lo = first_row;
  for (int r = lo; r < a.batch; ++r) {
    const RowSpan sp = row_span(a, r, false);
    if (sp.n == 0) continue;  // (a table outside the entries may begin anywhere: the rows behind it count)
    const int64_t first = (int64_t)sp.begin * per;
    if (first >= t1) break;
    __syncthreads();
    for (int h = threadIdx.x; h < a.num_qo_heads; h += kLineAccum) {
      const float l = lse[(int64_t)r * a.num_qo_heads + h];
      lse2[h] = l == -INFINITY ? INFINITY : l * kLog2e;  // a row that sees nothing gives nothing (-inf less -inf is NaN)
    }
    __syncthreads();
    const int64_t tile = t0 + threadIdx.x / kTile;
    const int64_t pos = (tile - first) * kTile + threadIdx.x % kTile;
    if (tile >= t1 || pos < 0 || pos >= sp.len) continue;
    if (pos >= capacity) {
      set_status(a.status, PL_ERR_ROW_CAPACITY);
      continue;
    }
    const float* sc = a.scores + tile * a.num_qo_heads * kTile + threadIdx.x % kTile;
    float* dst = weight + (int64_t)r * weight_stride + pos;
    const float old = *dst;
    float sum = 0.f;
    constexpr int kLoads = 16;  // in flight
    for (int h0 = 0; h0 < a.num_qo_heads; h0 += kLoads) {
      float v[kLoads];
#pragma unroll
      for (int h = 0; h < kLoads; ++h) v[h] = h0 + h < a.num_qo_heads ? __ldcg(sc + (h0 + h) * kTile) : -INFINITY;
#pragma unroll
      for (int h = 0; h < kLoads; ++h)
        if (h0 + h < a.num_qo_heads) sum += line_exp2(v[h] - lse2[h0 + h]);
    }
    *dst = old + sum;
  }
}

}  // namespace pl

// =================================================================== host
namespace {

int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

template <int D, int NT, bool kWeights>
int32_t launch_line(const CUtensorMap& map, const pl::LineArgs& a, void* stream) {
  using C = pl::LineCfg<D, NT>;
  auto kern = pl::line_decode_kernel<D, NT, kWeights>;
  int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (st != PL_OK) return st;
  st = pl_host::launch_pdl(kern, dim3(a.ctas), dim3(pl::kLineThreads), C::kSmemBytes, stream, map, a);
  if (st != PL_OK) return st;
  return pl_host::launch_line_finish<D>(a, stream);
}

template <bool kWeights>
int32_t run_line(const void* kv_cache, int32_t head_dim, const pl::LineArgs& a, void* stream) {
  CUtensorMap map;
  const int32_t st = pl_host::kv_tensor_map_rows(kv_cache, a.num_pages, a.num_kv_heads, head_dim, a.page_size,
                                                 pl::kTile, &map);
  if (st != PL_OK) return st;
  if (head_dim == 128)
    return a.group <= 8 ? launch_line<128, 1, kWeights>(map, a, stream) : launch_line<128, 2, kWeights>(map, a, stream);
  return a.group <= 8 ? launch_line<64, 1, kWeights>(map, a, stream) : launch_line<64, 2, kWeights>(map, a, stream);
}

pl::LineArgs line_args(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t num_pages, const int32_t* indptr,
                       const int32_t* indices, const int32_t* last_page_len, int64_t total_pages, int32_t batch,
                       int32_t hq, int32_t hkv, int32_t ps, float sm_scale, int32_t window, int32_t sinks, void* out,
                       int64_t o_stride_b, int64_t o_stride_h, float* out_lse, void* workspace, int32_t* status) {
  pl::LineArgs a = {};
  a.q = static_cast<const pl::bf16*>(q);
  a.q_stride_b = q_stride_b;
  a.q_stride_h = q_stride_h;
  a.indptr = indptr;
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.total_pages = total_pages;
  a.num_pages = num_pages;
  a.batch = batch;
  a.num_qo_heads = hq;
  a.num_kv_heads = hkv;
  a.group = hq / hkv;
  a.page_size = ps;
  a.window = window;
  a.sinks = sinks;
  a.item_heads = 1;
  a.items = hkv;
  a.ctas = pl_host::sm_count();
  a.pad = 2;         // an item's change costs about as much as two tiles
  a.min_tiles = 8;   // a tile for every warp
  a.scale_log2 = sm_scale * pl::kLog2e;
  a.out = static_cast<pl::bf16*>(out);
  a.o_stride_b = o_stride_b;
  a.o_stride_h = o_stride_h;
  a.out_lse = out_lse;
  a.partial = static_cast<float*>(workspace);
  a.status = status;
  return a;
}

}  // namespace

extern "C" int64_t pl_window_decode_workspace_bytes(int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || head_dim <= 0) return 0;
  const int ctas = pl_host::sm_count() > 0 ? pl_host::sm_count() : 148;
  return align256(pl_host::line_partial_bytes(ctas, num_qo_heads / num_kv_heads, head_dim));
}

extern "C" int32_t pl_paged_window_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv_cache,
                                          int64_t num_pages, const int32_t* indptr, const int32_t* indices,
                                          const int32_t* last_page_len, int64_t total_pages, int32_t batch,
                                          int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                          int32_t page_size, float sm_scale, int32_t window, int32_t sinks, void* out,
                                          int64_t o_stride_b, int64_t o_stride_h, float* out_lse, void* workspace,
                                          int64_t workspace_bytes, int32_t* status_dev, void* stream) {
  int32_t st = pl_host::line_check(q, q_stride_b, q_stride_h, kv_cache, num_pages, indptr, indices, last_page_len,
                                   total_pages, batch, num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale,
                                   window, sinks, out, o_stride_b, o_stride_h);
  if (st != PL_OK) return st;
  if (window < 1) return PL_ERR_INVALID_ARGUMENT;
  if (batch == 0) return PL_OK;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < pl_window_decode_workspace_bytes(num_qo_heads, num_kv_heads, head_dim))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  if (pl_host::sm_count() <= 0) return PL_ERR_NO_DEVICE;
  const pl::LineArgs a = line_args(q, q_stride_b, q_stride_h, num_pages, indptr, indices, last_page_len, total_pages,
                                   batch, num_qo_heads, num_kv_heads, page_size, sm_scale, window, sinks, out,
                                   o_stride_b, o_stride_h, out_lse, workspace, status_dev);
  return run_line<false>(kv_cache, head_dim, a, stream);
}

extern "C" int64_t pl_decode_weights_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                     int32_t head_dim, int32_t page_size, int64_t total_pages) {
  if (batch < 0 || total_pages < 0 || page_size <= 0) return 0;
  return pl_window_decode_workspace_bytes(num_qo_heads, num_kv_heads, head_dim) +
         align256((int64_t)batch * num_qo_heads * 4) + align256(total_pages * page_size * num_qo_heads * 4);
}

extern "C" int32_t pl_paged_decode_weights(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv_cache,
                                           int64_t num_pages, const int32_t* indptr, const int32_t* indices,
                                           const int32_t* last_page_len, int64_t total_pages, int32_t batch,
                                           int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int32_t page_size, float sm_scale, void* out, int64_t o_stride_b,
                                           int64_t o_stride_h, float* out_lse, float* weight, int64_t weight_stride,
                                           int32_t weight_capacity, void* workspace, int64_t workspace_bytes,
                                           int32_t* status_dev, void* stream) {
  int32_t st = pl_host::line_check(q, q_stride_b, q_stride_h, kv_cache, num_pages, indptr, indices, last_page_len,
                                   total_pages, batch, num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale, 0, 0,
                                   out, o_stride_b, o_stride_h);
  if (st != PL_OK) return st;
  if (weight_capacity < 0 || weight_stride < weight_capacity || (weight == nullptr && weight_capacity > 0))
    return PL_ERR_INVALID_ARGUMENT;
  if (num_qo_heads > 8192) return PL_ERR_UNSUPPORTED;
  if (batch == 0) return PL_OK;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < pl_decode_weights_workspace_bytes(batch, num_qo_heads, num_kv_heads, head_dim, page_size, total_pages))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  if (pl_host::sm_count() <= 0) return PL_ERR_NO_DEVICE;
  pl::LineArgs a = line_args(q, q_stride_b, q_stride_h, num_pages, indptr, indices, last_page_len, total_pages, batch,
                             num_qo_heads, num_kv_heads, page_size, sm_scale, 0, 0, out, o_stride_b, o_stride_h,
                             out_lse, workspace, status_dev);
  uint8_t* at = static_cast<uint8_t*>(workspace) +
                pl_window_decode_workspace_bytes(num_qo_heads, num_kv_heads, head_dim);
  if (a.out_lse == nullptr) a.out_lse = reinterpret_cast<float*>(at);
  a.scores = reinterpret_cast<float*>(at + align256((int64_t)batch * num_qo_heads * 4));
  st = run_line<true>(kv_cache, head_dim, a, stream);
  if (st != PL_OK || total_pages == 0) return st;
  const int64_t blocks = (total_pages * page_size + pl::kLineAccum - 1) / pl::kLineAccum;
  return pl_host::launch_pdl(pl::weight_add_kernel, dim3((unsigned)blocks), dim3(pl::kLineAccum),
                             (size_t)num_qo_heads * 4, stream, a, (const float*)a.out_lse, weight, weight_stride,
                             weight_capacity);
}
