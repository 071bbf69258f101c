// Eviction by accumulated attention weight: the weights that a prompt's
// tokens give the cached positions (pl_paged_prefill_weights), and the choice
// of the positions to keep (pl_evict_select).  The decode step's weights come
// with its attention (pl_window_decode.cu); pl_cache_compact moves what stays.
#include <type_traits>

#include "pl_line_decode.cuh"

namespace pl {

// ------------------------------------------------------- weights of a prompt
// weight[b][j] += sum over query tokens i and heads h of exp(scale q_ih.k_j -
// lse_ih), i at position p_i >= j.  The attention that gave lse has read V and
// written O; this is its score product alone, transposed.  One CTA takes a
// (request, run of 256 positions, kv head, chunk of the query tiles), keeps
// the run's K in shared memory and streams the query tiles (128 rows = tq
// tokens x the group's heads) that see it.
//   warp 0     TMA: K once, then the query tiles through a ring, and the log
//              sums of their columns;
//   warp 1     tcgen05.mma S^T = K.Q^T, two products of 128 positions a query
//              tile, each into one of two TMEM buffers;
//   warps 2-17 four groups of four, one for each buffer: a thread is a
//              position, reads its 128 scores, and adds 2^(s - lse) into its
//              own sums, so nothing is exchanged between threads.
// The sums of the kv heads and chunks go to the workspace and are added in
// this order by prompt_weight_add_kernel, so two runs give the same bits.
// 128 x 128 scores have 1024 cycles of exponentials on the multi-function
// units (16 a cycle) beside 512 cycles of products at head_dim 128, so a
// quarter of the pairs is computed on the FMA pipe instead (pw_exp2_pair, nine
// cycles an element; none 393, a quarter 381, half 421 us at 8192 tokens, 32
// heads).  Measured 377 us there, 0.73 PFLOP/s: 1250 cycles a product, of
// which the chain product -> commit -> read -> exponentials of a buffer and
// its successor's is what is left; tensor memory holds no third one.
constexpr int kPwM = 128;                   // positions of a product
constexpr int kPwTiles = 2;                 // products a CTA: 256 positions
constexpr int kPwN = 128;                   // rows of a query tile
constexpr int kPwThreads = 32 * (2 + 8 * kPwTiles);
constexpr int kPwSlots = 4;                 // query tiles in flight
constexpr int kPwLse = kPwSlots + 4;        // log sums: of tiles whose scores are not added yet
constexpr int kPwChunks = 4;                // at most as many chunks of a request's query tiles

struct PromptWeightArgs {
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_last;
  int64_t num_pages, total_pages;
  int32_t batch, total_q, num_qo_heads, num_kv_heads, group, page_size;
  int32_t tq;            // tokens of a tile
  int32_t chunk;         // token tiles of a chunk
  float scale_log2;
  const float* lse;   // [total_q, Hq]
  float* partial;     // [kPwChunks][Hkv][total_pages * page_size]
  int32_t* status;
};

template <int D>
struct PromptWeightCfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kKChunkBytes = kPwM * 128;                   // 64 channels of 128 positions
  static constexpr int kKBytes = kChunks * kKChunkBytes;
  static constexpr int kQChunkBytes = kPwN * 128;
  static constexpr int kQBytes = kChunks * kQChunkBytes;
  static constexpr int kSlotOff = kPwTiles * kKBytes;               // behind K
  static constexpr int kLseOff = kSlotOff + kPwSlots * kQBytes;     // [kPwLse][128]
  static constexpr int kBarOff = kLseOff + kPwLse * kPwN * 4;       // kfull qfull[] qempty[] sready[][2] sfree[][2] fin
  static constexpr int kSumOff = kBarOff + (2 + 2 * kPwSlots + 4 * kPwTiles) * 8;  // [tiles][128]
  static constexpr int kMiscOff = kSumOff + kPwTiles * kPwM * 4;
  static constexpr int kSmemBytes = 1024 + kMiscOff + 80;
  static_assert(kSmemBytes <= 232448, "tiles exceed the shared-memory limit");
};

// 2^x of a pair by range reduction to [-1/2, 1/2] and a polynomial of degree 5
// of least relative error there, 1 at 0 (1.2e-7 with its coefficients in fp32;
// 1.8e-7 with the roundings of its steps, where the multi-function unit has
// 2.4e-7).  x below -127 counts as -127, whose bits come out as 0, and above
// 128 as 128, whose bits are inf.  NaN has no bits that the exponent's addition
// would leave a NaN, so 0 x is added at the end.
__device__ __forceinline__ float2 pw_exp2_pair(float2 x) {
  auto clamp = [](float v) {
    float r;
    asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC2FE0000;\n\tmin.NaN.f32 %0, t, 0f43000000;\n\t}"  // -127, 128
        : "=f"(r)
        : "f"(v));
    return r;
  };
  auto both = [](float v) { return make_float2(v, v); };
  x = make_float2(clamp(x.x), clamp(x.y));
  const float2 r = add_f32x2(x, both(12582912.f));  // the nearest whole number, in the low bits
  const float2 n = add_f32x2(r, both(-12582912.f));
  const float2 f = fma_f32x2(n, both(-1.f), x);
  float2 p = fma_f32x2(both(0.001326458528637886f), f, both(0.0096714673563838f));
  p = fma_f32x2(p, f, both(0.05550733581185341f));
  p = fma_f32x2(p, f, both(0.24022242426872253f));
  p = fma_f32x2(p, f, both(0.6931470036506653f));
  p = fma_f32x2(p, f, both(1.f));
  p = make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)),
                  __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
  return fma_f32x2(x, both(0.f), p);
}

// Request and run of positions that block `x` of the line of runs takes; a
// table outside kv_indices has none.  One warp; false past the last run.
struct PwSpan {
  int req, run, kv_begin, n_pages, kv_len, q0, qlen;
};
constexpr int kPwRun = kPwTiles * kPwM;

__device__ __forceinline__ int pw_kv_len(const PromptWeightArgs& a, int b, bool report) {
  const int k0 = a.kv_indptr[b], k1 = a.kv_indptr[b + 1];
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1];
  int last = a.kv_last[b];
  last = last < 0 ? 0 : (last > a.page_size ? a.page_size : last);
  const int len = k1 > k0 ? (k1 - k0 - 1) * a.page_size + last : 0;
  if (k0 < 0 || k1 < k0 || (int64_t)k1 > a.total_pages || q0 < 0 || q1 < q0 || q1 > a.total_q || q1 - q0 > len) {
    if (report) set_status(a.status, PL_ERR_INVALID_ARGUMENT);
    return 0;
  }
  return q1 > q0 ? len : 0;
}

// First token tile whose queries see position `pos` of a request.
__device__ __forceinline__ int pw_first(const PromptWeightArgs& a, int pos, int kv_len, int qlen) {
  const int p0 = kv_len - qlen;
  return pos > p0 ? (pos - p0) / a.tq : 0;
}

__device__ __forceinline__ bool pw_find(const PromptWeightArgs& a, int x, PwSpan& s) {
  const int lane = threadIdx.x % 32;
  int before = 0;
  for (int base = 0; base < a.batch; base += 32) {
    const int b = base + lane;
    const int len = b < a.batch ? pw_kv_len(a, b, false) : 0;
    const int n = (len + kPwRun - 1) / kPwRun;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > x);
    if (hit != 0) {
      const int src = __ffs(hit) - 1;
      s.req = base + src;
      s.run = x - (before + __shfl_sync(0xffffffffu, incl - n, src));
      s.kv_len = __shfl_sync(0xffffffffu, len, src);
      s.kv_begin = a.kv_indptr[s.req];
      s.n_pages = a.kv_indptr[s.req + 1] - s.kv_begin;
      s.q0 = a.qo_indptr[s.req];
      s.qlen = a.qo_indptr[s.req + 1] - s.q0;
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

template <int D>
__global__ void __launch_bounds__(kPwThreads, 1)
    prompt_weight_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map,
                         const PromptWeightArgs a) {
  using C = PromptWeightCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* qfull = kfull + 1;              // [slots] query tile and log sums landed
  uint64_t* qempty = qfull + kPwSlots;      // [slots] query tile read
  uint64_t* sready = qempty + kPwSlots;     // [tiles][2] scores in TMEM
  uint64_t* sfree = sready + 2 * kPwTiles;  // [tiles][2] scores read (4 warps)
  uint64_t* fin = sfree + 2 * kPwTiles;     // every tensor-core op finished
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
  volatile int32_t* flags = reinterpret_cast<volatile int32_t*>(smem + C::kMiscOff + 16);  // abort, issued, consumed
  PwSpan* span = reinterpret_cast<PwSpan*>(smem + C::kMiscOff + 32);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = blockIdx.x % a.num_kv_heads, chunk = blockIdx.x / a.num_kv_heads % kPwChunks;

  if (threadIdx.x == 0) {
    mbar_init(kfull, 1);
    for (int i = 0; i < kPwSlots; ++i) {
      mbar_init(&qfull[i], 33);  // the copies, and the lanes' log sums
      mbar_init(&qempty[i], 1);
    }
    for (int i = 0; i < 2 * kPwTiles; ++i) {
      mbar_init(&sready[i], 1);
      mbar_init(&sfree[i], 4);
    }
    mbar_init(fin, 1);
    flags[0] = flags[1] = flags[2] = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == 32) {
    prefetch_tensormap(&kv_map);
    prefetch_tensormap(&q_map);
  }
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    PwSpan s = {};
    s.req = -1;
    pw_find(a, blockIdx.x / a.num_kv_heads / kPwChunks, s);
    if (lane == 0) *span = s;
  }
  __syncthreads();
  const PwSpan sp = *span;
  const int PS = a.page_size, kv0 = sp.run * kPwRun;
  // token tiles [j0, j1) of this chunk see the run
  const int j0 = max(chunk * a.chunk, pw_first(a, kv0, sp.kv_len, sp.qlen));
  const int j1 = min((chunk + 1) * a.chunk, (sp.qlen + a.tq - 1) / a.tq);
  if (sp.req < 0 || j0 >= j1) return;  // nothing was started
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  const int rows = a.tq * a.group;  // rows of a query tile in use; the others are 0
  for (int i = threadIdx.x; i < kPwSlots * C::kChunks * (kPwN - rows) * 8; i += kPwThreads) {
    const int c = i / ((kPwN - rows) * 8), u = i % ((kPwN - rows) * 8);
    reinterpret_cast<uint4*>(smem + C::kSlotOff + c * C::kQChunkBytes + rows * 128)[u] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n = j1 - j0;
  const int p_first = sp.kv_len - sp.qlen;
  const int tiles = min(kPwTiles, (sp.kv_len - kv0 + kPwM - 1) / kPwM);
  // the first of this CTA's tiles that sees product x
  auto first_of = [&](int x) { return max(0, pw_first(a, kv0 + x * kPwM, sp.kv_len, sp.qlen) - j0); };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int ppt = kPwM / PS, boxes = ppt * C::kChunks;  // <= 16
    {
      const int p = lane / C::kChunks, hh = lane % C::kChunks;
      if (lane == 0) mbar_arrive_expect_tx(kfull, tiles * C::kKBytes);
      __syncwarp();
      for (int x = 0; x < tiles; ++x) {
        if (lane < boxes) {
          const int page = (kv0 / kPwM + x) * ppt + p;
          int32_t coord = (int32_t)(2 * a.num_pages);  // out of range: zeros
          if (page < sp.n_pages) {
            const int32_t pid = a.kv_indices[sp.kv_begin + page];
            if (pid >= 0 && (int64_t)pid < a.num_pages)
              coord = 2 * pid;
            else
              set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
          }
          tma_load_4d(smem + x * C::kKBytes + hh * C::kKChunkBytes + p * PS * 128, &kv_map, hh * 64, kvh, 0, coord,
                      kfull);
        }
      }
    }
    // log sums of columns 4 lane .. 4 lane + 3; columns without a query: inf
    int tok[4], off[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      tok[e] = 4 * lane + e < rows ? (4 * lane + e) / a.group : 0x3fffffff;
      off[e] = (4 * lane + e) / a.group * a.num_qo_heads + (4 * lane + e) % a.group;
    }
    auto lse_of = [&](int j, float* v) {
      const float* src = a.lse + (int64_t)(sp.q0 + j * a.tq) * a.num_qo_heads + kvh * a.group;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = j * a.tq + tok[e] < sp.qlen ? __ldg(src + off[e]) : INFINITY;
    };
    int i = 0;
    float next[4];
    lse_of(j0, next);
    for (; i < n; ++i) {
      const int s = i % kPwSlots;
      bool ok = true;
      // (the products of tile i - 4 waited until tile i - 6 was read, and so tile i - 8 added, whose log sums'
      // place tile i takes)
      if (i >= kPwSlots) ok = mbar_wait(&qempty[s], ((i / kPwSlots) - 1) & 1);
      if (__any_sync(0xffffffffu, !ok || flags[0] != 0)) {
        if (!ok) set_status(a.status, PL_ERR_TIMEOUT);
        flags[0] = 1;
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&qfull[s], C::kChunks * rows * 128);
      __syncwarp();
      if (lane < C::kChunks)
        tma_load_4d(smem + C::kSlotOff + s * C::kQBytes + lane * C::kQChunkBytes, &q_map, lane * 64, 0, kvh,
                    sp.q0 + (j0 + i) * a.tq, &qfull[s]);
      float l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] = next[e] == -INFINITY ? -INFINITY : -next[e] * kLog2e;
      if (i + 1 < n) lse_of(j0 + i + 1, next);
      reinterpret_cast<float4*>(smem + C::kLseOff + i % kPwLse * kPwN * 4)[lane] = make_float4(l[0], l[1], l[2], l[3]);
      mbar_arrive(&qfull[s]);
    }
    if (lane == 0) flags[1] = i;
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    // The whole warp walks the loop, with counts that are uniform by
    // construction, and one lane issues: descriptors then stay in uniform
    // registers.  (With one lane alone in the loop every product's operands
    // went through the vector registers: about 125 cycles an instruction,
    // where 128 columns take 64.)
    constexpr uint32_t idesc = umma_idesc_bf16(kPwM, kPwN);
    const uint32_t leader = elect_one();
    const int nu = uniform(n), tu = uniform(tiles);
    int done[kPwTiles], from[kPwTiles];  // products issued, first token tile
#pragma unroll
    for (int x = 0; x < kPwTiles; ++x) {
      done[x] = 0;
      from[x] = uniform(first_of(x));
    }
    const uint32_t tm = uniform((int)tmem), base = smem_u32(smem);
    int consumed = 0;
    bool ok = __all_sync(0xffffffffu, mbar_wait(kfull, 0));
    for (int i = 0; ok && i < nu; ++i) {
      const int s = i % kPwSlots;
      ok = __all_sync(0xffffffffu, mbar_wait(&qfull[s], (i / kPwSlots) & 1) && !flags[0]);
      if (!ok) break;
      consumed = i + 1;
      const uint32_t qs = base + C::kSlotOff + s * C::kQBytes;
#pragma unroll
      for (int x = 0; x < kPwTiles; ++x) {
        if (x < tu && i >= from[x] && ok) {
          const int k = done[x]++, b = 2 * x + (k & 1);
          if (k >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&sfree[b], ((k >> 1) - 1) & 1));
          tc_fence_after();
          if (ok) {
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                umma_bf16_if(leader, tm + (uint32_t)(b * kPwN),
                             umma_desc_k_sw128(base + x * C::kKBytes + c * C::kKChunkBytes + 32 * e),
                             umma_desc_k_sw128(qs + c * C::kQChunkBytes + 32 * e), idesc, (c | e) ? 1u : 0u);
            umma_commit_if(leader, &sready[b]);
          }
        }
      }
      umma_commit_if(leader, &qempty[s]);
    }
    if (lane == 0) {
      if (!ok) {
        set_status(a.status, PL_ERR_TIMEOUT);
        flags[0] = 1;
      }
      flags[2] = consumed;
    }
    umma_commit_if(leader, fin);
    if (!mbar_wait(fin, 0)) set_status(a.status, PL_ERR_TIMEOUT);
    __syncwarp();
  } else {
    // -------------------------------------------------------- exponentials
    const int x = (warp - 2) / 8, b = (warp - 2) / 4, quad = warp & 3;  // product, buffer
    const int m = 32 * quad + lane;  // position within the product == TMEM lane
    const uint32_t row_tmem = tmem + ((uint32_t)(32 * quad) << 16);
    const int pos = kv0 + x * kPwM + m;
    const float2 sl2 = make_float2(a.scale_log2, a.scale_log2);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    bool ok = true;
    const int first_tile = first_of(x) + (b & 1);
    for (int i = first_tile, k = 0; x < tiles && i < n; i += 2, ++k) {
      ok = mbar_wait(&sready[b], k & 1);
      if (__any_sync(0xffffffffu, !ok || flags[0] != 0)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // column c is a query at position first + c / group: seen from column `from` on
      const int first = p_first + (j0 + i) * a.tq;
      const int from = pos > first ? (pos - first) * a.group : 0;
      const int to = (sp.qlen - (j0 + i) * a.tq) * a.group;  // columns behind are another request's queries
      const float4* lse4 = reinterpret_cast<const float4*>(smem + C::kLseOff + i % kPwLse * kPwN * 4);
      auto add_tile = [&](auto masked_t) {
        constexpr bool kMasked = decltype(masked_t)::value;
#pragma unroll 1
        for (int h = 0; h < kPwN / 32; ++h) {
          float v[32];
          tmem_ld32(row_tmem + (uint32_t)(b * kPwN + 32 * h), v);
          if (h == kPwN / 32 - 1) {  // read: the next product may come while these are added
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sfree[b]);
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 l = lse4[8 * h + c];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = 4 * c + 2 * e, pair = 2 * c + e;
              float2 p = fma_f32x2(make_float2(v[col], v[col + 1]), sl2,
                                   e == 0 ? make_float2(l.x, l.y) : make_float2(l.z, l.w));
              if (pair % 4 == 1)
                p = pw_exp2_pair(p);
              else
                p = make_float2(line_exp2(p.x), line_exp2(p.y));
              if constexpr (kMasked) {
                p.x = 32 * h + col >= from && 32 * h + col < to ? p.x : 0.f;
                p.y = 32 * h + col + 1 >= from && 32 * h + col + 1 < to ? p.y : 0.f;
              }
              sum[e] = add_f32x2(sum[e], p);
            }
          }
        }
      };
      if (kv0 + (x + 1) * kPwM - 1 > first || to < rows)
        add_tile(std::true_type{});
      else
        add_tile(std::false_type{});
    }
    if (!ok) {
      set_status(a.status, PL_ERR_TIMEOUT);
      flags[0] = 1;
    }
    // the sums of a product's two buffers
    float* sums = reinterpret_cast<float*>(smem + C::kSumOff) + x * kPwM;
    const float mine = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    if (b & 1) sums[m] = mine;
    named_barrier(1 + x, 256);
    if (!(b & 1) && flags[0] == 0 && pos < sp.kv_len)
      a.partial[((int64_t)chunk * a.num_kv_heads + kvh) * a.total_pages * PS + (int64_t)sp.kv_begin * PS + pos] =
          mine + sums[m];
  }

  __syncthreads();
  if (threadIdx.x == 0) {
    const int issued = flags[1], consumed = flags[2];
    for (int i = consumed; i < issued; ++i) (void)mbar_wait(&qfull[i % kPwSlots], (i / kPwSlots) & 1);
    (void)mbar_wait(kfull, 0);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// weight[b][pos] += the sums of the kv heads and of the chunks whose queries see
// the position's run, in this order; a thread per position of the page
// table's line.  The requests that hold the block's entries are looked for one
// by one, since requests with bad tables (which block 0 reports) may stand
// between them.
__global__ void __launch_bounds__(256)
    prompt_weight_add_kernel(const PromptWeightArgs a, int32_t hkv, float* weight, int64_t weight_stride,
                             int32_t capacity) {
  __shared__ int32_t owner[256 / 16];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t all = a.total_pages * a.page_size;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int entries = 256 / a.page_size, e0 = (int)(blockIdx.x * entries);
  if (threadIdx.x < entries) owner[threadIdx.x] = a.batch;
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += 256)
    if (pw_kv_len(a, b, blockIdx.x == 0) > 0)
      for (int e = max(a.kv_indptr[b], e0); e < min(a.kv_indptr[b + 1], e0 + entries); ++e) atomicMin(&owner[e - e0], b);
  __syncthreads();
  if (at >= all) return;
  const int lo = owner[threadIdx.x / a.page_size];
  if (lo >= a.batch) return;
  const int len = pw_kv_len(a, lo, false);
  const int64_t pos = at - (int64_t)a.kv_indptr[lo] * a.page_size;
  if (pos >= len) return;
  if (pos >= capacity) {
    set_status(a.status, PL_ERR_ROW_CAPACITY);
    return;
  }
  const int qlen = a.qo_indptr[lo + 1] - a.qo_indptr[lo];
  const int c0 = pw_first(a, (int)pos / kPwRun * kPwRun, len, qlen) / a.chunk, c1 = ((qlen + a.tq - 1) / a.tq - 1) / a.chunk;
  float sum = 0.f;
  for (int c = c0; c <= c1; ++c)
#pragma unroll 8
    for (int h = 0; h < hkv; ++h) sum += __ldcg(a.partial + ((int64_t)c * hkv + h) * all + at);
  weight[(int64_t)lo * weight_stride + pos] += sum;
}

// ------------------------------------------------------------------ select
// The positions that a row of len > budget keeps: the first `sinks`, the last
// `recent`, and the k = budget - sinks - recent others of the highest weight,
// the lowest position first among equals.  Weights compare as numbers (-0 as
// 0; a NaN above all).  A radix select over the bits finds the k-th largest:
// 11, 11 and 10 bits in three passes, each a histogram in shared memory; then
// every warp counts what its run of positions keeps, and after a scan of the
// counts writes it in ascending order.  A row is one CTA, or (kCluster) eight
// that share its positions; each adds up a slice of their histograms' bins through
// distributed shared memory, and all read the slices.  The ordered bits stay in shared memory from the
// first pass on (12 rows of 131072 positions: 49 us when every pass read the
// weights again); runs longer than fit there read the rest again.
constexpr int kSelThreads = 1024;
constexpr int kSelHeld = 49152;   // positions a CTA holds at most (192 KB)
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 2048;
constexpr int kSelCluster = 8;
constexpr int kSelSlice = kSelBins / kSelCluster;  // bins that a CTA of a cluster adds up

struct SelectArgs {
  const float* weight;
  int64_t weight_stride;
  int32_t capacity;     // columns of weight and out_weight
  const int32_t* lens;
  int32_t budget, sinks, recent;
  int32_t* keep_from;
  int32_t* keep;
  int64_t keep_stride;
  int32_t keep_width;
  int32_t* keep_count;
  float* out_weight;
  int64_t out_stride;
  int32_t held;         // keys that a warp holds in shared memory
  int32_t* status;
};

__device__ __forceinline__ uint32_t select_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

template <bool kCluster>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const SelectArgs a) {
  __shared__ __align__(16) int32_t hist[kSelBins];
  __shared__ __align__(16) int32_t slice[kCluster ? kSelSlice : 4];
  __shared__ int32_t scan[kSelWarps];
  __shared__ int32_t pick[2];                    // digit, count above it
  __shared__ int32_t counts[2 * kSelWarps + 2];  // per warp: above, equal; then the CTA's sums
  extern __shared__ uint32_t held[];             // [warps][a.held]: keys of the first positions of a warp's run
  constexpr int nr = kCluster ? kSelCluster : 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = kCluster ? blockIdx.x % kSelCluster : 0;
  const int row = kCluster ? blockIdx.x / kSelCluster : blockIdx.x;
  auto sync = [&]() {
    if constexpr (kCluster) cluster_sync_all(); else __syncthreads();
  };
  pdl_launch_dependents();
  pdl_wait();
  int len = a.lens[row];
  const float* w = a.weight + (int64_t)row * a.weight_stride;
  float* ow = a.out_weight + (int64_t)row * a.out_stride;
  int32_t* keep = a.keep + (int64_t)row * a.keep_stride;
  const bool cut = len > a.budget && len <= a.capacity;
  if (rank == 0 && threadIdx.x == 0) {
    if (len < 0 || len > a.capacity) set_status(a.status, PL_ERR_INVALID_ARGUMENT);
    a.keep_from[row] = cut ? a.sinks : (len < 0 ? 0 : len);
    a.keep_count[row] = cut ? a.budget - a.sinks : 0;
  }
  len = len < 0 ? 0 : (len > a.capacity ? a.capacity : len);
  const int kept = cut ? a.budget : len;
  const int tid = rank * kSelThreads + threadIdx.x;
  constexpr int all = nr * kSelThreads;
  // what does not depend on the choice
  const int k = a.budget - a.sinks - a.recent;
  auto fill = [&]() {
    const int listed = cut ? a.budget - a.sinks : 0, front = cut ? a.sinks : len;
    for (int i = listed + tid; i < a.keep_width; i += all) keep[i] = -1;
    for (int i = kept + tid; i < a.capacity; i += all) ow[i] = 0.f;
    for (int i = tid; i < front; i += all) ow[i] = w[i];
    if (cut)
      for (int i = tid; i < a.recent; i += all) {
        const int pos = len - a.recent + i;
        keep[k + i] = pos;
        ow[a.sinks + k + i] = w[pos];
      }
  };
  if (!cut) {
    fill();
    return;  // the whole row's CTAs alike
  }
  // this warp's run of the candidates [sinks, len - recent)
  const int c0 = a.sinks, n = len - a.recent - a.sinks;
  const int runs = nr * kSelWarps, per = ((n + runs - 1) / runs + 31) / 32 * 32;
  const int b = min(n, (rank * kSelWarps + warp) * per), e = min(n, b + per);
  uint32_t* mine_held = held + warp * a.held;
  const int eh = min(e, b + a.held);
  // f(key) of every candidate of the run
  auto walk = [&](auto f) {
#pragma unroll 8
    for (int i = b + lane; i < eh; i += 32) f(mine_held[i - b]);
#pragma unroll 4
    for (int i = eh + lane; i < e; i += 32) f(select_key(w[c0 + i]));
  };
#pragma unroll 8
  for (int i = b + lane; i < eh; i += 32) mine_held[i - b] = select_key(w[c0 + i]);

  uint32_t prefix = 0, mask = 0;
  int want = k;  // still to be found among the keys with this prefix
  if (k > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      for (int i = threadIdx.x; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      walk([&](uint32_t key) {
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1);
      });
      sync();
      if constexpr (kCluster) {
        if (threadIdx.x < kSelSlice) {
          const uint32_t at = smem_u32(hist + rank * kSelSlice + threadIdx.x);
          int sum = 0;
#pragma unroll
          for (int r = 0; r < nr; ++r) sum += __float_as_int(dsmem_ld_f32(dsmem_map(at, r)));
          slice[threadIdx.x] = sum;
        }
        cluster_sync_all();
      }
      // four bins a thread of the first half of the block, from the highest down
      const int bin = kSelBins - 4 - 4 * threadIdx.x;
      int4 h = make_int4(0, 0, 0, 0);
      if (bin >= 0) {
        if constexpr (kCluster) {
          const float4 f = dsmem_ld_f32x4(dsmem_map(smem_u32(slice + bin % kSelSlice), bin / kSelSlice));
          h = make_int4(__float_as_int(f.x), __float_as_int(f.y), __float_as_int(f.z), __float_as_int(f.w));
        } else {
          h = *reinterpret_cast<const int4*>(hist + bin);
        }
      }
      const int mine = h.x + h.y + h.z + h.w;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      int above = incl - mine;
      for (int i = 0; i < warp; ++i) above += scan[i];
      if (above < want && want <= above + mine) {
        int d = bin + 3;
        if (want > above + h.w) { above += h.w; --d;
          if (want > above + h.z) { above += h.z; --d;
            if (want > above + h.y) { above += h.y; --d; } } }
        pick[0] = d;
        pick[1] = above;
      }
      __syncthreads();  // the digit is known (another CTA writes its slice again behind the next cluster barrier only)
      prefix |= (uint32_t)pick[0] << shift;
      mask |= ((1u << bits) - 1) << shift;
      want -= pick[1];
    }
  } else {
    prefix = 0xffffffffu;
  }
  // counts of every warp's run: above the key, equal to it
  int gt = 0, eq = 0;
  walk([&](uint32_t key) {
    gt += key > prefix;
    eq += key == prefix;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) {
    counts[2 * warp] = gt;
    counts[2 * warp + 1] = eq;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int g = 0, q = 0;
    for (int i = 0; i < kSelWarps; ++i) {
      g += counts[2 * i];
      q += counts[2 * i + 1];
    }
    counts[2 * kSelWarps] = g;
    counts[2 * kSelWarps + 1] = q;
  }
  sync();
  gt = eq = 0;  // in front of this warp's run
  if constexpr (kCluster) {
    for (int r = 0; r < rank; ++r) {
      gt += __float_as_int(dsmem_ld_f32(dsmem_map(smem_u32(&counts[2 * kSelWarps]), r)));
      eq += __float_as_int(dsmem_ld_f32(dsmem_map(smem_u32(&counts[2 * kSelWarps + 1]), r)));
    }
  }
  for (int i = 0; i < warp; ++i) {
    gt += counts[2 * i];
    eq += counts[2 * i + 1];
  }
  if constexpr (kCluster) cluster_sync_all();  // the counts are read; no CTA's shared memory is needed by another now
  fill();  // (behind the barriers, which would wait for the stores)
  const unsigned below = (1u << lane) - 1;
  for (int i0 = b; i0 < e; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < eh ? mine_held[i - b] : (i < e ? select_key(w[c0 + i]) : 0u);
    const unsigned bg = __ballot_sync(0xffffffffu, i < e && key > prefix);
    const unsigned bq = __ballot_sync(0xffffffffu, i < e && key == prefix);
    const int g = gt + __popc(bg & below), q = eq + __popc(bq & below);
    const bool take = i < e && (key > prefix || (key == prefix && q < want));
    if (take) {
      const int at = g + min(q, want);
      keep[at] = c0 + i;
      ow[a.sinks + at] = w[c0 + i];
    }
    gt += __popc(bg);
    eq += __popc(bq);
  }
}

}  // namespace pl

// =================================================================== host
namespace {

int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

template <int D>
int32_t launch_prompt_weights(const CUtensorMap& kv_map, const CUtensorMap& q_map, const pl::PromptWeightArgs& a,
                              int64_t blocks, void* stream) {
  using C = pl::PromptWeightCfg<D>;
  auto kern = pl::prompt_weight_kernel<D>;
  const int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (st != PL_OK) return st;
  return pl_host::launch_pdl(kern, dim3((unsigned)blocks), dim3(pl::kPwThreads), C::kSmemBytes, stream, kv_map,
                             q_map, a);
}

}  // namespace

extern "C" int64_t pl_prefill_weights_workspace_bytes(int32_t num_kv_heads, int32_t page_size, int64_t total_pages) {
  if (num_kv_heads <= 0 || page_size <= 0 || total_pages < 0) return 0;
  return align256(pl::kPwChunks * total_pages * page_size * num_kv_heads * 4);
}

extern "C" int32_t pl_paged_prefill_weights(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv_cache,
                                            int64_t num_pages, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                            const int32_t* kv_indices, const int32_t* kv_last_page_len,
                                            int64_t total_pages, int32_t batch, int32_t total_q, int32_t num_qo_heads,
                                            int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float sm_scale,
                                            const float* lse, float* weight, int64_t weight_stride,
                                            int32_t weight_capacity, void* workspace, int64_t workspace_bytes,
                                            int32_t* status_dev, void* stream) {
  if (batch < 0 || total_q < 0 || num_pages <= 0 || total_pages < 0 || num_kv_heads <= 0 || num_qo_heads <= 0 ||
      num_qo_heads % num_kv_heads != 0 || kv_cache == nullptr || !(sm_scale > 0.f) || weight_capacity < 0 ||
      weight_stride < weight_capacity || (weight == nullptr && weight_capacity > 0))
    return PL_ERR_INVALID_ARGUMENT;
  const int group = num_qo_heads / num_kv_heads;
  if (group > 128 || (head_dim != 64 && head_dim != 128) ||
      (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) || num_kv_heads > 65535 ||
      total_pages * page_size > 0x7FFFFFFFll || num_pages > 0x3FFFFFFFll)
    return PL_ERR_UNSUPPORTED;
  if (batch == 0 || total_q == 0) return PL_OK;
  if (q == nullptr || qo_indptr == nullptr || kv_indptr == nullptr || (kv_indices == nullptr && total_pages > 0) ||
      kv_last_page_len == nullptr || lse == nullptr)
    return PL_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_cache)) & 15) != 0 || q_stride_t <= 0 || q_stride_h <= 0 || q_stride_t % 8 != 0 || q_stride_h % 8 != 0)
    return PL_ERR_INVALID_ARGUMENT;
  if (total_pages > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
                          workspace_bytes < pl_prefill_weights_workspace_bytes(num_kv_heads, page_size, total_pages)))
    return PL_ERR_WORKSPACE_TOO_SMALL;

  pl::PromptWeightArgs a = {};
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.kv_last = kv_last_page_len;
  a.num_pages = num_pages;
  a.total_pages = total_pages;
  a.batch = batch;
  a.total_q = total_q;
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.tq = pl::kPwN / group;
  // chunks share long prompts out (the first run of positions is seen by all queries, the last by few)
  a.chunk = ((total_q + a.tq - 1) / a.tq + pl::kPwChunks - 1) / pl::kPwChunks;
  if (a.chunk < 16) a.chunk = 16;
  a.page_size = page_size;
  a.scale_log2 = sm_scale * pl::kLog2e;
  a.lse = lse;
  a.partial = static_cast<float*>(workspace);
  a.status = status_dev;

  const int64_t add = (total_pages * page_size + 255) / 256;
  auto launch_add = [&](int64_t blocks) {
    return pl_host::launch_pdl(pl::prompt_weight_add_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a,
                               num_kv_heads, weight, weight_stride, weight_capacity);
  };
  if (total_pages == 0) return launch_add(1);  // tokens without a cached position: reported
  CUtensorMap kv_map, q_map;
  int32_t st = pl_host::kv_tensor_map(kv_cache, num_pages, num_kv_heads, head_dim, page_size, &kv_map);
  if (st != PL_OK) return st;
  pl_host::EncodeTiledFn enc = pl_host::encode_tiled_fn();
  if (enc == nullptr) return PL_ERR_CUDA;
  // q as {head_dim, heads of a group, kv heads, tokens}; a box is 64 channels of tq tokens
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)group, (cuuint64_t)num_kv_heads, (cuuint64_t)total_q};
  const cuuint64_t strides[3] = {(cuuint64_t)q_stride_h * 2, (cuuint64_t)q_stride_h * 2 * group,
                                 (cuuint64_t)q_stride_t * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)a.tq};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  if (enc(&q_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(q), dims, strides, box, ones,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return PL_ERR_INVALID_ARGUMENT;
  // a row of n positions has ceil(n / 256) <= n / 256 + 1 runs
  const int64_t blocks = (total_pages * page_size / pl::kPwRun + batch) * pl::kPwChunks * num_kv_heads;
  if (blocks > 0x7FFFFFFF) return PL_ERR_UNSUPPORTED;
  st = head_dim == 128 ? launch_prompt_weights<128>(kv_map, q_map, a, blocks, stream)
                       : launch_prompt_weights<64>(kv_map, q_map, a, blocks, stream);
  return st != PL_OK ? st : launch_add(add);
}

extern "C" int32_t pl_evict_select(const float* weight, int64_t weight_stride, int32_t capacity, const int32_t* lens,
                                   int32_t num_rows, int32_t budget, int32_t sinks, int32_t recent, int32_t* keep_from,
                                   int32_t* keep, int64_t keep_stride, int32_t keep_width, int32_t* keep_count,
                                   float* out_weight, int64_t out_stride, int32_t* status_dev, void* stream) {
  if (num_rows < 0 || capacity < 0 || budget < 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget ||
      keep_width < budget - sinks || keep_stride < keep_width || weight_stride < capacity || out_stride < capacity)
    return PL_ERR_INVALID_ARGUMENT;
  if (num_rows > 0x7FFFFFFF / pl::kSelCluster) return PL_ERR_UNSUPPORTED;
  if (num_rows == 0) return PL_OK;
  if (lens == nullptr || keep_from == nullptr || keep_count == nullptr || (keep == nullptr && keep_width > 0) ||
      (capacity > 0 && (weight == nullptr || out_weight == nullptr || weight == out_weight)))
    return PL_ERR_INVALID_ARGUMENT;
  pl::SelectArgs a;
  a.weight = weight;
  a.weight_stride = weight_stride;
  a.capacity = capacity;
  a.lens = lens;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.keep_from = keep_from;
  a.keep = keep;
  a.keep_stride = keep_stride;
  a.keep_width = keep_width;
  a.keep_count = keep_count;
  a.out_weight = out_weight;
  a.out_stride = out_stride;
  a.status = status_dev;
  // One CTA walks 8192 positions in about the time that a cluster's exchanges take.
  const bool cluster = capacity > 8192;
  const int64_t runs = pl::kSelWarps * (cluster ? pl::kSelCluster : 1);
  const int64_t per = ((capacity + runs - 1) / runs + 31) / 32 * 32;
  a.held = (int32_t)(per < pl::kSelHeld / pl::kSelWarps ? per : pl::kSelHeld / pl::kSelWarps);
  const size_t smem = (size_t)a.held * pl::kSelWarps * 4;
  auto kern = cluster ? pl::evict_select_kernel<true> : pl::evict_select_kernel<false>;
  const int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), pl::kSelHeld * 4);
  if (st != PL_OK) return st;
  if (cluster)
    return pl_host::launch_pdl_cluster(kern, dim3((unsigned)num_rows * pl::kSelCluster), dim3(pl::kSelThreads), smem,
                                       stream, pl::kSelCluster, a);
  return pl_host::launch_pdl(kern, dim3((unsigned)num_rows), dim3(pl::kSelThreads), smem, stream, a);
}
