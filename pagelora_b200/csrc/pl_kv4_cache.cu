// A paged K/V cache in 4 bits: quantising append, expansion of pages back to
// bf16, and decode attention straight over the codes.
//
// Record of one head of one token (K or V), D/2 + 16 bytes: the codes, two
// channels a byte (the even one in the low half), then four scales and four
// minima in bf16.  Channel c belongs to group c % 4; value = min + scale *
// code with min the group's smallest value (a bf16 value, kept exactly),
// scale = bf16((max - min) / 15) and code = rint((x - min) / scale) in 0..15.
// Interleaved groups make both products of the attention simple: masking a
// word of codes with 0x000F000F leaves two channels of ONE group (for K, where
// channels are summed over), and a word's nibbles of one position are the same
// row of eight output tiles (for V, where channels are rows).
// The records stand in the pool as [pages][2][page_size][kv heads][record], so
// the page operations move them like any other token.
#include <mutex>

#include "pl_line_decode.cuh"

namespace pl {

__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// The smaller and the larger of packed pairs; NaN where one is NaN.
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// a b - c
__device__ __forceinline__ uint32_t fms_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("{\n\t.reg .b32 n;\n\tneg.bf16x2 n, %3;\n\tfma.rn.bf16x2 %0, %1, %2, n;\n\t}" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// ----------------------------------------------------------------- append
// Eight lanes take one record (K or V of one head of one token): D / 8
// channels a lane, a group's extremes by three exchanges.  Differences are
// taken between halves of the values, which do not overflow, so every finite
// bf16 input has finite scales; they round (once, to fp32) where the values'
// exponents lie more than 16 apart.  A group with inf or NaN decodes to NaN.  A
// code comes from a product with 1 / scale and is put right by its remainder,
// exact for that difference (ties are common among bf16 values; dividing where
// one was near cost 44 us for 16384 tokens of 8 heads).
// Bound by HBM: 2 D bytes in, D / 2 + 16 out.
template <int D>
__global__ void __launch_bounds__(256)
    kv4_append_kernel(const bf16* k, int64_t k_stride, const bf16* v, int64_t v_stride, uint8_t* cache,
                      int64_t num_pages, const int32_t* page_id, const int32_t* page_off, int32_t tokens, int32_t hkv,
                      int32_t page_size, int32_t* status) {
  constexpr int E = D / 8, kRecord = D / 2 + 16;
  pdl_launch_dependents();
  pdl_wait();
  // record (token, K / V, head) of the line; the host keeps their number below 2^31
  const uint32_t rec = blockIdx.x * 32 + threadIdx.x / 8;
  const int sub = threadIdx.x % 8;
  const bool on = rec < (uint32_t)tokens * 2 * hkv;
  const uint32_t part = on ? rec / hkv : 0;
  const int h = on ? (int)(rec - part * hkv) : 0, kv = part & 1, tok = (int)(part >> 1);
  const bf16* src = (kv ? v + (int64_t)tok * v_stride : k + (int64_t)tok * k_stride) + (int64_t)h * D + sub * E;
  uint32_t x[E / 2];  // pairs of channels: groups 0, 1 and 2, 3 in turn
#pragma unroll
  for (int u = 0; u < E / 8; ++u) {
    const uint4 w = on ? __ldg(reinterpret_cast<const uint4*>(src) + u) : make_uint4(0, 0, 0, 0);
    x[4 * u] = w.x;
    x[4 * u + 1] = w.y;
    x[4 * u + 2] = w.z;
    x[4 * u + 3] = w.w;
  }
  uint32_t lo2[2] = {x[0], x[1]}, hi2[2] = {x[0], x[1]};
#pragma unroll
  for (int i = 2; i < E / 2; ++i) {
    lo2[i & 1] = min_bf16x2(lo2[i & 1], x[i]);
    hi2[i & 1] = max_bf16x2(hi2[i & 1], x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      lo2[c] = min_bf16x2(lo2[c], __shfl_xor_sync(0xffffffffu, lo2[c], o));
      hi2[c] = max_bf16x2(hi2[c], __shfl_xor_sync(0xffffffffu, hi2[c], o));
    }
  // lane `sub` has group sub % 4's scale and minimum, and tells the others
  float lo[4], step[4], inv[4];
  uint32_t tail;  // (scale, minimum) of the lane's group
  {
    const uint32_t lw = (sub & 2) ? lo2[1] : lo2[0], hw = (sub & 2) ? hi2[1] : hi2[0];
    const float l = 0.5f * ((sub & 1) ? bf_hi(lw) : bf_lo(lw)), h = 0.5f * ((sub & 1) ? bf_hi(hw) : bf_lo(hw));
    const bool good = l > -INFINITY && h < INFINITY;  // (NaN is neither)
    const float spread = bfr((h - l) / 7.5f), s = spread >= 7.52316384526264e-37f ? spread : 0.f;  // 2^-120: 1 / s is finite
    tail = good ? pack_bf16x2(s, 2.f * l) : 0x7FFF7FFFu;
    const float st = good && s > 0.f ? 0.5f * s : 1.f, iv = 1.f / st;  // a constant group: all codes 0
    const int from = threadIdx.x & 24;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      lo[c] = __shfl_sync(0xffffffffu, l, from + c);
      step[c] = __shfl_sync(0xffffffffu, st, from + c);
      inv[c] = __shfl_sync(0xffffffffu, iv, from + c);
    }
  }
  constexpr float kWhole = 12582912.f;  // adding it leaves the nearest whole number in the low bits
  auto half_of = [&](int i) { return 0.5f * ((i & 1) ? bf_hi(x[i / 2]) : bf_lo(x[i / 2])); };
  uint32_t code[E / 8];
#pragma unroll
  for (int u = 0; u < E / 8; ++u) {
    code[u] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i % 4;
      const float d = half_of(8 * u + i) - lo[c], w = fmaf(d, inv[c], kWhole);
      // the remainder is exact: above half a step, or half of one beside an odd code, the neighbour is right
      const float r = fmaf(kWhole - w, step[c], d), h = 0.5f * step[c];
      int q = __float_as_int(w);
      if (fabsf(r) > ((q & 1) ? __uint_as_float(__float_as_uint(h) - 1) : h)) q += r > 0.f ? 1 : -1;
      code[u] |= (uint32_t)(q & 15) << (4 * i);
    }
  }
  if (!on) return;
  const int32_t pid = page_id[tok], off = page_off[tok];
  if (pid < 0 || (int64_t)pid >= num_pages || off < 0 || off >= page_size) {
    if (sub == 0) set_status(status, PL_ERR_PAGE_OUT_OF_RANGE);
    return;
  }
  uint8_t* dst = cache + ((((int64_t)pid * 2 + kv) * page_size + off) * hkv + h) * kRecord;
  if constexpr (E == 16)
    *reinterpret_cast<uint2*>(dst + 8 * sub) = make_uint2(code[0], code[1]);
  else
    *reinterpret_cast<uint32_t*>(dst + 4 * sub) = code[0];
  if (sub < 4) {
    reinterpret_cast<uint16_t*>(dst + D / 2)[sub] = (uint16_t)tail;
    reinterpret_cast<uint16_t*>(dst + D / 2)[4 + sub] = (uint16_t)(tail >> 16);
  }
}

// ----------------------------------------------------------------- expand
// out[i] = bf16(min + scale * code) of page page_ids[i]; eight lanes a
// record.  Bound by HBM: D / 2 + 16 bytes in, 2 D out.
template <int D>
__global__ void __launch_bounds__(256)
    kv4_expand_kernel(const uint8_t* cache, int64_t num_pages, const int32_t* page_ids, int32_t per_page, bf16* out,
                      int32_t* status) {
  constexpr int E = D / 8, kRecord = D / 2 + 16;
  pdl_launch_dependents();
  pdl_wait();
  // 32 records of page i (per_page, K and V, is a multiple of 32 for pages of 16 tokens)
  const int blocks = per_page / 32, i = blockIdx.x / blocks;
  const int at = (blockIdx.x - i * blocks) * 32 + threadIdx.x / 8, sub = threadIdx.x % 8;
  const int32_t pid = page_ids[i];
  if (pid < 0 || (int64_t)pid >= num_pages) {
    if (pid != -1 && threadIdx.x == 0) set_status(status, PL_ERR_PAGE_OUT_OF_RANGE);
    return;
  }
  const uint8_t* src = cache + ((int64_t)pid * per_page + at) * kRecord;
  const uint4 tail = __ldg(reinterpret_cast<const uint4*>(src + D / 2));
  uint32_t code[E / 8];
  if constexpr (E == 16) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + 8 * sub));
    code[0] = w.x;
    code[1] = w.y;
  } else {
    code[0] = __ldg(reinterpret_cast<const uint32_t*>(src + 4 * sub));
  }
  // Pairs of channels G and G + 4 of a word: 128 + code as bf16 bits, less 128, and one packed fma, which rounds
  // min + scale * code once.
  uint32_t sc[4], mn[4];
  const uint32_t ts[4] = {tail.x, tail.x, tail.y, tail.y}, tm[4] = {tail.z, tail.z, tail.w, tail.w};
#pragma unroll
  for (int G = 0; G < 4; ++G) {
    sc[G] = __byte_perm(ts[G], 0, (G & 1) ? 0x3232 : 0x1010);
    mn[G] = __byte_perm(tm[G], 0, (G & 1) ? 0x3232 : 0x1010);
  }
  uint4* dst = reinterpret_cast<uint4*>(out + ((int64_t)i * per_page + at) * D + sub * E);
#pragma unroll
  for (int u = 0; u < E / 8; ++u) {
    uint32_t v[4];
#pragma unroll
    for (int G = 0; G < 4; ++G)
      v[G] = fma_bf16x2(sub_bf16x2(((code[u] >> (4 * G)) & 0x000F000Fu) | 0x43004300u, 0x43004300u), sc[G], mn[G]);
    dst[u] = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                        __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
  }
}

// ----------------------------------------------------------------- decode
// One query token per row, cut as one line of work (pl_line_decode.cuh); an
// item is a row and a block of up to eight kv heads.  A warp owns a kv head,
// or shares it with others that take the tiles of 16 positions in turn.  It
// brings its own tiles, 16 bytes a lane and copy, through a ring of its own,
// so no warp waits for another: records are 80 or 48 bytes, too short for TMA
// (boxes of one head's 16 records streamed 2.4 TB/s whatever the consumers
// did), and the warps of a CTA walk the heads of the same positions, whose
// records share sectors, at about the same time.  A record's pitch of 20 or 12
// words spreads the eight rows of a fragment over all banks.
//
// The products run on the codes, not on dequantised values.  A code's four
// bits, alone in the low half of a 16-bit word, are the bf16 number code *
// 2^-133 (subnormal, or of the first binade: bf16 bits below 256 are linear),
// and the next four bits, left where they are, 16 code * 2^-133; tensor core
// and bf16x2 arithmetic take such numbers exactly.  So w & 0x000F000F and w &
// 0x00F000F0 are operands as they stand, one instruction for two codes, and
// the other side carries the power of two back.  With Q_hG = sum of q over
// group G,
//   S_jh = sum_G s_jG (sum_{d in G} q_hd c_jd) + sum_G m_jG Q_hG,
//   O_dh = sum_j (p_jh s_jG)(c_jd - 8) + sum_j p_jh m_jG + 8 sum_j p_jh s_jG.
// sum_G m Q is one product with Q in three bf16 parts (exact to 2^-24); the
// last two sums are the rows of one product with the tile's tails.  K is
// exact.  p is rounded to bf16 (2^-8, as elsewhere); p s enters as a bf16 value
// and its exact remainder, since a group's spread can exceed a channel's: one
// rounded p s gave a relative error of 0.0031 in place of 0.0023 (and 616 us
// in place of 697, for 64 rows of 8192 positions and 32 kv heads; remainders
// of p too: 0.0017 and 740).  Codes of V are centred (one subtraction for two)
// since the tensor core's sums truncate in proportion to what they hold: an
// offset of 128 in place of the subnormals measured 0.039 at 8192 positions.
// P^T is turned into the operand layout before the scales go on, as packed
// pairs.
//
// The powers of two bound the range: q below 2^56 in size, V's values times the
// row's positions below 2^55 (p reaches 2^68, and their sums are fp32), and
// steps of 2^-76 in O where all of V is smaller than 2^-53.
//
// The bytes (160 a position and head at head_dim 128 where bf16 has 512) are
// within reach of HBM, 412 us there.  No unit is full: of the issue slots 59 %
// are taken (about 390 instructions a tile and head), of the logic pipe's 48,
// the tensor pipe is active for 32 %, HBM at 47.  What bounds it is the latency
// of dependent instructions with four warps a scheduler: an instruction of a
// warp takes 6.3 cycles, 1.3 of fixed latency, 1.0 for a pipe, 1.1 for its turn,
// 0.9 for memory.  Two CTAs share an SM where a group fits one column block (128
// registers a thread), and the next tile's scores stand between this one's
// values (646 -> 616 us), so that one's latencies are the other's issue slots.
template <int D, int NT>
struct Kv4Cfg {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kCtas = NT == 1 ? 2 : 1;           // per SM
  static constexpr int kRecord = D / 2 + 16;
  static constexpr int kWords = kRecord / 4;
  static constexpr int kPartBytes = kTile * kRecord;      // K (or V) of a tile
  static constexpr int kCopies = 2 * kPartBytes / 512;    // copies of 16 bytes a lane and tile
  static constexpr int kStages = 5;                       // tiles of a warp's ring
  static constexpr int kStageBytes = 2 * kPartBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kSteps = D / 64;                   // k16 steps of a group
  static constexpr int kTiles = D / 16;                   // output tiles
  static constexpr int kState = kTiles * 4 + 4;           // a lane's O, m and l of one column block
  static constexpr int kRegs = NT * kState;
  static constexpr int kRingOff = 36 * 8;                 // behind line_find's scratch
  static constexpr int kSmemBytes = kRingOff + kWarps * kRingBytes;
  static_assert(kRegs * 128 <= kRingBytes, "a warp's state joins through its ring");
  static_assert(2 * kPartBytes % 512 == 0, "whole copies");
  static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "the rings exceed the shared memory");
};

// Powers of two that the operands carry: codes 2^-133 (x 16 for odd groups),
// q 2^64 (/ 16), so scores 2^-69; p 2^60.
constexpr float kKv4Q = 18446744073709551616.f;           // 2^64
constexpr float kKv4Score = 590295810358705651712.f;      // 2^69
constexpr float kKv4P = 60.f;                             // exponent of p's factor
constexpr float kKv4Unp = 8.673617379884035e-19f;         // 2^-60
constexpr float kKv4Out = 9444732965739290427392.f;       // 2^73 = 2^(133 - 60)

struct Kv4Plan {
  int32_t heads;   // kv heads of an item
  int32_t share;   // warps that share a head (a power of two)
};

// 16 bytes to shared memory; zeros (src is not read) when bytes is 0.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <int D, int NT>
__global__ void __launch_bounds__(Kv4Cfg<D, NT>::kThreads, Kv4Cfg<D, NT>::kCtas)
    kv4_decode_kernel(const uint8_t* cache, const LineArgs a, const Kv4Plan pl) {
  using C = Kv4Cfg<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_launch_dependents();
  pdl_wait();
  int row0;
  int64_t row_start;
  const LineCut cut = line_find<C::kThreads>(a, blockIdx.x, reinterpret_cast<int64_t*>(smem), row0, row_start);
  if ((int64_t)blockIdx.x >= cut.ctas) return;
  const int64_t begin = cut.begin(blockIdx.x), end = cut.begin((int64_t)blockIdx.x + 1);

  const int hh = warp / pl.share, turn = warp % pl.share;
  if (hh >= pl.heads) return;  // (a head count that the warps do not divide into)
  const int g = lane >> 2, t = lane & 3;
  const int sharers = pl.heads * pl.share * 32;  // threads at the join's barriers
  const float sl2 = a.scale_log2 * kKv4Score;    // scores come x 2^-69
  uint8_t* ring = smem + C::kRingOff + warp * C::kRingBytes;
  // a lane's copies of a tile: 16-byte unit lane + 32 i of [K, V][position][record]
  const int64_t token_bytes = (int64_t)a.num_kv_heads * C::kRecord;
  const int log_per = __ffs(a.page_size) - 5;  // tiles of a page, a power of two
  const int tile_bytes = (int)token_bytes * kTile;
  const uint32_t ring_at = smem_u32(ring) + 16 * lane;
  const uint32_t tails_at = smem_u32(ring) + C::kPartBytes + (lane % kTile) * C::kRecord + D / 2;
  uint32_t src_off[C::kCopies];
#pragma unroll
  for (int i = 0; i < C::kCopies; ++i) {
    const int unit = lane + 32 * i, rec = unit / (C::kRecord / 16), c = unit % (C::kRecord / 16);
    src_off[i] = (uint32_t)((rec / kTile * a.page_size + rec % kTile) * token_bytes + 16 * c);
  }
  constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;  // codes of even groups; odd ones, x 16
  for_each_segment(a, row0, row_start, begin, end, [&](int row, const RowSpan& sp, int item, int lo, int hi) {
    const int kvh = item * pl.heads + hh;
    const bool head_on = kvh < a.num_kv_heads;
    // ---- Q as B operands: lane (g, t) has head g's words t, t + 4 .. of eight
    // channels; a pair is channels G and G + 4 of a word, as the masks leave them
    uint32_t qb[NT][4][C::kSteps][2], mq[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = 8 * nt + g;
      const bool on = head_on && h < a.group;
      const bf16* src = a.q + (int64_t)row * a.q_stride_b + (int64_t)(kvh * a.group + h) * a.q_stride_h;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 2 * C::kSteps; ++w) {
        const uint4 v = on ? __ldg(reinterpret_cast<const uint4*>(src) + t + 4 * w) : make_uint4(0, 0, 0, 0);
        const uint32_t p[4] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                               __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632)};
#pragma unroll
        for (int G = 0; G < 4; ++G) {
          const float x = bf_lo(p[G]), y = bf_hi(p[G]), f = (G & 1) ? kKv4Q / 16.f : kKv4Q;
          qb[nt][G][w >> 1][w & 1] = pack_bf16x2(x * f, y * f);
          sum[G] += x + y;
        }
      }
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], 1);
        sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], 2);
      }
      // the sums, as the scores x 2^-69, in three bf16 parts at k = 4 part + group
      const float x0 = ((t & 1) ? sum[2] : sum[0]) / kKv4Score, x1 = ((t & 1) ? sum[3] : sum[1]) / kKv4Score;
      const float h0 = bfr(x0), h1 = bfr(x1), m0 = bfr(x0 - h0), m1 = bfr(x1 - h1);
      mq[nt][0] = t < 2 ? pack_bf16x2(h0, h1) : pack_bf16x2(m0, m1);
      mq[nt][1] = t < 2 ? pack_bf16x2(x0 - h0 - m0, x1 - h1 - m1) : 0u;
    }
    float o[NT][C::kTiles][4];
    float pt[NT][4];  // rows G: sum p scale, rows 4 + G: sum p min (8 .. 15 unused)
    float ref[NT][2], l[NT][2];  // 60 - the reference of the exponentials, in log2; sum of p
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < C::kTiles; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      pt[nt][0] = pt[nt][1] = pt[nt][2] = pt[nt][3] = 0.f;
      ref[nt][0] = ref[nt][1] = INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // ---- this warp's tiles of the segment: lo + turn, lo + turn + share, ...
    const int n = hi - lo > turn ? (hi - lo - turn + pl.share - 1) / pl.share : 0;
    const uint8_t* head_base = cache + (int64_t)(head_on ? kvh : 0) * C::kRecord;
    auto tile_at = [&](int k) { return sp.tile(lo + turn + k * pl.share); };
    // places of 32 tiles in the pool (in tiles; -1: none) a load, one load ahead
    auto places = [&](int k) -> int32_t {
      if (k >= n) return -1;
      const int tile = tile_at(k);
      const int32_t pid = a.indices[sp.begin + (tile >> log_per)];
      if (pid >= 0 && (int64_t)pid < a.num_pages) return (pid << (log_per + 1)) + (tile & ((1 << log_per) - 1));
      set_status(a.status, PL_ERR_PAGE_OUT_OF_RANGE);
      return -1;
    };
    int32_t now = places(lane), next = places(32 + lane);
    auto issue = [&](int k, uint32_t stage) {
      if (k < n) {
        if (k != 0 && (k & 31) == 0) {
          now = next;
          next = places(k + 32 + lane);
        }
        const int32_t place = __shfl_sync(0xffffffffu, now, k & 31);
        const uint32_t bytes = place >= 0 ? 16 : 0;  // else zeros
        const uint8_t* src = head_base + (int64_t)max(place, 0) * tile_bytes;
        const uint32_t dst = ring_at + stage;
#pragma unroll
        for (int i = 0; i < C::kCopies; ++i) cp_async16(dst + 512 * i, src + src_off[i], bytes);
      }
      cp_async_commit();  // (an empty group past the last tile keeps the count)
    };
#pragma unroll
    for (int k = 0; k < C::kStages - 1; ++k) issue(k, k * C::kStageBytes);
    // Scores of a tile: the groups' products one by one (step), so that they
    // can stand between those of another tile's V.
    float sc[NT][4];  // 16 positions x 8 heads, x 2^-69
    uint32_t w0[2 * C::kSteps], w1[2 * C::kSteps];
    uint2 s0, s1;
    auto scores_begin = [&](uint32_t stage) {
      const uint8_t* kg = ring + stage + g * C::kRecord;  // K of position g
      const uint32_t* k0 = reinterpret_cast<const uint32_t*>(kg) + t;
#pragma unroll
      for (int w = 0; w < 2 * C::kSteps; ++w) {
        w0[w] = k0[4 * w];
        w1[w] = k0[8 * C::kWords + 4 * w];
      }
      const uint4 t0 = *reinterpret_cast<const uint4*>(kg + D / 2);
      const uint4 t1 = *reinterpret_cast<const uint4*>(kg + 8 * C::kRecord + D / 2);
      const uint32_t mm0 = (t & 1) ? t0.w : t0.z, mm1 = (t & 1) ? t1.w : t1.z;
      const uint32_t ma[4] = {mm0, mm1, mm0, mm1};
      s0 = make_uint2(t0.x, t0.y);
      s1 = make_uint2(t1.x, t1.y);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16_16816_zero(sc[nt], ma, mq[nt]);
    };
    auto scores_step = [&](int G) {
      if (G == 2) {
#pragma unroll
        for (int w = 0; w < 2 * C::kSteps; ++w) {
          w0[w] >>= 8;
          w1[w] >>= 8;
        }
      }
      const uint32_t mask = (G & 1) ? kOdd : kEven;
      const float f0 = (G & 1) ? bf_hi(G < 2 ? s0.x : s0.y) : bf_lo(G < 2 ? s0.x : s0.y);
      const float f1 = (G & 1) ? bf_hi(G < 2 ? s1.x : s1.y) : bf_lo(G < 2 ? s1.x : s1.y);
      float acc[NT][4];
#pragma unroll
      for (int st = 0; st < C::kSteps; ++st) {
        const uint32_t ka[4] = {w0[2 * st] & mask, w1[2 * st] & mask, w0[2 * st + 1] & mask, w1[2 * st + 1] & mask};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (st == 0)
            mma_bf16_16816_zero(acc[nt], ka, qb[nt][G][st]);
          else
            mma_bf16_16816(acc[nt], ka, qb[nt][G][st]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc[nt][0] = fmaf(acc[nt][0], f0, sc[nt][0]);
        sc[nt][1] = fmaf(acc[nt][1], f0, sc[nt][1]);
        sc[nt][2] = fmaf(acc[nt][2], f1, sc[nt][2]);
        sc[nt][3] = fmaf(acc[nt][3], f1, sc[nt][3]);
      }
    };
    uint32_t here = 0, freed = (C::kStages - 1) * C::kStageBytes;  // stages of tile k, of tile k - 1 (and k + 4)
    int u = lo + turn;                                  // tile k's place among the visible ones
    const int window_edge = sp.wlo > 0 ? sp.early : -1;  // (the sinks' tiles and the window's first)
    cp_async_wait<C::kStages - 2>();
    __syncwarp();
    scores_begin(0);
#pragma unroll
    for (int G = 0; G < 4; ++G) scores_step(G);
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      const uint8_t* vt = ring + here + C::kPartBytes + 2 * t * C::kRecord;  // V of position 2t
      const uint32_t tails = tails_at + here;
      uint8_t* v_tile = ring + here + C::kPartBytes;
      // positions of this tile may be hidden: in front of the window, or behind the last one
      const bool edge = u <= window_edge || u == sp.n - 1;
      const int u_here = u;
      u += pl.share;
      auto sees = [&](int i) {
        const int pos = sp.tile(u_here) * kTile + i;
        return pos < sp.len && (pos >= sp.wlo || pos < a.sinks);
      };
      if (edge) {  // p is 0 there, but 0 x NaN is NaN, so their V tails are cleared
        if (lane < kTile && !sees(lane))
          *reinterpret_cast<uint4*>(v_tile + lane * C::kRecord + D / 2) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      // exponents of p; one above 60 + the slack moves the reference (at first it is -inf)
      float x[NT][4];
      bool grow = false;
      auto exponents = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) x[nt][c] = fmaf(sc[nt][c], sl2, ref[nt][c & 1]);
        if (edge) {
          const bool see0 = sees(g), see1 = sees(g + 8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) x[nt][c] = (c < 2 ? see0 : see1) ? x[nt][c] : -INFINITY;
        }
      };
      exponents();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) grow |= x[nt][c] > kKv4P + kLineSlack;
      if (__any_sync(0xffffffffu, grow)) {
        const bool see0 = !edge || sees(g), see1 = !edge || sees(g + 8);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(see0 ? sc[nt][e] : -INFINITY, see1 ? sc[nt][2 + e] : -INFINITY);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
            const float next = fminf(kKv4P - top * sl2, ref[nt][e]);
            const float keep = ref[nt][e] == INFINITY ? 0.f : line_exp2(next - ref[nt][e]);  // 0 x NaN stays NaN
            ref[nt][e] = next;
            l[nt][e] *= keep;
            pt[nt][e] *= keep;
#pragma unroll
            for (int j = 0; j < C::kTiles; ++j) {
              o[nt][j][e] *= keep;
              o[nt][j][2 + e] *= keep;
            }
          }
        exponents();
      }
      // ---- P, its sums, and P^T (lane (g, t): head g, positions 2t, 2t+1 and 2t+8, 2t+9)
      uint32_t ph[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float p0 = line_exp2(x[nt][0]), p1 = line_exp2(x[nt][1]);
        const float p2 = line_exp2(x[nt][2]), p3 = line_exp2(x[nt][3]);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        ph[nt][0] = movmatrix_trans(pack_bf16x2(p0, p1));
        ph[nt][1] = movmatrix_trans(pack_bf16x2(p2, p3));
      }
      // ---- sum p scale and sum p min: rows of one product with the tails, turned as they are read
      {
        uint32_t ta[4] = {0u, 0u, 0u, 0u};
        asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                     : "=r"(ta[0]), "=r"(ta[2])
                     : "r"(tails));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(pt[nt], ta, ph[nt]);
      }
      const uint32_t* va = reinterpret_cast<const uint32_t*>(vt);
      // ---- scales of the positions, in pairs; those of odd groups / 16
      uint32_t ss[4][2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint2 s0 = *reinterpret_cast<const uint2*>(va + 8 * y * C::kWords + D / 8);
        const uint2 s1 = *reinterpret_cast<const uint2*>(va + (8 * y + 1) * C::kWords + D / 8);
        ss[0][y] = __byte_perm(s0.x, s1.x, 0x5410);
        ss[1][y] = mul_bf16x2(__byte_perm(s0.x, s1.x, 0x7632), 0x3D803D80u);
        ss[2][y] = __byte_perm(s0.y, s1.y, 0x5410);
        ss[3][y] = mul_bf16x2(__byte_perm(s0.y, s1.y, 0x7632), 0x3D803D80u);
      }
      // ---- tile k + 1 is there for all lanes, and all have done with tile k - 1
      cp_async_wait<C::kStages - 3>();
      __syncwarp();
      issue(k + C::kStages - 1, freed);
      freed = here;
      here = here == (C::kStages - 1) * C::kStageBytes ? 0 : here + C::kStageBytes;
      scores_begin(here);  // (behind the last tile: of a stage that nobody reads again)
      // ---- O^T += (codes - 8)^T . (P scale)^T; the two halves of a word in turn
      uint32_t lo01[C::kSteps], hi01[C::kSteps], lo89[C::kSteps], hi89[C::kSteps];
#pragma unroll
      for (int w = 0; w < C::kSteps; ++w) {
        const uint32_t a0 = va[g + 8 * w], a1 = va[C::kWords + g + 8 * w];
        const uint32_t a8 = va[8 * C::kWords + g + 8 * w], a9 = va[9 * C::kWords + g + 8 * w];
        lo01[w] = __byte_perm(a0, a1, 0x5410);
        hi01[w] = __byte_perm(a0, a1, 0x7632);
        lo89[w] = __byte_perm(a8, a9, 0x5410);
        hi89[w] = __byte_perm(a8, a9, 0x7632);
      }
      // head_dim 128: tile j = nibble j of words g and g + 8; 64: nibbles j and j + 4 of word g
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        if (G == 2) {
#pragma unroll
          for (int w = 0; w < C::kSteps; ++w) {
            lo01[w] >>= 8;
            hi01[w] >>= 8;
            lo89[w] >>= 8;
            hi89[w] >>= 8;
          }
        }
        const uint32_t mask = (G & 1) ? kOdd : kEven, mid = (G & 1) ? 0x00800080u : 0x00080008u;
        // p scale as a bf16 value and its (exact) remainder
        uint32_t hi[NT][2], lo_part[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            hi[nt][y] = mul_bf16x2(ph[nt][y], ss[G][y]);
            lo_part[nt][y] = fms_bf16x2(ph[nt][y], ss[G][y], hi[nt][y]);
          }
        uint32_t wa[C::kTiles / 4][4];
#pragma unroll
        for (int j = G; j < C::kTiles; j += 4) {
          uint32_t* w = wa[j / 4];
          if constexpr (D == 128) {
            w[0] = j < 4 ? lo01[0] : hi01[0];
            w[1] = j < 4 ? lo01[C::kSteps - 1] : hi01[C::kSteps - 1];
            w[2] = j < 4 ? lo89[0] : hi89[0];
            w[3] = j < 4 ? lo89[C::kSteps - 1] : hi89[C::kSteps - 1];
          } else {
            w[0] = lo01[0];
            w[1] = hi01[0];
            w[2] = lo89[0];
            w[3] = hi89[0];
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = sub_bf16x2(w[c] & mask, mid);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][j], w, hi[nt]);
        }
        scores_step(G);  // (between the two products of an accumulator)
#pragma unroll
        for (int j = G; j < C::kTiles; j += 4)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][j], wa[j / 4], lo_part[nt]);
      }
    }
    cp_async_wait<0>();
    __syncwarp();  // all lanes have done with the ring

    // ---- the warp's own O: powers of two out, minima and centres in
    float m[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
        l[nt][e] *= kKv4Unp;
        m[nt][e] = kKv4P - ref[nt][e];  // -inf: nothing seen
#pragma unroll
        for (int G = 0; G < 4; ++G) {
          const float ps = __shfl_sync(0xffffffffu, pt[nt][e], 4 * G + t);
          const float mn = __shfl_sync(0xffffffffu, pt[nt][e], 16 + 4 * G + t);
          const float off = kKv4Unp * fmaf(8.f, ps, mn);
#pragma unroll
          for (int j = G; j < C::kTiles; j += 4) {
            o[nt][j][e] = fmaf(o[nt][j][e], kKv4Out, off);
            o[nt][j][2 + e] = fmaf(o[nt][j][2 + e], kKv4Out, off);
          }
        }
      }
    // ---- join the warps that share the head, in turn order
    if (pl.share > 1) {
      float* slot = reinterpret_cast<float*>(ring) + lane;  // (turn 0 keeps its own)
      if (turn != 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* p = slot + nt * C::kState * 32;
#pragma unroll
          for (int j = 0; j < C::kTiles; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) p[(4 * j + c) * 32] = o[nt][j][c];
          p[(C::kTiles * 4 + 0) * 32] = m[nt][0];
          p[(C::kTiles * 4 + 1) * 32] = m[nt][1];
          p[(C::kTiles * 4 + 2) * 32] = l[nt][0];
          p[(C::kTiles * 4 + 3) * 32] = l[nt][1];
        }
      }
      named_barrier(1, sharers);
      if (turn == 0) {
#pragma unroll 1
        for (int other = 1; other < pl.share; ++other)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float* p = slot + other * (C::kRingBytes / 4) + nt * C::kState * 32;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float mo = p[(C::kTiles * 4 + e) * 32], lo_ = p[(C::kTiles * 4 + 2 + e) * 32];
              const float top = fmaxf(m[nt][e], mo);
              const float w0 = m[nt][e] == -INFINITY ? 0.f : exp2f(m[nt][e] - top);
              const float w1 = mo == -INFINITY ? 0.f : exp2f(mo - top);
              m[nt][e] = top;
              l[nt][e] = w0 * l[nt][e] + w1 * lo_;
#pragma unroll
              for (int j = 0; j < C::kTiles; ++j) {
                o[nt][j][e] = w0 * o[nt][j][e] + w1 * p[(4 * j + e) * 32];
                o[nt][j][2 + e] = w0 * o[nt][j][2 + e] + w1 * p[(4 * j + 2 + e) * 32];
              }
            }
          }
      }
    }
    // ---- lane (g, t) holds heads 2t, 2t + 1 of channels 8g .. 8g + 7 (and 64 + 8g ..)
    if (turn == 0 && head_on) {
      const bool whole = lo == 0 && hi == sp.n;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = 8 * nt + 2 * t + e;
          if (h >= a.group) continue;
          const float L = l[nt][e], M = m[nt][e];
          if (whole) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            const int head = kvh * a.group + h;
            bf16* dst = a.out + (int64_t)row * a.o_stride_b + (int64_t)head * a.o_stride_h + 8 * g;
            if constexpr (D == 128) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                uint32_t w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  w[c] = pack_bf16x2(o[nt][2 * c][2 * half + e] * inv, o[nt][2 * c + 1][2 * half + e] * inv);
                *reinterpret_cast<uint4*>(dst + 64 * half) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
              uint32_t w[4];
#pragma unroll
              for (int c = 0; c < 4; ++c)
                w[c] = pack_bf16x2(o[nt][(2 * c) % 4][2 * (c / 2) + e] * inv,
                                   o[nt][(2 * c + 1) % 4][2 * (c / 2) + e] * inv);
              *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (a.out_lse != nullptr && g == 0)
              a.out_lse[(int64_t)row * a.num_qo_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
          } else {
            float* piece = a.partial + (((int64_t)blockIdx.x * 2 + (lo == 0 ? 1 : 0)) * a.item_heads * a.group +
                                        hh * a.group + h) * (D + 4);
#pragma unroll
            for (int half = 0; half < D / 64; ++half) {
              float4 x, y;
              if constexpr (D == 128) {
                x = make_float4(o[nt][0][2 * half + e], o[nt][1][2 * half + e], o[nt][2][2 * half + e],
                                o[nt][3][2 * half + e]);
                y = make_float4(o[nt][C::kTiles - 4][2 * half + e], o[nt][C::kTiles - 3][2 * half + e],
                                o[nt][C::kTiles - 2][2 * half + e], o[nt][C::kTiles - 1][2 * half + e]);
              } else {
                x = make_float4(o[nt][0][e], o[nt][1][e], o[nt][2][e], o[nt][3][e]);
                y = make_float4(o[nt][0][2 + e], o[nt][1][2 + e], o[nt][2][2 + e], o[nt][3][2 + e]);
              }
              *reinterpret_cast<float4*>(piece + 64 * half + 8 * g) = x;
              *reinterpret_cast<float4*>(piece + 64 * half + 8 * g + 4) = y;
            }
            if (g == 0) *reinterpret_cast<float2*>(piece + D) = make_float2(M, L);
          }
        }
    }
    if (pl.share > 1) named_barrier(1, sharers);  // the states are read before the next item's come
    return true;
  });
}

}  // namespace pl

// =================================================================== host
namespace {

int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

// Up to eight kv heads an item: a warp each, or fewer heads that share the warps.
template <int D, int NT>
pl::Kv4Plan kv4_plan(int hkv) {
  using C = pl::Kv4Cfg<D, NT>;
  pl::Kv4Plan p;
  p.heads = hkv < C::kWarps ? hkv : C::kWarps;
  p.share = 1;
  while (2 * p.share * p.heads <= C::kWarps) p.share *= 2;
  return p;
}

template <int D, int NT>
int32_t launch_kv4(const void* cache, pl::LineArgs& a, void* stream) {
  using C = pl::Kv4Cfg<D, NT>;
  const pl::Kv4Plan p = kv4_plan<D, NT>(a.num_kv_heads);
  a.item_heads = p.heads;
  a.items = (a.num_kv_heads + p.heads - 1) / p.heads;
  a.ctas = C::kCtas * pl_host::sm_count();
  auto kern = pl::kv4_decode_kernel<D, NT>;
  int32_t st = pl_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (st != PL_OK) return st;
  st = pl_host::launch_pdl(kern, dim3(a.ctas), dim3(C::kThreads), C::kSmemBytes, stream,
                           static_cast<const uint8_t*>(cache), a, p);
  if (st != PL_OK) return st;
  return pl_host::launch_line_finish<D>(a, stream);
}

}  // namespace

extern "C" int64_t pl_kv4_decode_workspace_bytes(int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || head_dim <= 0) return 0;
  const int ctas = pl_host::sm_count() > 0 ? pl_host::sm_count() : 148;
  const int heads = num_kv_heads < 8 ? num_kv_heads : 8;
  return align256(pl_host::line_partial_bytes(2 * ctas, heads * (num_qo_heads / num_kv_heads), head_dim));
}

extern "C" int32_t pl_paged_kv4_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv4_cache,
                                       int64_t num_pages, const int32_t* indptr, const int32_t* indices,
                                       const int32_t* last_page_len, int64_t total_pages, int32_t batch,
                                       int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                       int32_t page_size, float sm_scale, int32_t window, int32_t sinks, void* out,
                                       int64_t o_stride_b, int64_t o_stride_h, float* out_lse, void* workspace,
                                       int64_t workspace_bytes, int32_t* status_dev, void* stream) {
  int32_t st = pl_host::line_check(q, q_stride_b, q_stride_h, kv4_cache, num_pages, indptr, indices, last_page_len,
                                   total_pages, batch, num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale,
                                   window, sinks, out, o_stride_b, o_stride_h);
  if (st != PL_OK) return st;
  if (batch == 0) return PL_OK;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < pl_kv4_decode_workspace_bytes(num_qo_heads, num_kv_heads, head_dim))
    return PL_ERR_WORKSPACE_TOO_SMALL;
  if (pl_host::sm_count() <= 0) return PL_ERR_NO_DEVICE;
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
  a.num_qo_heads = num_qo_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_qo_heads / num_kv_heads;
  a.page_size = page_size;
  a.window = window;
  a.sinks = sinks;
  a.pad = 2;
  a.min_tiles = 4;
  a.scale_log2 = sm_scale * pl::kLog2e;
  a.out = static_cast<pl::bf16*>(out);
  a.o_stride_b = o_stride_b;
  a.o_stride_h = o_stride_h;
  a.out_lse = out_lse;
  a.partial = static_cast<float*>(workspace);
  a.status = status_dev;
  if (head_dim == 128)
    return a.group <= 8 ? launch_kv4<128, 1>(kv4_cache, a, stream) : launch_kv4<128, 2>(kv4_cache, a, stream);
  return a.group <= 8 ? launch_kv4<64, 1>(kv4_cache, a, stream) : launch_kv4<64, 2>(kv4_cache, a, stream);
}

extern "C" int32_t pl_kv4_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* kv4_cache,
                                 int64_t num_pages, const int32_t* page_id, const int32_t* page_offset,
                                 int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                 int32_t* status_dev, void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || page_size <= 0 || num_pages <= 0 || kv4_cache == nullptr)
    return PL_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return PL_ERR_UNSUPPORTED;
  if (num_tokens == 0) return PL_OK;
  if (k == nullptr || v == nullptr || page_id == nullptr || page_offset == nullptr) return PL_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(kv4_cache)) & 15) !=
          0 || k_stride % 8 != 0 || v_stride % 8 != 0)
    return PL_ERR_INVALID_ARGUMENT;
  const int64_t records = (int64_t)num_tokens * 2 * num_kv_heads, blocks = (records + 31) / 32;
  if (records > 0x7FFFFFFF) return PL_ERR_UNSUPPORTED;
  auto kern = head_dim == 128 ? pl::kv4_append_kernel<128> : pl::kv4_append_kernel<64>;
  return pl_host::launch_pdl(kern, dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const pl::bf16*>(k),
                             k_stride, static_cast<const pl::bf16*>(v), v_stride, static_cast<uint8_t*>(kv4_cache),
                             num_pages, page_id, page_offset, num_tokens, num_kv_heads, page_size, status_dev);
}

extern "C" int32_t pl_kv4_expand(const void* kv4_cache, int64_t num_pages, const int32_t* page_ids, int32_t n,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t page_size, void* out,
                                 int32_t* status_dev, void* stream) {
  if (n < 0 || num_kv_heads <= 0 || page_size <= 0 || num_pages <= 0 || kv4_cache == nullptr)
    return PL_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128) || page_size % 16 != 0) return PL_ERR_UNSUPPORTED;
  if (n == 0) return PL_OK;
  if (page_ids == nullptr || out == nullptr ||
      ((reinterpret_cast<uintptr_t>(kv4_cache) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return PL_ERR_INVALID_ARGUMENT;
  const int64_t per_page = 2ll * page_size * num_kv_heads;
  const int64_t blocks = n * (per_page / 32);
  if (blocks > 0x7FFFFFFF || per_page > 0x7FFFFFFF) return PL_ERR_UNSUPPORTED;
  auto kern = head_dim == 128 ? pl::kv4_expand_kernel<128> : pl::kv4_expand_kernel<64>;
  return pl_host::launch_pdl(kern, dim3((unsigned)blocks), dim3(256), 0, stream,
                             static_cast<const uint8_t*>(kv4_cache), num_pages, page_ids, (int32_t)per_page,
                             static_cast<pl::bf16*>(out), status_dev);
}
