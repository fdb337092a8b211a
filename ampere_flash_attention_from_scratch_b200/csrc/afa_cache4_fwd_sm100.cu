// afa_cache4_fwd_sm100.cu -- attention over the paged 4-bit cache
// (afa_cache4_fwd_sm100, include/afa_sm100_ops.h).
//
// Mathematics.  With K = s c + m and V = s' c' + m' (codes c, one s and m for a
// token and group g of 64 channels), none of the 4-bit values is ever expanded:
//   score = sum_g [ s_g (q_g . c_g) + m_g sum(q_g) ]
//   O     = sum_t p_t s'_tg c'_t + sum_t p_t m'_tg
// so the matrix instructions multiply codes by 16-bit queries and by p s', and
// the steps and minima are a few fp32 operations a score.  A code masked in
// place, with no shift or conversion, is a subnormal fp16 number: the bits
// 0x000c are c 2^-24 and 0x00c0 are c 2^-20, exactly, and mma.sync takes
// subnormals.  One AND makes two operands.
//
//   * q is held in fp16 for either type, each row scaled by a power of two so
//     that its largest element lies in [2^13, 2^14); the product is exact.
//   * p s' is rounded to fp16: 2^-11 relative, as for a 16-bit P.  The exponent of
//     p is measured by the largest product p s' of the tokens the row has seen, which
//     stays between 2^7 and 2^15: products down to 2^-21 of it keep all their bits,
//     smaller ones are off by 2^-32 of it.
//   * p, its sum, the running maximum and both accumulators are fp32.
//
// Bound.  HBM would be: 1.125 bytes a channel and token for keys and values.  The
// kernel gets to 70 to 80 % of it for long contexts: 16 tokens of 128 channels take a
// warp 273 instructions -- some 75 masks, 25 shifts and permutes, 16 matrix
// instructions, 45 fp32 operations -- in 510 cycles of a sub-partition with as many
// warps as fit, from L2 or from HBM alike.  No one pipe is full (ALU 52 %, HMMA 26 %,
// issue slots 55 %): a mask takes 2 cycles and a matrix instruction 8, under which fp32
// operations find half their room (microbench/mma_sync_beside_alu.cu), and three warps
// do not fill the gaps.  Hence tokens on the M side of mma.m16n8k16 (16 tokens x 8 query
// rows): one row and eight cost the same, and no lane idles on a row block padded
// to 128, for which the codes would also have to be spread in shared memory.
// Measured: [8 x 131072 tokens, 32/8 heads, 128] bf16 261 us among other work = 4.6 TB/s
// (71 % of the measured copy bandwidth), 231 us in calls in a row (a version that took
// 240 took 203 with the arithmetic left out); among other work [32 x 256..8192, 32/8,
// 128] bf16 41 us = 3.8 TB/s, [16 x 250..4001, 32/32, 64] fp16 31 us = 2.6 TB/s (one
// of eight columns used, half the channels for the same softmax), [16 x 1024..16384, 5
// new tokens, 64/8, 128] fp16 154 us (three blocks of 16 rows; at 16 rows and head_dim
// 128 a thread has all 255 registers, and in bf16 20 bytes of them are spilled).
// 500 tokens: 8.3 us on the device, the work's division, two dependent loads and
// four steps of a warp.  4 CTAs an SM instead of 3 and 4 steps in the ring instead of 3: equal
// to 3 % slower.
//
// Work.  The (sequence, key/value head, row block) items are cut into units of
// kUnit tokens and the units dealt out evenly to the CTAs in one contiguous
// range each, from the lengths on the device: ragged batches stay balanced and
// the host never waits for a length.  A CTA that does not see an item's whole
// range leaves its share (unnormalised O, maximum, sum) in the workspace, and a
// second small kernel joins the shares in a fixed order.
#include <cmath>
#include <type_traits>

#include "afa_cache4_fwd_common.cuh"
#include "afa_cache4_wide_kernel.cuh"

namespace {

using namespace afa100;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 32;               // tokens of a warp's step
static_assert(kUnit == kWarps * kStep, "a unit is one step of every warp");
constexpr int kStages = 3;              // steps of a warp's ring, one less in flight

__device__ __forceinline__ uint32_t lds32(const char* a) { return *reinterpret_cast<const uint32_t*>(a); }
__device__ __forceinline__ uint2 lds64(const char* a) { return *reinterpret_cast<const uint2*>(a); }
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero: d = a b.
__device__ __forceinline__ void mma16816_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// With m's bits: the bits of w, or those of 15 - w where x has them too; without
// them: x.  One three-input operation.
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t m, uint32_t x) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(m), "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) { return pack2<false>(lo, hi); }

__device__ __forceinline__ float max_over_rows(float v) {  // over the eight lanes of equal lane % 4
#pragma unroll
  for (int i = 4; i < 32; i <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, i));
  return v;
}
__device__ __forceinline__ float sum_over_rows(float v) {
#pragma unroll
  for (int i = 4; i < 32; i <<= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
  return v;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
template <int kD, int kNT>
struct FwdLayout4 {
  static constexpr int kGroups = kD / 64;
  static constexpr int kRow = kD / 2 + kD / 16;
  static constexpr int kRows = kNT * 8;
  static constexpr int kSideBytes = kStep * kRow;      // keys, or values, of a step
  static constexpr int kStageBytes = 2 * kSideBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kShareBytes = kRows * kD * 4;   // a warp's O
  // A warp's O fits the stage it has just used, or has memory of its own.
  static constexpr bool kInStage = kShareBytes <= kStageBytes;
  static constexpr int kStats = kWarps * (kWarpBytes + (kInStage ? 0 : kShareBytes));
  static constexpr int kSmem = kStats + kWarps * kRows * 2 * 4 + kWarps * 4;
  static constexpr int kShare = kRows * (kD + 2);      // floats of a CTA's share of an item
};

template <int kD, bool kBF16, int kNT>
__global__ void __launch_bounds__(kThreads, kNT == 1 || kD == 64 ? 3 : 2) cache4_fwd_kernel(const FwdParams4 p) {
  using L = FwdLayout4<kD, kNT>;
  constexpr int kG = L::kGroups;
  constexpr int kRow = L::kRow;
  extern __shared__ __align__(16) char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * L::kWarpBytes;
  float* stats = reinterpret_cast<float*>(smem + L::kStats);                 // [warp][row][m, l]
  uint32_t* places = reinterpret_cast<uint32_t*>(stats + kWarps * L::kRows * 2);  // [warp] where its O is

  after_previous();  // and the join may take the SMs as they fall free
  Walk w;
  {
    const int per = (p.c.batch + 31) / 32;
    int before_lane;
    const Division div = divide(p, per, gridDim.x, &before_lane);
    const int cta = static_cast<int>(blockIdx.x);
    if (cta >= div.ctas) return;
    w.it = find_item(p, per, before_lane, div.first(cta));
    w.left = div.first(cta + 1) - div.first(cta);
    w.open(p, warp * kStep);
  }
  // Past pieces that are only the cost of an item whose tokens another CTA has; false at the end.
  auto skip_empty = [&](Walk& walk) {
    bool go = true;
    while (go && walk.unit_end <= p.item_units) go = walk.next(p, warp * kStep);
    return go;
  };

  if (!skip_empty(w)) return;

  // The queries of a piece, loaded before the arithmetic of the one before it is finished.
  uint4 raw[kNT][kG][2];
  auto load_queries = [&]() {
    const int head = w.it.which / p.row_tiles, tile = w.it.which - head * p.row_tiles;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int r = tile * L::kRows + nt * 8 + g;
      const int i = r / p.group, h = head * p.group + (r - i * p.group);
      const char* src = p.q + w.it.b * p.q_s[0] + i * p.q_s[1] + h * p.q_s[2] + t * 32;
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          raw[nt][gr][x] = make_uint4(0, 0, 0, 0);
          if (r < p.rows) raw[nt][gr][x] = *reinterpret_cast<const uint4*>(src + gr * 128 + x * 16);
        }
    }
  };
  load_queries();

  // --- loads run ahead of the arithmetic, through the ends of pieces -----------------------------------
  // A step is 32 tokens of keys and of values, from one page or from two of 16
  // tokens.  Lane i looks up the pages of the i-th step from the last look-up on.
  Walk ahead = w;
  bool more = true;
  const char* side = nullptr;  // the head of the piece the loads are in, in page 0
  const bool small_pages = p.c.page_size < kStep;
  int page[2] = {0, 0}, page_step = 0;
  auto look_up = [&]() {
    page_step = 0;
    const int at = ahead.tok + lane * kUnit;
    const int* table = p.c.page_table + ahead.it.b * p.c.table_stride;
    if (at < ahead.tok_end) page[0] = table[at >> p.page_shift];
    if (small_pages && at + 16 < ahead.tok_end) page[1] = table[(at + 16) >> p.page_shift];
  };
  // To the next piece with tokens for this warp, if the loads have reached the end of theirs.
  auto settle = [&]() {
    while (more && ahead.tok >= ahead.tok_end) more = ahead.next(p, warp * kStep);
    if (more) {
      const int head = ahead.it.which / p.row_tiles;
      side = static_cast<const char*>(p.c.cache) + static_cast<int64_t>(head) * 2 * p.c.page_size * kRow + lane * 16;
      look_up();
    }
  };
  // `tokens` rows from place `at` of a page: keys to dst, values kSideBytes behind
  auto copy = [&](auto tokens, int pg, uint32_t at, uint32_t dst) {
    constexpr int kBytes = decltype(tokens)::value * kRow;
    uint32_t bytes = 16;
    if (static_cast<uint32_t>(pg) >= static_cast<uint32_t>(p.c.n_pages)) {
      report(p.c.status, AFA_DEV_BAD_PAGE);  // zeros in place of a page that does not exist
      pg = 0;
      bytes = 0;
    }
    const char* keys = far(far(side, pg, p.page_stride), at, kRow);
    const char* values = far(keys, p.c.page_size, kRow);
#pragma unroll
    for (int x = 0; x < kBytes; x += 512)
      if (x + 512 <= kBytes || lane * 16 + x < kBytes) {
        cp_async16(dst + x, keys + x, bytes);
        cp_async16(dst + L::kSideBytes + x, values + x, bytes);
      }
  };
  auto load = [&](uint32_t dst) {  // dst: the stage, and this lane's 16 bytes of it
    if (more) {
      const int pg = __shfl_sync(0xffffffffu, page[0], page_step);
      if (!small_pages) {
        copy(std::integral_constant<int, kStep>{}, pg, ahead.tok & (p.c.page_size - 1), dst);
      } else {
        const int pg1 = __shfl_sync(0xffffffffu, page[1], page_step);
        copy(std::integral_constant<int, 16>{}, pg, 0, dst);
        if (ahead.tok + 16 < ahead.tok_end) copy(std::integral_constant<int, 16>{}, pg1, 0, dst + 16 * kRow);
      }
      ahead.tok += kUnit;
      if (ahead.tok >= ahead.tok_end)
        settle();
      else if (++page_step == 32)
        look_up();
    }
    cp_async_commit();
  };
  settle();
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) load(ring + s * L::kStageBytes + lane * 16);
  int stage = 0;  // of the next step; the one before it is free

  for (;;) {
    const Item it = w.it;
    const int head = it.which / p.row_tiles, tile = it.which - head * p.row_tiles;
    const bool starts = it.unit <= p.item_units, whole = starts && w.unit_end == it.units;
    const int fresh = p.c.new_lens != nullptr ? p.c.new_lens[it.b] : p.seq_len;

    // --- queries: rows on the N side, their channels in the order the codes come ------------------------
    uint32_t qf[kNT][kG][8];
    float a_of[kNT][2], qs[kNT][kG][2];
    int limit[kNT][2];
    int limit_min = it.tokens;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float big = 0.0f, sum[kG];
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        sum[gr] = 0.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t v4[4] = {raw[nt][gr][x].x, raw[nt][gr][x].y, raw[nt][gr][x].z, raw[nt][gr][x].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = unpack2<kBF16>(v4[e]);
            big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
            sum[gr] += v.x + v.y;
          }
        }
      }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], x);
      }
      // 2^e with e = 13 - floor(log2(big)), from the exponent field; within fp32's normal range
      int e = big > 0.0f ? 13 + 127 - static_cast<int>(__float_as_uint(big) >> 23) : 0;
      e = e > 90 ? 90 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * 16777216.0f * p.scale_log2;
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t v4[4] = {raw[nt][gr][x].x, raw[nt][gr][x].y, raw[nt][gr][x].z, raw[nt][gr][x].w};
          float v[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = unpack2<kBF16>(v4[y]);
            v[2 * y] = f.x * up;
            v[2 * y + 1] = f.y * up;
          }
          // odd channels' codes come as c 2^-20
          qf[nt][gr][x * 4 + 0] = half2_of(v[0], v[4]);
          qf[nt][gr][x * 4 + 1] = half2_of(v[1] * 0.0625f, v[5] * 0.0625f);
          qf[nt][gr][x * 4 + 2] = half2_of(v[2], v[6]);
          qf[nt][gr][x * 4 + 3] = half2_of(v[3] * 0.0625f, v[7] * 0.0625f);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int from = (2 * t + x) * 4;
        a_of[nt][x] = __shfl_sync(0xffffffffu, down, from);
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) qs[nt][gr][x] = __shfl_sync(0xffffffffu, sum[gr] * p.scale_log2, from);
        // tokens the row sees; rows that are not there see all, and are not written
        const int rr = tile * L::kRows + nt * 8 + 2 * t + x;
        limit[nt][x] = rr < p.rows && p.causal ? min(it.tokens, max(0, it.tokens - fresh + rr / p.group + 1)) : it.tokens;
      }
    }
    if (p.causal) limit_min = min(it.tokens, max(0, it.tokens - fresh + tile * L::kRows / p.group + 1));

    // --- the walk over the tokens ------------------------------------------------------------------------
    // A weight is held as p = 2^(score + off): off takes off the row's reference (none yet: -inf), so that p s' stays
    // within 2^(kRescale + kHeadroom).
    float ref[kNT][2], off[kNT][2], limit_s[kNT][2], l[kNT][2];
    float step_max = 0.0f;
    float acc[kNT][kG][4][4], acc_m[kNT][kG][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        ref[nt][x] = limit_s[nt][x] = -INFINITY;
        off[nt][x] = l[nt][x] = 0.0f;
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          acc_m[nt][gr][x] = 0.0f;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) acc[nt][gr][mt][x] = acc[nt][gr][mt][2 + x] = 0.0f;
        }
      }

    // Values' codes are multiplied with a mean taken off, which m' gives back: the accumulators then stay near the
    // result instead of growing with the 7.5 s' a token that m' would take off at the end -- their roundings with
    // them, which the matrix instruction makes towards zero.  For an fp16 result 8 from every code, by an exact
    // fp16 subtraction (relative error 2.9e-4 against 5.5e-4 without; the output's own rounding is 2.1e-4).  For
    // bf16 (1.7e-3) 15 from odd tokens only, which costs nothing and leaves the sum's mean near zero as well.
    const float taken = g & 1 ? 15.0f : 0.0f;

    // 16 tokens from tok0 on, at `kb` (keys) and behind them (values)
    auto compute = [&](auto masked_tag, int tok0, const char* kb) {
      constexpr bool kMasked = decltype(masked_tag)::value;
      float s[kNT][4];
      float vs[2][kG], vm[2][kG];  // s' and what m' becomes (below) of tokens g, g + 8
      float vs_max = 0.0f;
      {
        uint32_t par[2][2][kG];  // keys, values; tokens g, g + 8
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const char* a = kb + kv * L::kSideBytes + (g + 8 * y) * kRow + kD / 2;
            if constexpr (kG == 2) {
              const uint2 v = lds64(a);
              par[kv][y][0] = v.x;
              par[kv][y][1] = v.y;
            } else {
              par[kv][y][0] = lds32(a);
            }
          }
        float part[kNT][4], mins[kNT][4];
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          uint32_t v[2][2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const char* a = kb + (g + 8 * y) * kRow + gr * 32 + t * 8;
            if constexpr (kG == 2) {
              const uint2 x = lds64(a);
              v[y][0] = x.x;
              v[y][1] = x.y;
            } else {  // rows of 36 bytes: 4-byte loads
              v[y][0] = lds32(a);
              v[y][1] = lds32(a + 4);
            }
          }
          float dot[kNT][4];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t lo = v[0][x] >> (8 * z), hi = v[1][x] >> (8 * z);
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt) {
                const uint32_t b0 = qf[nt][gr][x * 4 + z * 2], b1 = qf[nt][gr][x * 4 + z * 2 + 1];
                if (x == 0 && z == 0)
                  mma16816_new(dot[nt], lo & 0x000f000fu, hi & 0x000f000fu, lo & 0x00f000f0u, hi & 0x00f000f0u, b0, b1);
                else
                  mma16816(dot[nt], lo & 0x000f000fu, hi & 0x000f000fu, lo & 0x00f000f0u, hi & 0x00f000f0u, b0, b1);
              }
            }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float2 sm = unpack2<kBF16>(par[0][y][gr]);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                part[nt][2 * y + x] = gr == 0 ? sm.x * dot[nt][2 * y + x] : fmaf(sm.x, dot[nt][2 * y + x], part[nt][2 * y + x]);
                mins[nt][2 * y + x] = fmaf(sm.y, qs[nt][gr][x], gr == 0 ? off[nt][x] : mins[nt][2 * y + x]);
              }
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int at = tok0 + g + 8 * y;
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float v = fmaf(a_of[nt][x], part[nt][2 * y + x], mins[nt][2 * y + x]);
              if (kMasked && at >= limit[nt][x]) v = -INFINITY;
              s[nt][2 * y + x] = v;
            }
#pragma unroll
          for (int gr = 0; gr < kG; ++gr) {
            float2 sm = unpack2<kBF16>(par[1][y][gr]);
            if (kMasked && at >= it.tokens) sm = make_float2(0.0f, 0.0f);  // not a token: whatever the page held
            vs[y][gr] = sm.x;
            vm[y][gr] = fmaf(kBF16 ? taken : 8.0f, sm.x, sm.y);
            vs_max = fmaxf(vs_max, fabsf(sm.x));
          }
        }
      }

      // A row's reference moves where p s' of a token it sees would pass 2^(kRescale + kHeadroom).  As long as no step
      // passes step_max (a power of two), no score above limit_s tells that; otherwise the products are looked at.
      // What a row does not see moves nothing but step_max.
      bool look = vs_max > step_max;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) look |= fmaxf(s[nt][x], s[nt][2 + x]) > limit_s[nt][x];
      if (__any_sync(0xffffffffu, look)) {
        float size[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          size[y] = kLeastSize;
#pragma unroll
          for (int gr = 0; gr < kG; ++gr) size[y] = size_of(size[y], vs[y][gr], vm[y][gr]);
        }
        const float seen = max_over_rows(fmaxf(size[0], size[1]));
        if (seen > step_max) step_max = power_above(seen);
        const float limit = kRescale + kHeadroom - log2_of_power(step_max);
        size[0] = lg2_approx(size[0]);
        size[1] = lg2_approx(size[1]);
        float top[kNT][2];
        bool passes = false;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            top[nt][x] = fmaxf(s[nt][x] + size[0], s[nt][2 + x] + size[1]);
            passes |= top[nt][x] > (ref[nt][x] == -INFINITY ? -INFINITY : kRescale + kHeadroom);
            if (ref[nt][x] != -INFINITY) limit_s[nt][x] = limit;
          }
        if (__any_sync(0xffffffffu, passes)) {
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float most = max_over_rows(top[nt][x]);
              const bool none = ref[nt][x] == -INFINITY;
              const bool pass = most > (none ? -INFINITY : kRescale + kHeadroom);
              const float to = pass ? kHeadroom - (most - off[nt][x]) : off[nt][x], shift = to - off[nt][x];
              // as a square, since steps that grow by more than 2^126 leave weights that still count
              const float by = none ? 1.0f : ex2_approx(0.5f * shift);
              if (pass) {
                limit_s[nt][x] = limit;
                ref[nt][x] = most - off[nt][x];
              }
              off[nt][x] = to;
              s[nt][x] += shift;
              s[nt][2 + x] += shift;
              l[nt][x] = l[nt][x] * by * by;
#pragma unroll
              for (int gr = 0; gr < kG; ++gr) {
                acc_m[nt][gr][x] = acc_m[nt][gr][x] * by * by;
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                  acc[nt][gr][mt][x] = acc[nt][gr][mt][x] * by * by;
                  acc[nt][gr][mt][2 + x] = acc[nt][gr][mt][2 + x] * by * by;
                }
              }
            }
        }
      }

      const char* vb = kb + L::kSideBytes;
      uint32_t pf[kNT][kG][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float pr[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          pr[x] = ex2_approx(s[nt][x]);
          l[nt][x & 1] += pr[x];
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float ps[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float pp = pr[2 * y + x];
              ps[x] = pp * vs[y][gr];
              float mm = vm[y][gr];
              if (kMasked && tok0 + g + 8 * y >= limit[nt][x]) {  // its s' and m' may be NaN
                ps[x] = 0.0f;
                mm = 0.0f;
              }
              acc_m[nt][gr][x] = fmaf(pp, mm, acc_m[nt][gr][x]);
            }
            pf[nt][gr][y] = transpose8x8(half2_of(ps[0], ps[1]));
          }
      }
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        // rows of tokens 2t, 2t + 1, 2t + 8, 2t + 9; channels 8g .. 8g + 7 of the group
        const char* a = vb + 2 * t * kRow + gr * 32 + g * 4;
        const uint32_t w0 = lds32(a), w1 = lds32(a + kRow), w2 = lds32(a + 8 * kRow), w3 = lds32(a + 9 * kRow);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t sel = z ? 0x7632u : 0x5410u;
          const uint32_t lo = __byte_perm(w0, w1, sel), hi = __byte_perm(w2, w3, sel);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t lo8 = lo >> (8 * y), hi8 = hi >> (8 * y);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              float(&d)[4] = acc[nt][gr][2 * z + y];
              const uint32_t b0 = pf[nt][gr][0], b1 = pf[nt][gr][1];
              if constexpr (kBF16) {
                // c' and c' - 15 by turns (odd tokens, the high halves)
                mma16816(d, pick(lo8, 0x000f000fu, 0x800f0000u), pick(lo8, 0x00f000f0u, 0x80f00000u),
                         pick(hi8, 0x000f000fu, 0x800f0000u), pick(hi8, 0x00f000f0u, 0x80f00000u), b0, b1);
              } else {
                // c' - 8, and 16 times that
                mma16816(d, sub2(pick(lo8, 0x000f000fu, 0x64006400u), 0x64086408u),
                         sub2(pick(lo8, 0x00f000f0u, 0x64006400u), 0x64806480u),
                         sub2(pick(hi8, 0x000f000fu, 0x64006400u), 0x64086408u),
                         sub2(pick(hi8, 0x00f000f0u, 0x64006400u), 0x64806480u), b0, b1);
              }
            }
          }
        }
      }
    };

    for (; w.tok < w.tok_end; w.tok += kUnit) {
      cp_async_wait<kStages - 2>();
      __syncwarp();  // every lane's part of the step has landed, and the stage loaded next has been read
      load(ring + (stage == 0 ? kStages - 1 : stage - 1) * L::kStageBytes + lane * 16);
      const char* base = smem + warp * L::kWarpBytes + stage * L::kStageBytes;
      if (w.tok + kStep <= limit_min) {
        compute(std::false_type{}, w.tok, base);
        compute(std::false_type{}, w.tok + 16, base + 16 * kRow);
      } else {
#pragma unroll 1
        for (int c = 0; c < 2 && w.tok + 16 * c < w.tok_end; ++c)
          compute(std::true_type{}, w.tok + 16 * c, base + c * 16 * kRow);
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    __syncwarp();

    const bool go = w.next(p, warp * kStep) && skip_empty(w);
    if (go) load_queries();

    // --- the warps' shares -> the CTA's -------------------------------------------------------------------
    const uint32_t place = L::kInStage ? warp * L::kWarpBytes + (stage == 0 ? kStages - 1 : stage - 1) * L::kStageBytes
                                       : kWarps * L::kWarpBytes + warp * L::kShareBytes;
    float* mine = reinterpret_cast<float*>(smem + place);  // [row][channel]
    if (lane == 0) places[warp] = place;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = nt * 8 + 2 * t + x;
        const float sum = sum_over_rows(l[nt][x]);
        if (g == 0) {
          stats[(warp * L::kRows + row) * 2] = ref[nt][x] == -INFINITY ? -INFINITY : -off[nt][x];
          stats[(warp * L::kRows + row) * 2 + 1] = sum;
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const float mn = sum_over_rows(acc_m[nt][gr][x]);
          // what the codes' places left out
          const float even = kBF16 ? 16777216.0f : 1.0f, odd = kBF16 ? 1048576.0f : 0.0625f;
          float* dst = mine + row * kD + gr * 64 + g * 8;
#pragma unroll
          for (int mt = 0; mt < 4; mt += 2)
            *reinterpret_cast<float4*>(dst + 2 * mt) =
                make_float4(fmaf(acc[nt][gr][mt][x], even, mn), fmaf(acc[nt][gr][mt][2 + x], odd, mn),
                            fmaf(acc[nt][gr][mt + 1][x], even, mn), fmaf(acc[nt][gr][mt + 1][2 + x], odd, mn));
        }
      }
    __syncthreads();
    // A range that starts within an item is the CTA's first, one that ends within an item its last.
    float* share = p.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (starts ? 1 : 0)) * L::kShare;
    for (int i = threadIdx.x; i < L::kRows * (kD / 4); i += kThreads) {
      const int row = i / (kD / 4), c4 = i - row * (kD / 4);
      float m[kWarps], top = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        m[v] = stats[(v * L::kRows + row) * 2];
        top = fmaxf(top, m[v]);
      }
      float sum = 0.0f;
      float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        // a square, as above
        const float by = m[v] == -INFINITY && top == -INFINITY ? 1.0f : ex2_approx(0.5f * (m[v] - top));
        sum = fmaf(by, by * stats[(v * L::kRows + row) * 2 + 1], sum);
        const float4 f = *reinterpret_cast<const float4*>(smem + places[v] + (row * kD + c4 * 4) * 4);
        o.x = fmaf(by, by * f.x, o.x);
        o.y = fmaf(by, by * f.y, o.y);
        o.z = fmaf(by, by * f.z, o.z);
        o.w = fmaf(by, by * f.w, o.w);
      }
      const int r = tile * L::kRows + row;
      if (whole) {
        if (r < p.rows) {
          const int n = r / p.group, h = head * p.group + (r - n * p.group);
          const bool some = n < fresh && !(sum == 0.0f);
          const float inv = some ? 1.0f / sum : 0.0f;
          uint2 v = make_uint2(0, 0);
          if (some) v = make_uint2(pack2<kBF16>(o.x * inv, o.y * inv), pack2<kBF16>(o.z * inv, o.w * inv));
          *reinterpret_cast<uint2*>(p.o + it.b * p.o_s[0] + n * p.o_s[1] + h * p.o_s[2] + c4 * 8) = v;
          if (p.lse != nullptr && c4 == 0)
            p.lse[(static_cast<int64_t>(it.b) * p.n_heads + h) * p.seq_len + n] =
                some ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
        }
      } else {
        *reinterpret_cast<float4*>(share + row * kD + c4 * 4) = o;
        if (c4 == 0) {
          share[L::kRows * kD + row * 2] = top;
          share[L::kRows * kD + row * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();  // the shares have been read: their memory takes the next steps
    if (!go) break;
  }
  cp_async_wait<0>();
}

// Joins the shares of the items that several CTAs worked on: CTA i takes the
// item its range starts within, if the CTA before it holds that item's start;
// one warp a row (blockIdx.y).  The shares are added in the order of the CTAs.
// Launched while the first kernel still runs: it finds its item meanwhile and
// waits for that kernel's end before it reads a share.
template <int kD, bool kBF16, int kNT>
__global__ void __launch_bounds__(128) cache4_join_kernel(const FwdParams4 p) {
  using L = FwdLayout4<kD, kNT>;
  constexpr int kPer = kD / 32;  // channels of a lane
  const int lane = threadIdx.x & 31;
  const int per = (p.c.batch + 31) / 32;
  int before_lane;
  const Division div = divide(p, per, gridDim.x + 1, &before_lane);
  const int cta = blockIdx.x + 1;
  bool mine = cta < div.ctas;
  int head = 0, tile = 0, fresh = 0, last = 0, b = 0;
  if (mine) {
    const int u = div.first(cta);
    const Item it = find_item(p, per, before_lane, u);
    const int begin = u - it.unit + p.item_units, end = u - it.unit + it.units;  // of the tokens' units
    mine = u > begin && div.first(cta - 1) <= begin;
    head = it.which / p.row_tiles;
    tile = it.which - head * p.row_tiles;
    b = it.b;
    fresh = p.c.new_lens != nullptr ? p.c.new_lens[b] : p.seq_len;
    last = div.holder(end - 1);
  }
  // (The next kernel's CTAs are not let in before the end: [32 x 8192, 32/8, 128] calls in a row 41.2 us, else 44.8.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!mine) return;
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5), r = tile * L::kRows + row;
  if (r >= p.rows) return;
  auto share = [&](int i) { return p.ws + (static_cast<int64_t>(i) * 2 + (i == cta - 1 ? 1 : 0)) * L::kShare; };
  // in one pass, so that no load waits for the maximum
  float top = -INFINITY, sum = 0.0f, o[kPer];
#pragma unroll
  for (int x = 0; x < kPer; ++x) o[x] = 0.0f;
#pragma unroll 8
  for (int i = cta - 1; i <= last; ++i) {
    const float* sh = share(i);
    const float2 ml = *reinterpret_cast<const float2*>(sh + L::kRows * kD + row * 2);
    const float now = fmaxf(top, ml.x);
    // (squares of these, as in the first kernel)
    const float old = now == -INFINITY ? 1.0f : ex2_approx(0.5f * (top - now));
    const float by = now == -INFINITY ? 1.0f : ex2_approx(0.5f * (ml.x - now));
    top = now;
    sum = fmaf(by, by * ml.y, sum * old * old);
#pragma unroll
    for (int x = 0; x < kPer; x += 2) {
      const float2 v = *reinterpret_cast<const float2*>(sh + row * kD + lane * kPer + x);
      o[x] = fmaf(by, by * v.x, o[x] * old * old);
      o[x + 1] = fmaf(by, by * v.y, o[x + 1] * old * old);
    }
  }
  const int n = r / p.group, h = head * p.group + (r - n * p.group);
  const bool some = n < fresh && !(sum == 0.0f);
  const float inv = some ? 1.0f / sum : 0.0f;
  char* dst = p.o + b * p.o_s[0] + n * p.o_s[1] + h * p.o_s[2] + lane * kPer * 2;
#pragma unroll
  for (int x = 0; x < kPer; x += 2)
    *reinterpret_cast<uint32_t*>(dst + x * 2) = some ? pack2<kBF16>(o[x] * inv, o[x + 1] * inv) : 0u;
  if (p.lse != nullptr && lane == 0)
    p.lse[(static_cast<int64_t>(b) * p.n_heads + h) * p.seq_len + n] =
        some ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Kernel4 {
  int rows, share_floats;
  cudaError_t (*prepare)(int* ctas_per_sm);
  cudaError_t (*launch)(const FwdParams4&, unsigned grid, cudaStream_t);
};

template <int kD, bool kBF16, int kNT>
cudaError_t prepare4(int* ctas_per_sm) {
  using L = FwdLayout4<kD, kNT>;
  cudaError_t e = cudaFuncSetAttribute(cache4_fwd_kernel<kD, kBF16, kNT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       L::kSmem);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas_per_sm, cache4_fwd_kernel<kD, kBF16, kNT>, kThreads,
                                                       L::kSmem);
}

template <int kD, bool kBF16, int kNT>
cudaError_t join4(const FwdParams4& p, unsigned grid, cudaStream_t s) {
  using L = FwdLayout4<kD, kNT>;
  if (grid == 1 || p.item_units == 0) return cudaSuccess;  // one CTA or no split item: no shares
  return ops_launch(cache4_join_kernel<kD, kBF16, kNT>, dim3(grid - 1, L::kRows / 4), 128, 0, s, p);
}

template <int kD, bool kBF16, int kNT>
cudaError_t launch4(const FwdParams4& p, unsigned grid, cudaStream_t s) {
  const cudaError_t e =
      ops_launch(cache4_fwd_kernel<kD, kBF16, kNT>, dim3(grid), kThreads, FwdLayout4<kD, kNT>::kSmem, s, p);
  return e != cudaSuccess ? e : join4<kD, kBF16, kNT>(p, grid, s);
}

// The kernel for many rows; its shares are those of 16 blocks of 8.
template <int kD, bool kBF16>
cudaError_t prepare_wide(int* ctas_per_sm) {
  using L = WideLayout<kD>;
  static_assert(L::kShare == FwdLayout4<kD, 16>::kShare && L::kRows == FwdLayout4<kD, 16>::kRows, "one join for both");
  // By design two CTAs an SM, in registers, shared and tensor memory.  (The occupancy query answers 1 for a kernel
  // that allocates tensor memory.)
  *ctas_per_sm = 2;
  return cudaFuncSetAttribute(cache4_wide_kernel<kD, kBF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
}

template <int kD, bool kBF16>
cudaError_t launch_wide(const FwdParams4& p, unsigned grid, cudaStream_t s) {
  using L = WideLayout<kD>;
  const cudaError_t e = ops_launch(cache4_wide_kernel<kD, kBF16>, dim3(grid), L::kThreads, L::kSmem, s, p);
  return e != cudaSuccess ? e : join4<kD, kBF16, 16>(p, grid, s);
}

#define AFA_KERNEL4(D, BF, NT) \
  { FwdLayout4<D, NT>::kRows, FwdLayout4<D, NT>::kShare, &prepare4<D, BF, NT>, &launch4<D, BF, NT> }
#define AFA_WIDE4(D, BF) \
  { WideLayout<D>::kRows, WideLayout<D>::kShare, &prepare_wide<D, BF>, &launch_wide<D, BF> }
#define AFA_ROWS4(D, BF) \
  { AFA_KERNEL4(D, BF, 1), AFA_KERNEL4(D, BF, 2), AFA_WIDE4(D, BF) }
// [head_dim 64, 128][fp16, bf16][8, 16, 128 rows]
const Kernel4 kKernels4[2][2][3] = {{AFA_ROWS4(64, false), AFA_ROWS4(64, true)},
                                    {AFA_ROWS4(128, false), AFA_ROWS4(128, true)}};

std::mutex g_mu4;
int g_ctas_per_sm[kOpsMaxDevices][2][2][3] = {};

// Kernel, grid and row blocks of a call, and whether its items are not split.
int plan4(const AfaCache4* c, int32_t seq_len, int32_t n_heads, const Kernel4** kernel, int32_t* grid,
          int32_t* row_tiles, bool* whole) {
  int rc = ops_check_cache(c);
  if (rc != AFA_OK) return rc;
  if (seq_len <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads != 0) return AFA_ERR_INVALID_ARGUMENT;
  const int64_t rows = int64_t{seq_len} * (n_heads / c->n_kv_heads);
  if (rows > INT32_MAX - 64) return AFA_ERR_TOO_LARGE;
  // mma.sync repeats its unpacking for every 16 rows; tcgen05 does it once for 128, but starts and ends more slowly.
  // Both, us, 8 key/value heads, fp16:
  //   sequences x tokens      16 x 16384  16 x 4000  16 x 1000  4 x 4000  4 x 1000  1 x 2000
  //   d 128,  48 rows          272 / 286   84 / 100    36 / 53   30 / 45   17 / 33   17 / 27
  //           64               359 / 288  107 / 102    43 / 55   36 / 46   20 / 34   16 / 29
  //          128               703 / 396  201 / 134    76 / 68   60 / 58   26 / 41   18 / 33
  //   d 64,   64               201 / 203    62 / 72    27 / 39   24 / 34   14 / 25   15 / 20
  //          128               388 / 270   112 / 93    44 / 49   37 / 43   19 / 31   15 / 24
  // One border for all is a compromise: it loses up to a fifth at 49 to 64 rows of many long sequences, and up to half
  // at 65 to 128 rows of short ones.  The lengths are on the device; the table's capacity bounds them and would tell.
  const int di = c->head_dim == 128, ti = c->dtype == AFA_DTYPE_BF16, ni = rows > 64 ? 2 : rows > 8;
  const Kernel4& k = kKernels4[di][ti][ni];
  const int64_t tiles = (rows + k.rows - 1) / k.rows;
  if (c->n_pages > 1 && c->page_stride > UINT32_MAX) return AFA_ERR_TOO_LARGE;
  // units are counted in 31 bits
  const int64_t items = tiles * c->n_kv_heads;
  const int64_t units = (int64_t{c->max_pages} * c->page_size + kUnit - 1) / kUnit + kItemUnits;
  if (items > INT32_MAX || items * c->batch > INT32_MAX / units) return AFA_ERR_TOO_LARGE;
  int dev = 0, sms = 0;
  rc = ops_device(&dev, &sms);
  if (rc != AFA_OK) return rc;
  {
    std::lock_guard<std::mutex> lock(g_mu4);
    int& per_sm = g_ctas_per_sm[dev][di][ti][ni];
    if (per_sm == 0) {
      int n = 0;
      if (k.prepare(&n) != cudaSuccess || n < 1) {
        cudaGetLastError();
        return AFA_ERR_LAUNCH;
      }
      per_sm = n;
    }
    *grid = sms * per_sm;
  }
  // Short sequences, few of them: one CTA an item.  The host then launches one kernel instead of two (7.5 us a call
  // instead of 9.8), and on the device 32/8 heads of 128 in bf16 take, split -> whole, us in a row: 32 sequences of
  // 500 tokens 16.4 -> 12.3, 1 of 500 10.2 -> 10.2, 1 of 1000 10.3 -> 12.7.  The tcgen05 kernel keeps the split.
  // It is the table's width that counts: the same 32 sequences by tables of 131072 tokens take 15.2.
  *whole = ni < 2 && int64_t{c->max_pages} * c->page_size <= kWholeTokens && items * c->batch <= *grid;
  // no more CTAs than units at the sequences' largest possible lengths
  const int64_t most = *whole ? items * c->batch : units * items * c->batch;
  if (most < *grid) *grid = static_cast<int32_t>(most);
  *kernel = &k;
  *row_tiles = static_cast<int32_t>(tiles);
  return AFA_OK;
}

}  // namespace

extern "C" {

int64_t afa_cache4_fwd_workspace(const AfaCache4* cache, int32_t seq_len, int32_t n_heads) {
  const Kernel4* k = nullptr;
  int32_t grid = 0, tiles = 0;
  bool whole = false;
  const int rc = plan4(cache, seq_len, n_heads, &k, &grid, &tiles, &whole);
  if (rc != AFA_OK) return -static_cast<int64_t>(rc);
  return int64_t{2} * grid * k->share_floats * static_cast<int64_t>(sizeof(float));
}

int afa_cache4_fwd_sm100(const AfaCache4* cache, const AfaCache4FwdArgs* a, void* stream) {
  int rc = ops_check_cache(cache);
  if (rc != AFA_OK) return rc;
  if (a == nullptr || a->q == nullptr || a->o == nullptr || a->workspace == nullptr ||
      (a->causal != 0 && a->causal != 1) || a->seq_len <= 0 || a->n_heads <= 0 ||
      !(a->scale < 1e38f))  // NaN, or beyond fp32 times log2(e)
    return AFA_ERR_INVALID_ARGUMENT;
  if (!ops_aligned16(a->q) || !ops_aligned16(a->o) || !ops_aligned16(a->workspace) ||
      (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0u ||
      !ops_strides_ok(a->q_strides, cache->batch, a->seq_len, a->n_heads, false) ||
      !ops_strides_ok(a->o_strides, cache->batch, a->seq_len, a->n_heads, true))
    return AFA_ERR_MISALIGNED;
  const Kernel4* k = nullptr;
  int32_t grid = 0, tiles = 0;
  bool whole = false;
  rc = plan4(cache, a->seq_len, a->n_heads, &k, &grid, &tiles, &whole);
  if (rc != AFA_OK) return rc;
  if (a->workspace_bytes < int64_t{2} * grid * k->share_floats * static_cast<int64_t>(sizeof(float)))
    return AFA_ERR_SCRATCH_LIMIT;

  FwdParams4 p{};
  p.c = *cache;
  p.q = static_cast<const char*>(a->q);
  p.o = static_cast<char*>(a->o);
  for (int i = 0; i < 3; ++i) {
    p.q_s[i] = a->q_strides[i] * 2;
    p.o_s[i] = a->o_strides[i] * 2;
  }
  p.lse = a->lse;
  p.ws = static_cast<float*>(a->workspace);
  p.seq_len = a->seq_len;
  p.n_heads = a->n_heads;
  p.group = a->n_heads / cache->n_kv_heads;
  p.rows = a->seq_len * p.group;
  p.row_tiles = tiles;
  p.page_shift = ops_log2(cache->page_size);
  p.page_stride = static_cast<uint32_t>(cache->page_stride);
  p.unit_tokens = whole ? kWholeTokens : kUnit;
  p.item_units = whole ? 0 : kItemUnits;
  p.causal = a->causal;
  p.timeout_ns = a->timeout_ns != 0 ? a->timeout_ns : 4000000000ull;
  p.test_flags = a->test_flags;
  const double scale = a->scale > 0.f ? a->scale : 1.0 / (cache->head_dim == 64 ? 8.0 : 11.313708498984761);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  if (k->launch(p, static_cast<unsigned>(grid), static_cast<cudaStream_t>(stream)) != cudaSuccess) {
    cudaGetLastError();
    return AFA_ERR_LAUNCH;
  }
  return AFA_OK;
}

}  // extern "C"
