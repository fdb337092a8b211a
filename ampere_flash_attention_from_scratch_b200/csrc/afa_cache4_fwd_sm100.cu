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
//   * p s' is rounded to fp16 after a scaling by a power of two a warp keeps for
//     each group (the largest step so far), at most 2^13: relative 2^-12 as for
//     a 16-bit P, with 2^-38 of the largest as the smallest step.
//   * p, its sum, the running maximum and both accumulators are fp32.
//
// Bound: HBM for a few query rows -- 1.125 bytes a channel and token for keys
// and values -- and the issue slots of unpacking and of the softmax beyond
// about 16 rows a key/value head.  Hence: tokens on the M side of
// mma.m16n8k16 (16 tokens x 8 query rows), so that one row and eight cost the
// same and no lane idles on a padded row block of 64 or 128; tcgen05 would need
// the codes expanded into shared memory, 3.6 times the bytes that arrive.
//
// Work.  The (sequence, key/value head, row block) items are cut into units of
// kUnit tokens and the units dealt out evenly to the CTAs in one contiguous
// range each, from the lengths on the device: ragged batches stay balanced and
// the host never waits for a length.  A CTA that does not see an item's whole
// range leaves its share (unnormalised O, maximum, sum) in the workspace, and a
// second small kernel joins the shares in a fixed order.
#include <cmath>
#include <type_traits>

#include "ops_common.cuh"
#include "sm100_ptx.cuh"

namespace {

using namespace afa100;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 32;               // tokens of a warp's step
constexpr int kUnit = kWarps * kStep;   // tokens of a unit
constexpr int kStages = 4;              // steps in flight for a warp
constexpr float kRescale = 8.0f;        // log2 units a score may pass the reference maximum by
constexpr float kPScale = 32.0f;        // p s' is at most 2^kRescale * kPScale = 2^13

struct FwdParams4 {
  AfaCache4 c;
  const char* q;
  char* o;
  int64_t q_s[3];  // bytes: batch, seq, head
  int64_t o_s[3];
  float* lse;
  float* ws;
  int32_t seq_len, n_heads, group;
  int32_t rows;       // seq_len * group query rows of a key/value head
  int32_t row_tiles;  // blocks of kRows of them
  int32_t page_shift;
  int32_t causal;
  int32_t min_units;  // units a CTA takes at least
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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
// The division of the work, formed alike by every warp of both kernels
// ---------------------------------------------------------------------------

// Tokens of sequence b, 0 (reported) where the lengths are not possible.
__device__ __forceinline__ int tokens_of(const FwdParams4& p, int b) {
  const int kv = p.c.kv_lens[b];
  const int fresh = p.c.new_lens != nullptr ? p.c.new_lens[b] : p.seq_len;
  if (kv < 0 || kv > p.c.max_pages * p.c.page_size || fresh < 0 || fresh > p.seq_len) {
    report(p.c.status, AFA_DEV_BAD_LENGTH);
    return 0;
  }
  return kv;
}
__device__ __forceinline__ int units_of(int tokens) { return tokens <= kUnit ? 1 : (tokens + kUnit - 1) / kUnit; }

struct Division {
  long long total;  // units of the call
  int ctas;         // CTAs that share them
  // First unit of CTA i.
  __device__ __forceinline__ long long first(int i) const { return total * i / ctas; }
};

// Sum of units over this lane's share of the sequences, a contiguous range of
// `per` of them, and from it the division.
__device__ __forceinline__ Division divide(const FwdParams4& p, int per, long long* before_lane) {
  const int lane = static_cast<int>(threadIdx.x & 31u);
  long long mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < p.c.batch) mine += units_of(tokens_of(p, b));
  }
  mine *= static_cast<long long>(p.c.n_kv_heads) * p.row_tiles;
  long long upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, i);
    if (lane >= i) upto += v;
  }
  *before_lane = upto - mine;
  Division d;
  d.total = __shfl_sync(0xffffffffu, upto, 31);
  const long long most = (d.total + p.min_units - 1) / p.min_units;
  d.ctas = static_cast<int>(most < gridDim.x ? most : gridDim.x);
  return d;
}

struct Item {
  int b;      // sequence
  int which;  // key/value head * row_tiles + row block
  int unit;   // unit within the item
  int units;
  int tokens;
};

// The item that unit u belongs to.
__device__ __forceinline__ Item find_item(const FwdParams4& p, int per, long long before_lane, long long u) {
  const int items = p.c.n_kv_heads * p.row_tiles;
  const unsigned owners = __ballot_sync(0xffffffffu, before_lane <= u);
  const int owner = 31 - __clz(owners);
  long long left = u - __shfl_sync(0xffffffffu, before_lane, owner);
  // lanes behind the last sequence own nothing and start where it ends: u is below that
  Item it;
  it.b = owner * per;
  for (;;) {
    it.tokens = tokens_of(p, it.b);
    it.units = units_of(it.tokens);
    const long long here = static_cast<long long>(it.units) * items;
    if (left < here || it.b + 1 >= p.c.batch) break;
    left -= here;
    ++it.b;
  }
  it.which = static_cast<int>(left / it.units);
  it.unit = static_cast<int>(left - static_cast<long long>(it.which) * it.units);
  return it;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
template <int kD, int kNT>
struct FwdLayout4 {
  static constexpr int kGroups = kD / 64;
  static constexpr int kRow = kD / 2 + kD / 16;
  static constexpr int kRows = kNT * 8;
  static constexpr int kTileBytes = 16 * kRow;           // 16 tokens of keys or values
  static constexpr int kStageBytes = 4 * kTileBytes;     // [16 tokens][keys, values]
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kSmem = kWarps * kWarpBytes + kWarps * kRows * 2 * 4;
  static constexpr int kShare = kRows * (kD + 2);        // floats of a CTA's share of an item
  static_assert(kRows * kD * 4 <= kWarpBytes, "a warp's O fits its own stages");
};

template <int kD, bool kBF16, int kNT>
__global__ void __launch_bounds__(kThreads, kNT == 1 ? 3 : 2) cache4_fwd_kernel(const FwdParams4 p) {
  using L = FwdLayout4<kD, kNT>;
  constexpr int kG = L::kGroups;
  constexpr int kRow = L::kRow;
  extern __shared__ __align__(16) char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * L::kWarpBytes;
  float* stats = reinterpret_cast<float*>(smem + kWarps * L::kWarpBytes);  // [warp][row][m, l]

  const int per = (p.c.batch + 31) / 32;
  long long before_lane;
  const Division div = divide(p, per, &before_lane);
  const int cta = blockIdx.x;
  if (cta >= div.ctas) return;
  long long u = div.first(cta);
  const long long u_end = div.first(cta + 1);
  Item it = find_item(p, per, before_lane, u);

  while (u < u_end) {
    const int head = it.which / p.row_tiles, tile = it.which - head * p.row_tiles;
    const int unit_end = u_end - u < it.units - it.unit ? it.unit + static_cast<int>(u_end - u) : it.units;
    const bool whole = it.unit == 0 && unit_end == it.units;
    const int tok_begin = it.unit * kUnit;
    const int tok_end = min(it.tokens, unit_end * kUnit);
    const int fresh = p.c.new_lens != nullptr ? p.c.new_lens[it.b] : p.seq_len;

    // --- loads: a step is two 16-token pieces of keys and of values -------------------------------------
    const char* side = static_cast<const char*>(p.c.cache) + static_cast<int64_t>(head) * 2 * p.c.page_size * kRow;
    const int* table = p.c.page_table + it.b * p.c.table_stride;
    auto load = [&](int tok, int stage) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int at = tok + 16 * c;
        if (at < tok_end) {
          int page = table[at >> p.page_shift];
          uint32_t bytes = 16;
          if (page < 0 || page >= p.c.n_pages) {  // zeros in place of a page that does not exist
            report(p.c.status, AFA_DEV_BAD_PAGE);
            page = 0;
            bytes = 0;
          }
          const char* src =
              side + page * p.c.page_stride + static_cast<int64_t>(at & (p.c.page_size - 1)) * kRow + lane * 16;
          const uint32_t dst = ring + stage * L::kStageBytes + c * 2 * L::kTileBytes + lane * 16;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int x = 0; x < L::kTileBytes; x += 512)
              if (x + 512 <= L::kTileBytes || lane * 16 + x < L::kTileBytes)
                cp_async16(dst + kv * L::kTileBytes + x, src + static_cast<int64_t>(kv) * p.c.page_size * kRow + x,
                           bytes);
        }
      }
      cp_async_commit();
    };
    int tok = tok_begin + warp * kStep;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(tok + s * kUnit, s);

    // --- queries: rows on the N side, their channels in the order the codes come ------------------------
    uint32_t qf[kNT][kG][8];
    float a_of[kNT][2], qs[kNT][kG][2];
    int limit[kNT][2];
    int limit_min = it.tokens;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int r = tile * L::kRows + nt * 8 + g;
      const int i = r / p.group, h = head * p.group + (r - i * p.group);
      uint4 raw[kG][2];
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          raw[gr][x] = make_uint4(0, 0, 0, 0);
          if (r < p.rows)
            raw[gr][x] = *reinterpret_cast<const uint4*>(p.q + it.b * p.q_s[0] + i * p.q_s[1] + h * p.q_s[2] +
                                                         gr * 128 + t * 32 + x * 16);
        }
      float big = 0.0f, sum[kG];
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        sum[gr] = 0.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t w[4] = {raw[gr][x].x, raw[gr][x].y, raw[gr][x].z, raw[gr][x].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = unpack2<kBF16>(w[e]);
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
          const uint32_t w[4] = {raw[gr][x].x, raw[gr][x].y, raw[gr][x].z, raw[gr][x].w};
          float v[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = unpack2<kBF16>(w[y]);
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
    float m_ref[kNT][2], l[kNT][2], e_ref[kG], inv_e[kG];
    float acc[kNT][kG][4][4], acc_m[kNT][kG][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m_ref[nt][x] = -INFINITY;
        l[nt][x] = 0.0f;
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          acc_m[nt][gr][x] = 0.0f;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) acc[nt][gr][mt][x] = acc[nt][gr][mt][2 + x] = 0.0f;
        }
      }
#pragma unroll
    for (int gr = 0; gr < kG; ++gr) {
      e_ref[gr] = 0.0f;
      inv_e[gr] = 0.0f;
    }

    auto compute = [&](auto masked_tag, int tok0, uint32_t base) {
      constexpr bool kMasked = decltype(masked_tag)::value;
      float s[2][kNT][4];
      float vs[2][2][kG], vm[2][2][kG];  // s' and m' of tokens g, g + 8 of each 16
      float vs_max[kG];
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) vs_max[gr] = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t kb = base + c * 2 * L::kTileBytes;
        float part[kNT][4], mins[kNT][4];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) part[nt][x] = mins[nt][x] = 0.0f;
        uint32_t par[2][2][kG];  // keys, values; tokens g, g + 8
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t a = kb + kv * L::kTileBytes + (g + 8 * y) * kRow + kD / 2;
            if constexpr (kG == 2) {
              const uint2 w = lds64(a);
              par[kv][y][0] = w.x;
              par[kv][y][1] = w.y;
            } else {
              par[kv][y][0] = lds32(a);
            }
          }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          uint32_t w[2][2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t a = kb + (g + 8 * y) * kRow + gr * 32 + t * 8;
            if constexpr (kG == 2) {
              const uint2 v = lds64(a);
              w[y][0] = v.x;
              w[y][1] = v.y;
            } else {  // rows of 36 bytes: 4-byte loads
              w[y][0] = lds32(a);
              w[y][1] = lds32(a + 4);
            }
          }
          float dot[kNT][4];
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) dot[nt][x] = 0.0f;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t lo = w[0][x] >> (8 * z), hi = w[1][x] >> (8 * z);
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
                mma16816(dot[nt], lo & 0x000f000fu, hi & 0x000f000fu, lo & 0x00f000f0u, hi & 0x00f000f0u,
                         qf[nt][gr][x * 4 + z * 2], qf[nt][gr][x * 4 + z * 2 + 1]);
            }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float2 sm = unpack2<kBF16>(par[0][y][gr]);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                part[nt][2 * y + x] = fmaf(sm.x, dot[nt][2 * y + x], part[nt][2 * y + x]);
                mins[nt][2 * y + x] = fmaf(sm.y, qs[nt][gr][x], mins[nt][2 * y + x]);
              }
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int at = tok0 + 16 * c + g + 8 * y;
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float v = fmaf(a_of[nt][x], part[nt][2 * y + x], mins[nt][2 * y + x]);
              if (kMasked && at >= limit[nt][x]) v = -INFINITY;
              s[c][nt][2 * y + x] = v;
            }
#pragma unroll
          for (int gr = 0; gr < kG; ++gr) {
            float2 sm = unpack2<kBF16>(par[1][y][gr]);
            if (kMasked && at >= it.tokens) sm = make_float2(0.0f, 0.0f);  // not a token: whatever the page held
            vs[c][y][gr] = sm.x;
            vm[c][y][gr] = sm.y;
            vs_max[gr] = fmaxf(vs_max[gr], fabsf(sm.x));
          }
        }
      }

      // New references only where a score passes the old one by 2^kRescale, or a step the old scale.
      bool moved = false;
      float top[kNT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[nt][x] = fmaxf(fmaxf(s[0][nt][x], s[0][nt][2 + x]), fmaxf(s[1][nt][x], s[1][nt][2 + x]));
          moved |= top[nt][x] > m_ref[nt][x] + kRescale;
        }
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) moved |= vs_max[gr] > e_ref[gr];
      if (__any_sync(0xffffffffu, moved)) {
        float by_e[kG];
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const float big = max_over_rows(vs_max[gr]);
          by_e[gr] = 1.0f;
          if (big > e_ref[gr]) {
            // the power of two above, from 2^-90 on, so that its reciprocal is normal too
            const uint32_t ex = min(max(__float_as_uint(big) >> 23, 36u), 252u) + 1u;
            const float now = __uint_as_float(ex << 23);
            by_e[gr] = e_ref[gr] / now;
            e_ref[gr] = now;
            inv_e[gr] = __uint_as_float((254u - ex) << 23) * kPScale;
          }
        }
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float now = fmaxf(m_ref[nt][x], max_over_rows(top[nt][x]));
            const float by = now == -INFINITY ? 1.0f : ex2_approx(m_ref[nt][x] - now);
            m_ref[nt][x] = now;
            l[nt][x] *= by;
#pragma unroll
            for (int gr = 0; gr < kG; ++gr) {
              acc_m[nt][gr][x] *= by;
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) {
                acc[nt][gr][mt][x] *= by * by_e[gr];
                acc[nt][gr][mt][2 + x] *= by * by_e[gr];
              }
            }
          }
      }

#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t vb = base + (c * 2 + 1) * L::kTileBytes;
        uint32_t pf[kNT][kG][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float pr[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float ref = m_ref[nt][x & 1];
            pr[x] = ex2_approx(s[c][nt][x] - (kMasked && ref == -INFINITY ? 0.0f : ref));
            l[nt][x & 1] += pr[x];
          }
#pragma unroll
          for (int gr = 0; gr < kG; ++gr)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float sc = vs[c][y][gr] * inv_e[gr];
              float w[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float pp = pr[2 * y + x];
                w[x] = pp * sc;
                float mm = vm[c][y][gr];
                if (kMasked && tok0 + 16 * c + g + 8 * y >= limit[nt][x]) {  // its s' and m' may be NaN
                  w[x] = 0.0f;
                  mm = 0.0f;
                }
                acc_m[nt][gr][x] = fmaf(pp, mm, acc_m[nt][gr][x]);
              }
              pf[nt][gr][y] = transpose8x8(half2_of(w[0], w[1]));
            }
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          // rows of tokens 2t, 2t + 1, 2t + 8, 2t + 9; channels 8g .. 8g + 7 of the group
          const uint32_t a = vb + 2 * t * kRow + gr * 32 + g * 4;
          const uint32_t w0 = lds32(a), w1 = lds32(a + kRow), w2 = lds32(a + 8 * kRow), w3 = lds32(a + 9 * kRow);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t sel = z ? 0x7632u : 0x5410u;
            const uint32_t lo = __byte_perm(w0, w1, sel), hi = __byte_perm(w2, w3, sel);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t lo8 = lo >> (8 * y), hi8 = hi >> (8 * y);
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
                mma16816(acc[nt][gr][2 * z + y], lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu,
                         hi8 & 0x00f000f0u, pf[nt][gr][0], pf[nt][gr][1]);
            }
          }
        }
      }
    };

    int stage = 0;
    for (; tok < tok_end; tok += kUnit) {
      cp_async_wait<kStages - 2>();
      __syncwarp();  // every lane's part of the step has landed, and the stage loaded next has been read
      const int next = stage == 0 ? kStages - 1 : stage - 1;
      load(tok + (kStages - 1) * kUnit, next);
      const uint32_t base = ring + stage * L::kStageBytes;
      if (tok + kStep <= limit_min)
        compute(std::false_type{}, tok, base);
      else
        compute(std::true_type{}, tok, base);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    __syncwarp();

    // --- the warps' shares -> the CTA's -------------------------------------------------------------------
    float* mine = reinterpret_cast<float*>(smem + warp * L::kWarpBytes);  // [row][channel]
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = nt * 8 + 2 * t + x;
        const float sum = sum_over_rows(l[nt][x]);
        if (g == 0) {
          stats[(warp * L::kRows + row) * 2] = m_ref[nt][x];
          stats[(warp * L::kRows + row) * 2 + 1] = sum;
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const float mn = sum_over_rows(acc_m[nt][gr][x]);
          const float even = e_ref[gr] * (16777216.0f / kPScale), odd = e_ref[gr] * (1048576.0f / kPScale);
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
    float* share = p.ws + (static_cast<int64_t>(cta) * 2 + (it.unit == 0 ? 1 : 0)) * L::kShare;
    for (int i = threadIdx.x; i < L::kRows * (kD / 4); i += kThreads) {
      const int row = i / (kD / 4), c4 = i - row * (kD / 4);
      float m[kWarps], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        m[w] = stats[(w * L::kRows + row) * 2];
        top = fmaxf(top, m[w]);
      }
      float sum = 0.0f;
      float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float by = m[w] == -INFINITY && top == -INFINITY ? 1.0f : ex2_approx(m[w] - top);
        sum = fmaf(by, stats[(w * L::kRows + row) * 2 + 1], sum);
        const float4 v = *reinterpret_cast<const float4*>(smem + w * L::kWarpBytes + (row * kD + c4 * 4) * 4);
        o.x = fmaf(by, v.x, o.x);
        o.y = fmaf(by, v.y, o.y);
        o.z = fmaf(by, v.z, o.z);
        o.w = fmaf(by, v.w, o.w);
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
    __syncthreads();  // the shares have been read: their memory takes the next item's steps

    u += unit_end - it.unit;
    it.unit = 0;
    if (++it.which == p.c.n_kv_heads * p.row_tiles && u < u_end) {
      it.which = 0;
      ++it.b;
      it.tokens = tokens_of(p, it.b);
      it.units = units_of(it.tokens);
    }
  }
}

// Joins the shares of the items that several CTAs worked on: CTA i takes the
// item its range starts within, if the CTA before it holds that item's start;
// one warp a row (blockIdx.y).  The shares are added in the order of the CTAs.
template <int kD, bool kBF16, int kNT>
__global__ void __launch_bounds__(128) cache4_join_kernel(const FwdParams4 p) {
  using L = FwdLayout4<kD, kNT>;
  constexpr int kPer = kD / 32;  // channels of a lane
  const int lane = threadIdx.x & 31;
  const int per = (p.c.batch + 31) / 32;
  long long before_lane;
  const Division div = divide(p, per, &before_lane);
  const int cta = blockIdx.x;
  if (cta == 0 || cta >= div.ctas) return;
  const long long u = div.first(cta);
  const Item it = find_item(p, per, before_lane, u);
  const long long begin = u - it.unit, end = begin + it.units;
  if (it.unit == 0 || div.first(cta - 1) > begin) return;
  const int head = it.which / p.row_tiles, tile = it.which - head * p.row_tiles;
  const int fresh = p.c.new_lens != nullptr ? p.c.new_lens[it.b] : p.seq_len;
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < L::kRows; row += gridDim.y * 4) {
    const int r = tile * L::kRows + row;
    if (r >= p.rows) break;
    auto share = [&](int i) { return p.ws + (static_cast<int64_t>(i) * 2 + (i == cta - 1 ? 1 : 0)) * L::kShare; };
    float top = -INFINITY;
    int last = cta;
    while (last + 1 < div.ctas && div.first(last + 1) < end) ++last;
    for (int i = cta - 1 + lane; i <= last; i += 32) top = fmaxf(top, share(i)[L::kRows * kD + row * 2]);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum = 0.0f, o[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) o[x] = 0.0f;
#pragma unroll 4
    for (int i = cta - 1; i <= last; ++i) {
      const float* sh = share(i);
      const float m = sh[L::kRows * kD + row * 2];
      const float by = m == -INFINITY && top == -INFINITY ? 1.0f : ex2_approx(m - top);
      sum = fmaf(by, sh[L::kRows * kD + row * 2 + 1], sum);
#pragma unroll
      for (int x = 0; x < kPer; x += 2) {
        const float2 v = *reinterpret_cast<const float2*>(sh + row * kD + lane * kPer + x);
        o[x] = fmaf(by, v.x, o[x]);
        o[x + 1] = fmaf(by, v.y, o[x + 1]);
      }
    }
    const int n = r / p.group, h = head * p.group + (r - n * p.group);
    const bool some = n < fresh && !(sum == 0.0f);
    const float inv = some ? 1.0f / sum : 0.0f;
    char* dst = p.o + it.b * p.o_s[0] + n * p.o_s[1] + h * p.o_s[2] + lane * kPer * 2;
#pragma unroll
    for (int x = 0; x < kPer; x += 2)
      *reinterpret_cast<uint32_t*>(dst + x * 2) = some ? pack2<kBF16>(o[x] * inv, o[x + 1] * inv) : 0u;
    if (p.lse != nullptr && lane == 0)
      p.lse[(static_cast<int64_t>(it.b) * p.n_heads + h) * p.seq_len + n] =
          some ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Kernel4 {
  int rows, smem, share_floats;
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
cudaError_t launch4(const FwdParams4& p, unsigned grid, cudaStream_t s) {
  using L = FwdLayout4<kD, kNT>;
  cache4_fwd_kernel<kD, kBF16, kNT><<<grid, kThreads, L::kSmem, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || grid == 1) return e;
  cache4_join_kernel<kD, kBF16, kNT><<<dim3(grid, L::kRows / 4), 128, 0, s>>>(p);
  return cudaGetLastError();
}

#define AFA_KERNEL4(D, BF, NT)                                                                                 \
  {                                                                                                            \
    FwdLayout4<D, NT>::kRows, FwdLayout4<D, NT>::kSmem, FwdLayout4<D, NT>::kShare,                             \
        &prepare4<D, BF, NT>, &launch4<D, BF, NT>                                                              \
  }
// [head_dim 64, 128][fp16, bf16][8, 16 rows]
const Kernel4 kKernels4[2][2][2] = {
    {{AFA_KERNEL4(64, false, 1), AFA_KERNEL4(64, false, 2)}, {AFA_KERNEL4(64, true, 1), AFA_KERNEL4(64, true, 2)}},
    {{AFA_KERNEL4(128, false, 1), AFA_KERNEL4(128, false, 2)}, {AFA_KERNEL4(128, true, 1), AFA_KERNEL4(128, true, 2)}}};

std::mutex g_mu4;
int g_ctas_per_sm[kOpsMaxDevices][2][2][2] = {};

// Kernel, grid and row blocks of a call.
int plan4(const AfaCache4* c, int32_t seq_len, int32_t n_heads, const Kernel4** kernel, int32_t* grid,
          int32_t* row_tiles) {
  int rc = ops_check_cache(c);
  if (rc != AFA_OK) return rc;
  if (seq_len <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads != 0) return AFA_ERR_INVALID_ARGUMENT;
  const int64_t rows = int64_t{seq_len} * (n_heads / c->n_kv_heads);
  if (rows > INT32_MAX - 64) return AFA_ERR_TOO_LARGE;
  const int di = c->head_dim == 128, ti = c->dtype == AFA_DTYPE_BF16, ni = rows > 8;
  const Kernel4& k = kKernels4[di][ti][ni];
  const int64_t tiles = (rows + k.rows - 1) / k.rows;
  // items and units are counted in 32 and 64 bits, with a factor of the grid's size to spare
  const int64_t items = tiles * c->n_kv_heads;
  const int64_t units = (int64_t{c->max_pages} * c->page_size + kUnit - 1) / kUnit;
  if (items > INT32_MAX || items * c->batch > (int64_t{1} << 48) / units) return AFA_ERR_TOO_LARGE;
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
  // no more CTAs than units at the sequences' largest possible lengths
  const int64_t most = units * items * c->batch;
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
  const int rc = plan4(cache, seq_len, n_heads, &k, &grid, &tiles);
  if (rc != AFA_OK) return -static_cast<int64_t>(rc);
  return int64_t{2} * grid * k->share_floats * static_cast<int64_t>(sizeof(float));
}

int afa_cache4_fwd_sm100(const AfaCache4* cache, const AfaCache4FwdArgs* a, void* stream) {
  int rc = ops_check_cache(cache);
  if (rc != AFA_OK) return rc;
  if (a == nullptr || a->q == nullptr || a->o == nullptr || a->workspace == nullptr ||
      (a->causal != 0 && a->causal != 1) || a->seq_len <= 0 || a->n_heads <= 0)
    return AFA_ERR_INVALID_ARGUMENT;
  if (!ops_aligned16(a->q) || !ops_aligned16(a->o) || !ops_aligned16(a->workspace) ||
      (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0u ||
      !ops_strides_ok(a->q_strides, cache->batch, a->seq_len, a->n_heads, false) ||
      !ops_strides_ok(a->o_strides, cache->batch, a->seq_len, a->n_heads, true))
    return AFA_ERR_MISALIGNED;
  const Kernel4* k = nullptr;
  int32_t grid = 0, tiles = 0;
  rc = plan4(cache, a->seq_len, a->n_heads, &k, &grid, &tiles);
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
  p.causal = a->causal;
  p.min_units = 1;
  const double scale = a->scale > 0.f ? a->scale : 1.0 / (cache->head_dim == 64 ? 8.0 : 11.313708498984761);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  if (k->launch(p, static_cast<unsigned>(grid), static_cast<cudaStream_t>(stream)) != cudaSuccess) {
    cudaGetLastError();
    return AFA_ERR_LAUNCH;
  }
  return AFA_OK;
}

}  // extern "C"
