// afa_cache4_fwd_common.cuh -- what the kernels of attention over the 4-bit cache
// share: their parameters and the division of the work among the CTAs.
#pragma once

#include "ops_common.cuh"
#include "sm100_ptx.cuh"

namespace afa100 {

constexpr int kUnit = 128;        // tokens of a unit of work
constexpr int kItemUnits = 4;     // units an item is charged beside its tokens'
constexpr int kWholeTokens = 512; // items that cannot be longer are not split, if there is a CTA for each
// What a row's weights are measured by, so that p s' fits fp16: its reference is the largest score + log2(size) of the
// tokens it sees, and p = 2^(score + kHeadroom - reference).  A token's size is its larger step; 2^-20 of its minima
// and 2^-60 at least, so that p itself and p m' stay far from fp32's largest where there are no steps.
constexpr float kRescale = 8.0f;   // log2 units the product may pass the reference by
constexpr float kHeadroom = 7.0f;  // log2 of the product at the reference
constexpr float kLeastSize = 8.673617379884035e-19f;
constexpr float kMinimaSize = 9.5367431640625e-07f;

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
  uint32_t page_stride;
  int32_t causal;
  int32_t unit_tokens;  // kUnit, or kWholeTokens where items are not split
  int32_t item_units;   // kItemUnits, or 0
  float scale_log2;
  uint64_t timeout_ns;  // of a wait (the kernel for many rows; the other one waits for nothing)
  uint32_t test_flags;  // AFA_TEST_PRODUCER_IDLE
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A token's size from one group's step and minimum (above); what is not finite has none.
__device__ __forceinline__ float size_of(float size, float step, float minimum) {
  const float a = fabsf(step), b = fabsf(minimum) * kMinimaSize;
  return fmax3(size, a < INFINITY ? a : 0.0f, b < INFINITY ? b : 0.0f);
}
// The power of two above, to 2^126; its logarithm.
__device__ __forceinline__ float power_above(float x) { return __uint_as_float((min(__float_as_uint(x) >> 23, 252u) + 1u) << 23); }
__device__ __forceinline__ float log2_of_power(float x) { return static_cast<float>(static_cast<int>(__float_as_uint(x) >> 23) - 127); }
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// p + n * stride bytes
__device__ __forceinline__ const char* far(const char* p, uint32_t n, uint32_t stride) {
  uint64_t r;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(n), "r"(stride), "l"(reinterpret_cast<uint64_t>(p)));
  return reinterpret_cast<const char*>(r);
}

// ---------------------------------------------------------------------------
// The division of the work, formed alike by every warp of both kernels
// ---------------------------------------------------------------------------

// Tokens of sequence b; 0 where no row needs them, or (reported) where the lengths are not possible.
__device__ __forceinline__ int tokens_of(const FwdParams4& p, int b) {
  const int kv = p.c.kv_lens[b];
  const int fresh = p.c.new_lens != nullptr ? p.c.new_lens[b] : p.seq_len;
  if (kv < 0 || kv > p.c.max_pages * p.c.page_size || fresh < 0 || fresh > p.seq_len) {
    report(p.c.status, AFA_DEV_BAD_LENGTH);
    return 0;
  }
  return fresh == 0 ? 0 : kv;
}
// Units of an item: item_units that stand for what starting and ending an item
// costs, then those of its tokens (one at least).
__device__ __forceinline__ int units_of(const FwdParams4& p, int tokens) {
  return p.item_units + (tokens <= p.unit_tokens ? 1 : (tokens + kUnit - 1) / kUnit);
}

struct Division {
  int ctas;  // CTAs that share the units: the first `more` of them take each + 1, the others `each`
  int each, more;
  // First unit of CTA i.
  __device__ __forceinline__ int first(int i) const { return i * each + min(i, more); }
  // The CTA that holds unit u.
  __device__ __forceinline__ int holder(int u) const {
    const int longer = more * (each + 1);
    return u < longer ? u / (each + 1) : more + (u - longer) / each;
  }
};

// Sum of units over this lane's share of the sequences, a contiguous range of
// `per` of them, and from it the division.  The host has made sure that the
// units of the call fit 31 bits.
__device__ __forceinline__ Division divide(const FwdParams4& p, int per, int grid, int* before_lane) {
  const int lane = static_cast<int>(threadIdx.x & 31u);
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < p.c.batch) mine += units_of(p, tokens_of(p, b));
  }
  mine *= p.c.n_kv_heads * p.row_tiles;
  int upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, i);
    if (lane >= i) upto += v;
  }
  *before_lane = upto - mine;
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  Division d;
  d.ctas = min(total, grid);
  d.each = total / d.ctas;
  d.more = total - d.each * d.ctas;
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
__device__ __forceinline__ Item find_item(const FwdParams4& p, int per, int before_lane, int u) {
  const int items = p.c.n_kv_heads * p.row_tiles;
  const unsigned owners = __ballot_sync(0xffffffffu, before_lane <= u);
  const int owner = 31 - __clz(owners);
  int left = u - __shfl_sync(0xffffffffu, before_lane, owner);
  // lanes behind the last sequence own nothing and start where it ends: u is below that
  Item it;
  it.b = owner * per;
  for (;;) {
    it.tokens = tokens_of(p, it.b);
    it.units = units_of(p, it.tokens);
    const int here = it.units * items;
    if (left < here || it.b + 1 >= p.c.batch) break;
    left -= here;
    ++it.b;
  }
  it.which = left / it.units;
  it.unit = left - it.which * it.units;
  return it;
}

// A CTA's walk through its units, piece by piece (a piece: its part of one item).
// `offset`: the first token of a piece that the caller works on, from its begin.
struct Walk {
  Item it;
  int left;      // units of the CTA from this piece on
  int unit_end;  // end of the piece within the item
  int tok, tok_end;
  __device__ __forceinline__ void open(const FwdParams4& p, int offset) {
    unit_end = it.unit + left < it.units ? it.unit + left : it.units;
    tok = max(it.unit - p.item_units, 0) * p.unit_tokens + offset;
    tok_end = min(it.tokens, max(unit_end - p.item_units, 0) * p.unit_tokens);
  }
  // To the next piece; false at the end of the CTA's units.
  __device__ __forceinline__ bool next(const FwdParams4& p, int offset) {
    left -= unit_end - it.unit;
    if (left <= 0) return false;
    it.unit = 0;
    if (++it.which == p.c.n_kv_heads * p.row_tiles) {
      if (it.b + 1 >= p.c.batch) return false;  // only if the lengths changed under the kernel
      it.which = 0;
      ++it.b;
      it.tokens = tokens_of(p, it.b);
      it.units = units_of(p, it.tokens);
    }
    open(p, offset);
    return true;
  }
};

}  // namespace afa100
