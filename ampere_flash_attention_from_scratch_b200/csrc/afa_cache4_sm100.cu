// afa_cache4_sm100.cu -- quantising keys and values as they are written to the
// paged 4-bit cache, and reading them back (afa_cache4_write_sm100,
// afa_cache4_read_sm100, include/afa_sm100_ops.h).
//
// Mathematics, per group of 64 channels: m = min(x), s = round16((max - min) / 15),
// code = round((x - m) / s), halves to even, at most 15; a code stands for
// s * code + m.  m is one of the inputs and so exact in 16 bits.  Both roundings
// are those of the exact quotients (below), so a row's bytes do not depend on
// how the arithmetic is arranged.
//
// Bound: HBM.  A value costs 2 bytes on one side and 0.5625 on the other.  Eight
// neighbouring lanes hold one group, eight channels (16 bytes) a lane; minimum
// and maximum travel together as one packed pair through three shuffles.  A CTA
// takes a tile of tokens of one sequence times (head, keys or values), tokens
// fastest, so that the rows it writes are neighbours in a page.
#include "ops_common.cuh"

namespace {

using namespace afa100;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows a lane has in flight

struct Cache4Params {
  AfaCache4 c;
  char* x[2];  // k, v: read by the writer, written by the reader
  int64_t x_s[2][3];  // bytes: batch, seq, head
  int32_t seq_len;
  int32_t page_shift;
  int32_t tile_shift;  // tokens of a CTA's tile, a power of two
  int32_t n_tiles;     // tiles along seq_len
  int32_t n_sides;     // CTAs along 2 * n_kv_heads
};

// --- exact roundings ------------------------------------------------------------------------------------

// a - b rounded to odd: exact, or the one of the two neighbouring fp32 values
// with an odd significand.  Compared with any value of at most 23 bits it
// orders as the exact difference does.
__device__ __forceinline__ float sub_odd(float a, float b) {
  const float lo = __fsub_rz(a, b);
  return lo == __fsub_ru(a, b) && lo == __fsub_rd(a, b) ? lo : __uint_as_float(__float_as_uint(lo) | 1u);
}

template <bool kBF16>
__device__ __forceinline__ uint32_t round16(float x) {
  return pack2<kBF16>(x, 0.f) & 0xffffu;
}

// (max - min) / 15 rounded once to 16 bits.  The quick quotient is within 2^-22
// of the exact one; only where that much decides the rounding is the quotient
// formed rounded to odd, whose 24 bits then round to 16 as the exact one would
// (a value halfway between two 16-bit ones has at most 12 bits).
template <bool kBF16>
__device__ __forceinline__ uint32_t step16(float high, float low) {
  const float d = high - low;
  const float q = d * (1.0f / 15.0f);
  const uint32_t both = pack2<kBF16>(q * 0.99999904632568359375f, q * 1.00000095367431640625f);
  if ((both & 0xffffu) == (both >> 16) && q > 1e-30f) return both & 0xffffu;
  const float e = sub_odd(high, low);
  float z = __fdiv_rz(e, 15.0f);
  if (__fmaf_rn(-15.0f, z, e) != 0.0f) z = __uint_as_float(__float_as_uint(z) | 1u);
  return round16<kBF16>(z);
}

// round((x - m) / s), halves to even, at most 15, from exact comparisons with
// the borders (c + 1/2) s, which have at most 16 bits.
__device__ __noinline__ uint32_t code_exact(float x, float m, float s) {
  const float d = sub_odd(x, m);
  uint32_t code = 0;
  for (int c = 0; c < 15; ++c) {
    const float border = (static_cast<float>(c) + 0.5f) * s;
    code += (d > border || (d == border && (c & 1))) ? 1u : 0u;
  }
  return code;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kBF16)
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool kBF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kBF16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight channels of one lane to eight codes; the lane's group is the eight lanes
// that differ in the lowest three bits.  *params: s and m.
template <bool kBF16>
__device__ __forceinline__ uint32_t quantise8(const uint4 x, uint32_t* params) {
  uint32_t lo = min2_nan<kBF16>(min2_nan<kBF16>(x.x, x.y), min2_nan<kBF16>(x.z, x.w));
  uint32_t hi = max2_nan<kBF16>(max2_nan<kBF16>(x.x, x.y), max2_nan<kBF16>(x.z, x.w));
  // {minimum, -maximum}, so that one minimum a shuffle carries both
  uint32_t mm = min2_nan<kBF16>(__byte_perm(lo, hi ^ 0x80008000u, 0x5410), __byte_perm(lo, hi ^ 0x80008000u, 0x7632));
#pragma unroll
  for (int i = 1; i < 8; i <<= 1) mm = min2_nan<kBF16>(mm, __shfl_xor_sync(0xffffffffu, mm, i));
  const float2 ends = unpack2<kBF16>(mm);
  const float low = ends.x, high = -ends.y;
  if (!(high - low < __int_as_float(0x7f800000))) {  // an infinity, a NaN, or a range beyond fp32
    *params = 0x7fff7fffu;
    return 0u;
  }
  const uint32_t s16 = step16<kBF16>(high, low);
  *params = s16 | (mm << 16);
  const float s = unpack2<kBF16>(s16).x;
  if (s == 0.0f) return 0u;
  // The quick quotient is within 2^-18 of the exact one (15 * 2^-22): unless it is
  // that close to halfway, it rounds the same.
  const float inv = 1.0f / s;
  bool close = s < 1e-30f;
  uint32_t word = 0;
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<kBF16>(xs[i]);
    const float q0 = fminf((v.x - low) * inv, 15.0f), q1 = fminf((v.y - low) * inv, 15.0f);
    const float r0 = rintf(q0), r1 = rintf(q1);
    close |= fmaxf(fabsf(q0 - r0), fabsf(q1 - r1)) > 0.5f - 7.62939453125e-06f;
    word |= static_cast<uint32_t>(__float2int_rn(fmaf(r1, 16.0f, r0))) << (8 * i);
  }
  if (close) {
    word = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = i < 4 ? (i < 2 ? x.x : x.y) : (i < 6 ? x.z : x.w);
      const float2 v = unpack2<kBF16>(w);
      word |= code_exact(i & 1 ? v.y : v.x, low, s) << (4 * i);
    }
  }
  return word;
}

// Where the CTA's row `r` is: its token, its side (head * 2 + keys or values) and
// whether it exists.
struct RowAt {
  int token;
  int side;
};

template <int kD>
struct Tile {
  static constexpr int kLanes = kD / 8;                  // lanes of a row
  static constexpr int kRows = kThreads / kLanes;        // rows of a CTA at a time
  static constexpr int kTile = kRows * kUnroll;          // rows of a CTA
  static constexpr int kRow = kD / 2 + kD / 16;          // bytes of a cache row
};

// Byte offset of a cache row, or -1 (reported) where its page does not exist.
template <int kD>
__device__ __forceinline__ int64_t cache_row(const Cache4Params& p, int b, int pos, int side) {
  const int page = p.c.page_table[b * p.c.table_stride + (pos >> p.page_shift)];
  if (page < 0 || page >= p.c.n_pages) {
    report(p.c.status, AFA_DEV_BAD_PAGE);
    return -1;
  }
  const int place = pos & (p.c.page_size - 1);
  return page * p.c.page_stride + (static_cast<int64_t>(side) * p.c.page_size + place) * Tile<kD>::kRow;
}

template <int kD, bool kBF16>
__global__ void __launch_bounds__(kThreads) cache4_write_kernel(const Cache4Params p) {
  using T = Tile<kD>;
  const int b = blockIdx.x / (p.n_tiles * p.n_sides);
  const int rest = blockIdx.x - b * (p.n_tiles * p.n_sides);
  const int token0 = (rest / p.n_sides) << p.tile_shift;
  const int side0 = (rest % p.n_sides) * (T::kTile >> p.tile_shift);
  const NewRows fresh = new_rows(p.c, b, p.seq_len);
  const int lane = threadIdx.x % T::kLanes;
  uint4 x[kUnroll];
  int64_t at[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int r = u * T::kRows + threadIdx.x / T::kLanes;
    const int token = token0 + (r & ((1 << p.tile_shift) - 1)), side = side0 + (r >> p.tile_shift);
    at[u] = -1;
    x[u] = make_uint4(0, 0, 0, 0);
    if (token < fresh.count && side < 2 * p.c.n_kv_heads) {
      at[u] = cache_row<kD>(p, b, fresh.first + token, side);
      const int w = side & 1;
      x[u] = ldg_stream(p.x[w] + b * p.x_s[w][0] + token * p.x_s[w][1] + (side >> 1) * p.x_s[w][2] + lane * 16);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t params;
    const uint32_t word = quantise8<kBF16>(x[u], &params);
    if (at[u] >= 0) {
      char* row = static_cast<char*>(p.c.cache) + at[u];
      *reinterpret_cast<uint32_t*>(row + lane * 4) = word;
      if (lane % 8 == 0) *reinterpret_cast<uint32_t*>(row + kD / 2 + lane / 8 * 4) = params;
    }
  }
}

// s * c + m for the eight codes of a word, rounded once (a 16-bit fused multiply-add; codes, s and m are
// exact operands).  A 16-bit value with the bits of 1024 (bf16: 128) and the code in its last places is
// 1024 + c; the subtraction is exact.
template <bool kBF16>
__device__ __forceinline__ uint4 dequantise8(uint32_t word, uint32_t params) {
  const uint32_t s2 = __byte_perm(params, 0, 0x1010), m2 = __byte_perm(params, 0, 0x3232);
  uint32_t v[4];  // channels {0, 4}, {1, 5}, {2, 6}, {3, 7}
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = (word >> (4 * i)) & 0x000f000fu;
    if constexpr (kBF16) {
      const uint32_t biased = c | 0x43004300u, neg = 0xc300c300u, one = 0x3f803f80u;
      uint32_t f;
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(f) : "r"(biased), "r"(one), "r"(neg));
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[i]) : "r"(f), "r"(s2), "r"(m2));
    } else {
      const uint32_t biased = c | 0x64006400u, neg = 0xe400e400u;
      uint32_t f;
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(f) : "r"(biased), "r"(neg));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v[i]) : "r"(f), "r"(s2), "r"(m2));
    }
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                    __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
}

template <int kD, bool kBF16>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const Cache4Params p) {
  using T = Tile<kD>;
  const int b = blockIdx.x / (p.n_tiles * p.n_sides);
  const int rest = blockIdx.x - b * (p.n_tiles * p.n_sides);
  const int token0 = (rest / p.n_sides) << p.tile_shift;
  const int side0 = (rest % p.n_sides) * (T::kTile >> p.tile_shift);
  const NewRows fresh = new_rows(p.c, b, p.seq_len);
  const int lane = threadIdx.x % T::kLanes;
  uint32_t word[kUnroll], params[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int r = u * T::kRows + threadIdx.x / T::kLanes;
    const int token = token0 + (r & ((1 << p.tile_shift) - 1)), side = side0 + (r >> p.tile_shift);
    word[u] = params[u] = 0;
    if (token < fresh.count && side < 2 * p.c.n_kv_heads) {
      const int64_t at = cache_row<kD>(p, b, fresh.first + token, side);
      if (at >= 0) {
        const char* row = static_cast<const char*>(p.c.cache) + at;
        word[u] = *reinterpret_cast<const uint32_t*>(row + lane * 4);
        params[u] = *reinterpret_cast<const uint32_t*>(row + kD / 2 + lane / 8 * 4);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int r = u * T::kRows + threadIdx.x / T::kLanes;
    const int token = token0 + (r & ((1 << p.tile_shift) - 1)), side = side0 + (r >> p.tile_shift);
    if (token < p.seq_len && side < 2 * p.c.n_kv_heads) {
      const int w = side & 1;
      char* dst = p.x[w] + b * p.x_s[w][0] + token * p.x_s[w][1] + (side >> 1) * p.x_s[w][2] + lane * 16;
      *reinterpret_cast<uint4*>(dst) = dequantise8<kBF16>(word[u], params[u]);
    }
  }
}

template <bool kWrite>
int cache4_move(const AfaCache4* c, const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                int32_t seq_len, void* stream) {
  int rc = ops_check_cache(c);
  if (rc != AFA_OK) return rc;
  if (k == nullptr || v == nullptr || k_strides == nullptr || v_strides == nullptr || seq_len <= 0)
    return AFA_ERR_INVALID_ARGUMENT;
  if (!ops_aligned16(k) || !ops_aligned16(v) ||
      !ops_strides_ok(k_strides, c->batch, seq_len, c->n_kv_heads, !kWrite) ||
      !ops_strides_ok(v_strides, c->batch, seq_len, c->n_kv_heads, !kWrite))
    return AFA_ERR_MISALIGNED;
  Cache4Params p{};
  p.c = *c;
  p.x[0] = const_cast<char*>(static_cast<const char*>(k));
  p.x[1] = const_cast<char*>(static_cast<const char*>(v));
  for (int i = 0; i < 3; ++i) {
    p.x_s[0][i] = k_strides[i] * 2;
    p.x_s[1][i] = v_strides[i] * 2;
  }
  p.seq_len = seq_len;
  p.page_shift = ops_log2(c->page_size);
  const int tile = c->head_dim == 64 ? Tile<64>::kTile : Tile<128>::kTile;
  p.tile_shift = ops_log2(seq_len < tile ? seq_len : tile);
  const int64_t n_tiles = (int64_t{seq_len} + (1 << p.tile_shift) - 1) >> p.tile_shift;
  const int64_t sides = tile >> p.tile_shift;
  const int64_t n_sides = (int64_t{2} * c->n_kv_heads + sides - 1) / sides;
  const int64_t grid = c->batch * n_tiles * n_sides;
  if (n_tiles * n_sides > INT32_MAX || grid > INT32_MAX || int64_t{2} * c->n_kv_heads > INT32_MAX / 2)
    return AFA_ERR_TOO_LARGE;
  p.n_tiles = static_cast<int32_t>(n_tiles);
  p.n_sides = static_cast<int32_t>(n_sides);

  int dev = 0, sms = 0;
  rc = ops_device(&dev, &sms);
  if (rc != AFA_OK) return rc;
  const unsigned g = static_cast<unsigned>(grid);
  const auto s = static_cast<cudaStream_t>(stream);
  const bool bf = c->dtype == AFA_DTYPE_BF16;
#define AFA_MOVE(D, BF)                                             \
  if (kWrite)                                                       \
    cache4_write_kernel<D, BF><<<g, kThreads, 0, s>>>(p);           \
  else                                                              \
    cache4_read_kernel<D, BF><<<g, kThreads, 0, s>>>(p)
  if (c->head_dim == 64) {
    if (bf) { AFA_MOVE(64, true); } else { AFA_MOVE(64, false); }
  } else {
    if (bf) { AFA_MOVE(128, true); } else { AFA_MOVE(128, false); }
  }
#undef AFA_MOVE
  return ops_launched();
}

}  // namespace

extern "C" {

int afa_sm100_ops_version(void) { return 100; }

int32_t afa_cache4_row_bytes(int32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? head_dim / 2 + head_dim / 16 : -1;
}

int afa_cache4_write_sm100(const AfaCache4* cache, const void* k, const void* v, const int64_t k_strides[3],
                           const int64_t v_strides[3], int32_t seq_len, void* stream) {
  return cache4_move<true>(cache, k, v, k_strides, v_strides, seq_len, stream);
}

int afa_cache4_read_sm100(const AfaCache4* cache, void* k, void* v, const int64_t k_strides[3],
                          const int64_t v_strides[3], int32_t seq_len, void* stream) {
  return cache4_move<false>(cache, k, v, k_strides, v_strides, seq_len, stream);
}

}  // extern "C"
