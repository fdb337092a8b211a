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
// Bound: HBM.  A value costs 2 bytes on one side and 0.5625 on the other.  Four
// neighbouring lanes hold one group, sixteen channels (32 bytes, one access) a lane;
// minimum and maximum travel together as one packed pair through two shuffles.  A CTA
// takes a tile of tokens of one sequence times (head, keys or values), tokens
// fastest, so that the rows it writes are neighbours in a page.
// Measured: reading back 131072 tokens [8, 128] bf16 117 us among other work = 5.9
// TB/s (90 % of the measured copy bandwidth), 109 us in calls in a row.  Eight prompts of 4096 down to 2304 tokens
// [8, 128] fp16, written and read back: 66 us = 4.5 TB/s (69 %); the reader is
// at the bandwidth there too, the writer at its arithmetic (about 17
// instructions a value, 69 % of the issue slots), so one row a lane (83 us) and
// four (76 us) are slower than two.
#include "ops_common.cuh"

namespace {

using namespace afa100;

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // rows a lane has in flight

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

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}

// Two quotients of each of eight values, 2^-20 below and above the exact one (the
// difference, the reciprocal and the product are off by less than 2^-21 together),
// each rounded to an integer by the addition of 1.5 * 2^23 in the same operation.
// Where both round alike, so does the exact one; a tie or nearly one (common among
// values of 8 bits) shows as two neighbours, and the exact difference decides.
template <bool kBF16>
__device__ __forceinline__ uint32_t codes8(const uint32_t (&xs)[4], float low, float s, float below, float above) {
  const float2 big = make_float2(12582912.0f, 12582912.0f);
  uint32_t a[8], differ = 0, word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = add2(unpack2<kBF16>(xs[i]), make_float2(-low, -low));
    const float2 r = fma2(v, make_float2(below, below), big), t = fma2(v, make_float2(above, above), big);
    a[2 * i] = __float_as_uint(r.x);
    a[2 * i + 1] = __float_as_uint(r.y);
    differ |= (__float_as_uint(r.x) ^ __float_as_uint(t.x)) | (__float_as_uint(r.y) ^ __float_as_uint(t.y));
  }
  // the integers' bits are 0x4b400000 + code: their sum over 16^i carries a constant with it
#pragma unroll
  for (int i = 7; i >= 0; --i) word = word * 16u + a[i];
  word -= 0x4b400000u * 0x11111111u;
  if (differ != 0) {
    const float half = 0.5f * s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v2 = unpack2<kBF16>(xs[i / 2]);
      const float v = i & 1 ? v2.y : v2.x;
      if (__float_as_uint(fmaf(v - low, above, 12582912.0f)) != a[i]) {
        const uint32_t c = a[i] & 15u;
        const float border = fmaf(static_cast<float>(c), s, half), d = sub_odd(v, low);
        if (d > border || (d == border && (c & 1u))) word += 1u << (4 * i);
      }
    }
  }
  return word;
}

// Sixteen channels of one lane to sixteen codes; the lane's group is the four
// lanes that differ in the lowest two bits.  *params: s and m.
template <bool kBF16>
__device__ __forceinline__ uint2 quantise16(const uint32_t (&x)[2][4], uint32_t* params) {
  uint32_t lo = x[0][0], hi = x[0][0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min2_nan<kBF16>(lo, x[i / 4][i % 4]);
    hi = max2_nan<kBF16>(hi, x[i / 4][i % 4]);
  }
  hi ^= 0x80008000u;
  // {minimum, -maximum}, so that one minimum a shuffle carries both
  uint32_t mm = min2_nan<kBF16>(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
  for (int i = 1; i < 4; i <<= 1) mm = min2_nan<kBF16>(mm, __shfl_xor_sync(0xffffffffu, mm, i));
  const float2 ends = unpack2<kBF16>(mm);
  const float low = ends.x, high = -ends.y;
  if (!(high - low < __int_as_float(0x7f800000))) {  // an infinity, a NaN, or a range beyond fp32
    *params = 0x7fff7fffu;
    return make_uint2(0, 0);
  }
  const uint32_t s16 = step16<kBF16>(high, low);
  *params = s16 | (mm << 16);
  const float s = unpack2<kBF16>(s16).x;
  if (s == 0.0f) return make_uint2(0, 0);
  // Steps so small that 16 bits round them by more than 1/30 (fp16), or that their reciprocal is not an fp32
  // number: the codes one by one.
  if (s < (kBF16 ? 1e-30f : 1.9073486328125e-06f)) {
    uint2 word = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 v = unpack2<kBF16>(x[i / 8][i / 2 % 4]);
      const uint32_t c = code_exact(i & 1 ? v.y : v.x, low, s) << (4 * (i & 7));
      if (i < 8)
        word.x |= c;
      else
        word.y |= c;
    }
    return word;
  }
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float below = inv * 0.99999904632568359375f, above = inv * 1.00000095367431640625f;
  return make_uint2(codes8<kBF16>(x[0], low, s, below, above), codes8<kBF16>(x[1], low, s, below, above));
}

template <int kD>
struct Tile {
  static constexpr int kLanes = kD / 16;           // lanes of a row, 16 channels each
  static constexpr int kRows = kThreads / kLanes;  // rows of a CTA at a time
  static constexpr int kTile = kRows * kUnroll;    // rows of a CTA
  static constexpr int kRow = kD / 2 + kD / 16;    // bytes of a cache row
};

// A CTA's tile: kTile rows, 2^tile_shift tokens of some sides (head * 2 + keys or
// values) of one sequence.  Where a sequence's rows fill it (kLong) there is one
// side, and a thread's rows lie a fixed distance apart.
template <int kD, bool kLong>
struct Place {
  int b, token0, side0;
  __device__ __forceinline__ explicit Place(const Cache4Params& p) {
    const int per = p.n_tiles * p.n_sides;
    b = blockIdx.x / per;
    const int rest = blockIdx.x - b * per, tile = rest / p.n_sides;
    token0 = tile << p.tile_shift;
    side0 = (rest - tile * p.n_sides) * (Tile<kD>::kTile >> p.tile_shift);
  }
  // Token and side of the thread's u-th row.
  __device__ __forceinline__ int token(const Cache4Params& p, int u) const {
    const int r = u * Tile<kD>::kRows + threadIdx.x / Tile<kD>::kLanes;
    return token0 + (kLong ? r : r & ((1 << p.tile_shift) - 1));
  }
  __device__ __forceinline__ int side(const Cache4Params& p, int u) const {
    const int r = u * Tile<kD>::kRows + threadIdx.x / Tile<kD>::kLanes;
    return kLong ? side0 : side0 + (r >> p.tile_shift);
  }
};

// The lane's 32 bytes of a row of k or v.
template <int kD>
__device__ __forceinline__ char* outer_row(const Cache4Params& p, int b, int token, int side) {
  const int w = side & 1;
  return p.x[w] + b * p.x_s[w][0] + (side >> 1) * p.x_s[w][2] + token * p.x_s[w][1] +
         threadIdx.x % Tile<kD>::kLanes * 32;
}

// The cache's row, or null (reported) where its page does not exist.
template <int kD>
__device__ __forceinline__ char* cache_row(const Cache4Params& p, int b, int pos, int side) {
  const int page = p.c.page_table[b * p.c.table_stride + (pos >> p.page_shift)];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.c.n_pages)) {
    report(p.c.status, AFA_DEV_BAD_PAGE);
    return nullptr;
  }
  const int64_t of_side = static_cast<int64_t>(side) * p.c.page_size * Tile<kD>::kRow;
  return static_cast<char*>(p.c.cache) + of_side + page * p.c.page_stride + (pos & (p.c.page_size - 1)) * Tile<kD>::kRow;
}

template <int kD, bool kBF16, bool kLong>
__global__ void __launch_bounds__(kThreads) cache4_write_kernel(const Cache4Params p) {
  using T = Tile<kD>;
  const Place<kD, kLong> at(p);
  after_previous();
  const NewRows fresh = new_rows(p.c, at.b, p.seq_len);
  if (at.token0 >= fresh.count) return;
  const int lane = threadIdx.x % T::kLanes;
  uint32_t x[kUnroll][2][4];
  char* row[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int token = at.token(p, u), side = at.side(p, u);
    row[u] = nullptr;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[u][i / 4][i % 4] = 0;
    if (token < fresh.count && (kLong || side < 2 * p.c.n_kv_heads)) {
      load32<true>(x[u], outer_row<kD>(p, at.b, token, side));
      row[u] = cache_row<kD>(p, at.b, fresh.first + token, side);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t params;
    const uint2 word = quantise16<kBF16>(x[u], &params);
    if (row[u] != nullptr) {
      if constexpr (kD == 128) {
        *reinterpret_cast<uint2*>(row[u] + lane * 8) = word;
      } else {  // rows of 36 bytes
        *reinterpret_cast<uint32_t*>(row[u] + lane * 8) = word.x;
        *reinterpret_cast<uint32_t*>(row[u] + lane * 8 + 4) = word.y;
      }
      if (lane % 4 == 0) *reinterpret_cast<uint32_t*>(row[u] + kD / 2 + lane) = params;
    }
  }
}

// s * c + m for the eight codes of a word, rounded once (a 16-bit fused multiply-add; codes, s and m are
// exact operands).  A 16-bit value with the bits of 1024 (bf16: 128) and the code in its last places is
// 1024 + c; the subtraction is exact.
template <bool kBF16>
__device__ __forceinline__ void dequantise8(uint32_t (&out)[4], uint32_t word, uint32_t s2, uint32_t m2) {
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
  out[0] = __byte_perm(v[0], v[1], 0x5410);
  out[1] = __byte_perm(v[2], v[3], 0x5410);
  out[2] = __byte_perm(v[0], v[1], 0x7632);
  out[3] = __byte_perm(v[2], v[3], 0x7632);
}

template <int kD, bool kBF16, bool kLong>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const Cache4Params p) {
  using T = Tile<kD>;
  const Place<kD, kLong> at(p);
  after_previous();
  const NewRows fresh = new_rows(p.c, at.b, p.seq_len);
  const int lane = threadIdx.x % T::kLanes;
  uint2 word[kUnroll];
  uint32_t params[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int token = at.token(p, u), side = at.side(p, u);
    word[u] = make_uint2(0, 0);
    params[u] = 0;
    if (token < fresh.count && (kLong || side < 2 * p.c.n_kv_heads)) {
      const char* row = cache_row<kD>(p, at.b, fresh.first + token, side);
      if (row != nullptr) {
        if constexpr (kD == 128) {
          word[u] = *reinterpret_cast<const uint2*>(row + lane * 8);
        } else {  // rows of 36 bytes
          word[u].x = *reinterpret_cast<const uint32_t*>(row + lane * 8);
          word[u].y = *reinterpret_cast<const uint32_t*>(row + lane * 8 + 4);
        }
        params[u] = *reinterpret_cast<const uint32_t*>(row + kD / 2 + lane / 4 * 4);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int token = at.token(p, u), side = at.side(p, u);
    if (token < p.seq_len && (kLong || side < 2 * p.c.n_kv_heads)) {
      const uint32_t s2 = __byte_perm(params[u], 0, 0x1010), m2 = __byte_perm(params[u], 0, 0x3232);
      uint32_t v[2][4];
      dequantise8<kBF16>(v[0], word[u].x, s2, m2);
      dequantise8<kBF16>(v[1], word[u].y, s2, m2);
      store32(outer_row<kD>(p, at.b, token, side), v);
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
  const bool one_side = (1 << p.tile_shift) == tile;
#define AFA_MOVE_AS(D, BF, LONG) \
  ops_launch(kWrite ? cache4_write_kernel<D, BF, LONG> : cache4_read_kernel<D, BF, LONG>, dim3(g), kThreads, 0, s, p)
#define AFA_MOVE(D, BF)          \
  if (one_side) {                \
    AFA_MOVE_AS(D, BF, true);    \
  } else {                       \
    AFA_MOVE_AS(D, BF, false);   \
  }
  if (c->head_dim == 64) {
    if (bf) { AFA_MOVE(64, true) } else { AFA_MOVE(64, false) }
  } else {
    if (bf) { AFA_MOVE(128, true) } else { AFA_MOVE(128, false) }
  }
#undef AFA_MOVE
#undef AFA_MOVE_AS
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
