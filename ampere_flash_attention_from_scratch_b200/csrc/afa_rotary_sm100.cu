// afa_rotary_sm100.cu -- rotary positions with several axes
// (afa_rotary_sm100, include/afa_sm100_ops.h).
//
// Mathematics.  Pair j of a row is turned by angle = position * frequency:
// (a, b) -> (a cos - b sin, b cos + a sin).  The angle is formed in 64 bits and
// reduced to a fraction of a turn there -- at position 10^6 a 32-bit product is
// off by up to 0.03 rad -- and only that fraction, at most half a turn, goes to
// the 32-bit sine and cosine.  A rotation's transpose is the rotation back, so
// the gradient is the same kernel with the sine negated.
//
// Bound: HBM.  Each 16-bit element is read once and written once, 4 bytes in
// all, against 3 fp32 operations.  The angles are shared by all heads of a
// token, so a CTA forms them once for its tokens (rot_dim / 2 of them a token),
// keeps cosine and sine in shared memory and turns every query and key head of
// those tokens in the same pass: one launch for q and k.  32 bytes an access
// where the layout allows it, two or four rows of a thread in flight.
// Measured: [2, 8190, 32 + 32, 64] fp16, three axes, neighbouring pairs 44 us =
// 5.9 TB/s (89 % of the measured copy bandwidth; 6.5 TB/s inside the kernel);
// [4, 4099, 32 + 8, 128] bf16 forward and backward 117 us = 5.8 TB/s in two
// launches; 64 tokens [32 + 8, 128] 2.7 us, the launch itself.
#include "ops_common.cuh"

namespace {

using namespace afa100;

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;   // of a CTA

struct RotaryParams {
  const char* in[2];  // q, k
  char* out[2];
  int64_t in_s[2][3];  // bytes
  int64_t out_s[2][3];
  const void* pos;
  int64_t pos_s[3];
  const float* inv_freq;
  int32_t axis_end[AFA_ROTARY_MAX_AXES];  // first pair behind each axis
  int32_t n_axes, pos_type;
  int32_t seq_len, n_heads, heads_all, head_dim, half;
  uint32_t heads_magic;      // ceil(2^32 / heads_all): row / heads_all is the high half of row * heads_magic
                             // (of more than one head; rows < 2^17)
  int32_t n_tokens, tokens;  // all of them, and of one CTA
  int32_t inverse;
};

// How a thread's channels lie in a row.
enum Layout {
  kHalvesWide,    // 16 of one half and the 16 that pair with them: two accesses of 32 bytes
  kHalvesNarrow,  // 8 and 8: two accesses of 16 bytes, for halves that are not a multiple of 16
  kNeighbours,    // 16 in a row, pairs side by side: one access of 32 bytes
};

__device__ __forceinline__ double load_position(const RotaryParams& p, int64_t at) {
  if (p.pos_type == AFA_POS_INT64) return static_cast<double>(static_cast<const long long*>(p.pos)[at]);
  if (p.pos_type == AFA_POS_INT32) return static_cast<double>(static_cast<const int*>(p.pos)[at]);
  return static_cast<double>(static_cast<const float*>(p.pos)[at]);
}

// Cosine and sine of an angle given in 64 bits.  1/(2 pi) in two parts, so the
// fraction of a turn keeps about 2^-50 even for angles of 10^9.
__device__ __forceinline__ float2 cos_sin(double angle) {
  const double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;
  const double turns = angle * kHi;
  double f = turns - rint(turns);
  f += fma(angle, kHi, -turns) + angle * kLo;
  float s, c;
  sincospif(static_cast<float>(2.0 * f), &s, &c);
  return make_float2(c, s);
}

// Each thread turns the same channels of several rows (a row: one head of one
// token), kUnroll of them at a time, and copies the channels behind rot_dim.
template <bool kBF16, Layout kLayout>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  constexpr int kPairs = kLayout == kHalvesWide ? 16 : 8;  // of a thread
  constexpr int kUnroll = kLayout == kHalvesWide ? 2 : 4;  // 128 bytes of loads in flight
  extern __shared__ float4 table[];  // [tokens][kPairs / 2][blocks of kPairs]: cos, sin, cos, sin
  __shared__ longlong2 base[kMaxTokens][2];  // a token's first q and k row: in, out
  const int token0 = blockIdx.x * p.tokens;
  const int n_tok = min(p.tokens, p.n_tokens - token0);
  const int blocks = p.half / kPairs;
  after_previous();
  if (threadIdx.x < 2 * n_tok) {
    const int t = threadIdx.x >> 1, w = threadIdx.x & 1;
    const int b = (token0 + t) / p.seq_len, n = (token0 + t) - b * p.seq_len;
    base[t][w] = make_longlong2(reinterpret_cast<long long>(p.in[w]) + b * p.in_s[w][0] + n * p.in_s[w][1],
                                reinterpret_cast<long long>(p.out[w]) + b * p.out_s[w][0] + n * p.out_s[w][1]);
  }
  for (int i = threadIdx.x; i < n_tok * p.half; i += kThreads) {
    const int t = i / p.half, j = i - t * p.half;
    const int b = (token0 + t) / p.seq_len, n = (token0 + t) - b * p.seq_len;
    int axis = 0;
    while (axis < p.n_axes - 1 && j >= p.axis_end[axis]) ++axis;
    const double pos = load_position(p, axis * p.pos_s[0] + b * p.pos_s[1] + n * p.pos_s[2]);
    float2 cs = cos_sin(pos * static_cast<double>(p.inv_freq[j]));
    if (p.inverse) cs.y = -cs.y;
    // neighbouring threads read neighbouring blocks: their entries lie side by side
    reinterpret_cast<float2*>(table + t * (p.half / 2) + j % kPairs / 2 * blocks + j / kPairs)[j & 1] = cs;
  }
  __syncthreads();

  const int per_row = p.head_dim / (2 * kPairs);
  const int j = threadIdx.x % per_row;
  const int step = kThreads / per_row;
  if (threadIdx.x >= step * per_row) return;
  const bool turned = j < blocks;
  // byte offsets of the thread's two pieces within a row
  const int off0 = kLayout == kNeighbours || !turned ? j * 4 * kPairs : j * 2 * kPairs;
  const int off1 = kLayout == kNeighbours || !turned ? off0 + 2 * kPairs : off0 + p.half * 2;
  const int rows = n_tok * p.heads_all;
  for (int r0 = threadIdx.x / per_row; r0 < rows; r0 += step * kUnroll) {
    uint32_t x[kUnroll][kPairs];  // the two pieces
    char* dst[kUnroll];
    int tok[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = r0 + u * step;
      dst[u] = nullptr;
      if (r < rows) {
        const int t = p.heads_all == 1 ? r : __umulhi(static_cast<uint32_t>(r), p.heads_magic);
        int h = r - t * p.heads_all;
        const int w = h >= p.n_heads;  // 0: q, 1: k
        if (w) h -= p.n_heads;
        const longlong2 at = base[t][w];
        const char* src = reinterpret_cast<const char*>(at.x) + h * p.in_s[w][2];
        dst[u] = reinterpret_cast<char*>(at.y) + h * p.out_s[w][2];
        tok[u] = t;
        if constexpr (kLayout == kHalvesWide) {
          load32<false>(reinterpret_cast<uint32_t(&)[2][4]>(x[u][0]), src + off0);
          load32<false>(reinterpret_cast<uint32_t(&)[2][4]>(x[u][8]), src + off1);
        } else if constexpr (kLayout == kNeighbours) {
          load32<false>(reinterpret_cast<uint32_t(&)[2][4]>(x[u][0]), src + off0);
        } else {
          reinterpret_cast<uint4&>(x[u][0]) = *reinterpret_cast<const uint4*>(src + off0);
          reinterpret_cast<uint4&>(x[u][4]) = *reinterpret_cast<const uint4*>(src + off1);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (dst[u] == nullptr) continue;
      if (turned) {
        const float4* cs = table + tok[u] * (p.half / 2) + j;
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
          const float4 c = cs[i * blocks];  // of pairs 2i and 2i + 1
          if constexpr (kLayout == kNeighbours) {
            const float2 v = unpack2<kBF16>(x[u][2 * i]), w = unpack2<kBF16>(x[u][2 * i + 1]);
            x[u][2 * i] = pack2<kBF16>(v.x * c.x - v.y * c.y, v.y * c.x + v.x * c.y);
            x[u][2 * i + 1] = pack2<kBF16>(w.x * c.z - w.y * c.w, w.y * c.z + w.x * c.w);
          } else {
            const float2 a = unpack2<kBF16>(x[u][i]), b = unpack2<kBF16>(x[u][i + kPairs / 2]);
            x[u][i] = pack2<kBF16>(a.x * c.x - b.x * c.y, a.y * c.z - b.y * c.w);
            x[u][i + kPairs / 2] = pack2<kBF16>(b.x * c.x + a.x * c.y, b.y * c.z + a.y * c.w);
          }
        }
      }
      if constexpr (kLayout == kHalvesWide) {
        store32(dst[u] + off0, reinterpret_cast<uint32_t(&)[2][4]>(x[u][0]));
        store32(dst[u] + off1, reinterpret_cast<uint32_t(&)[2][4]>(x[u][8]));
      } else if constexpr (kLayout == kNeighbours) {
        store32(dst[u] + off0, reinterpret_cast<uint32_t(&)[2][4]>(x[u][0]));
      } else {
        *reinterpret_cast<uint4*>(dst[u] + off0) = reinterpret_cast<uint4&>(x[u][0]);
        *reinterpret_cast<uint4*>(dst[u] + off1) = reinterpret_cast<uint4&>(x[u][4]);
      }
    }
  }
}

template <bool kBF16>
void launch_rotary(Layout layout, unsigned grid, size_t smem, cudaStream_t s, const RotaryParams& p) {
  if (layout == kNeighbours)
    ops_launch(rotary_kernel<kBF16, kNeighbours>, dim3(grid), kThreads, smem, s, p);
  else if (layout == kHalvesWide)
    ops_launch(rotary_kernel<kBF16, kHalvesWide>, dim3(grid), kThreads, smem, s, p);
  else
    ops_launch(rotary_kernel<kBF16, kHalvesNarrow>, dim3(grid), kThreads, smem, s, p);
}

}  // namespace

extern "C" int afa_rotary_sm100(const AfaRotaryArgs* a, void* stream) {
  if (a == nullptr) return AFA_ERR_INVALID_ARGUMENT;
  if (a->dtype != AFA_DTYPE_FP16 && a->dtype != AFA_DTYPE_BF16) return AFA_ERR_UNSUPPORTED_DTYPE;
  if (a->head_dim <= 0 || a->head_dim % 16 != 0 || a->head_dim > 512 || a->rot_dim < 16 || a->rot_dim % 16 != 0 ||
      a->rot_dim > a->head_dim)
    return AFA_ERR_NO_KERNEL;
  const bool has_k = a->k != nullptr;
  if (a->q == nullptr || a->q_out == nullptr || a->positions == nullptr || a->inv_freq == nullptr ||
      (has_k && a->k_out == nullptr))
    return AFA_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->seq_len <= 0 || a->n_heads <= 0 || (has_k && a->n_k_heads <= 0))
    return AFA_ERR_INVALID_ARGUMENT;
  if (a->n_axes < 1 || a->n_axes > AFA_ROTARY_MAX_AXES || a->pos_type < AFA_POS_INT32 || a->pos_type > AFA_POS_FP32 ||
      (a->interleaved != 0 && a->interleaved != 1) || (a->inverse != 0 && a->inverse != 1))
    return AFA_ERR_INVALID_ARGUMENT;
  RotaryParams p{};
  int64_t pairs = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    if (a->sections[i] < 0) return AFA_ERR_INVALID_ARGUMENT;
    pairs += a->sections[i];
    p.axis_end[i] = static_cast<int32_t>(pairs > INT32_MAX ? INT32_MAX : pairs);
  }
  if (pairs != a->rot_dim / 2) return AFA_ERR_INVALID_ARGUMENT;
  const uintptr_t pos_mask = a->pos_type == AFA_POS_INT64 ? 7u : 3u;
  if (!ops_aligned16(a->q) || !ops_aligned16(a->q_out) || !ops_aligned16(a->k) || !ops_aligned16(a->k_out) ||
      (reinterpret_cast<uintptr_t>(a->positions) & pos_mask) != 0u ||
      (reinterpret_cast<uintptr_t>(a->inv_freq) & 3u) != 0u)
    return AFA_ERR_MISALIGNED;
  if (!ops_strides_ok(a->q_strides, a->batch, a->seq_len, a->n_heads, false) ||
      !ops_strides_ok(a->q_out_strides, a->batch, a->seq_len, a->n_heads, true))
    return AFA_ERR_MISALIGNED;
  if (has_k && (!ops_strides_ok(a->k_strides, a->batch, a->seq_len, a->n_k_heads, false) ||
                !ops_strides_ok(a->k_out_strides, a->batch, a->seq_len, a->n_k_heads, true)))
    return AFA_ERR_MISALIGNED;
  const int64_t tokens = int64_t{1} * a->batch * a->seq_len;
  const int64_t heads = int64_t{1} * a->n_heads + (has_k ? a->n_k_heads : 0);
  if (tokens > INT32_MAX - 64 || heads > AFA_ROTARY_MAX_HEADS) return AFA_ERR_TOO_LARGE;

  int dev = 0, sms = 0;
  const int rc = ops_device(&dev, &sms);
  if (rc != AFA_OK) return rc;

  p.in[0] = static_cast<const char*>(a->q);
  p.out[0] = static_cast<char*>(a->q_out);
  p.in[1] = static_cast<const char*>(a->k);
  p.out[1] = static_cast<char*>(a->k_out);
  for (int i = 0; i < 3; ++i) {
    p.in_s[0][i] = a->q_strides[i] * 2;
    p.out_s[0][i] = a->q_out_strides[i] * 2;
    p.in_s[1][i] = a->k_strides[i] * 2;
    p.out_s[1][i] = a->k_out_strides[i] * 2;
    p.pos_s[i] = a->pos_strides[i];
  }
  p.pos = a->positions;
  p.inv_freq = a->inv_freq;
  p.n_axes = a->n_axes;
  p.pos_type = a->pos_type;
  p.seq_len = a->seq_len;
  p.n_heads = a->n_heads;
  p.heads_all = static_cast<int32_t>(heads);
  p.head_dim = a->head_dim;
  p.half = a->rot_dim / 2;
  p.n_tokens = static_cast<int32_t>(tokens);
  p.inverse = a->inverse;
  p.heads_magic = static_cast<uint32_t>(((uint64_t{1} << 32) + heads - 1) / heads);
  const Layout layout = a->interleaved                                             ? kNeighbours
                        : p.half % 16 == 0 && (a->head_dim - a->rot_dim) % 32 == 0 ? kHalvesWide
                                                                                   : kHalvesNarrow;
  // Tokens a CTA: as many as keep each thread busy for two rounds of loads, unless
  // the GPU would then have fewer than four CTAs an SM.
  const int rows = layout == kHalvesWide ? 4 * (kThreads / (a->head_dim / 32)) : 8 * (kThreads / (a->head_dim / 16));
  int64_t t = (rows + heads - 1) / heads;
  const int64_t fill = tokens / (4 * static_cast<int64_t>(sms));
  t = t > fill ? fill : t;
  t = t < 1 ? 1 : (t > kMaxTokens ? kMaxTokens : t);
  p.tokens = static_cast<int32_t>(t);
  const unsigned grid = static_cast<unsigned>((tokens + t - 1) / t);
  const size_t smem = static_cast<size_t>(t) * p.half * sizeof(float2);  // at most 16 * 256 * 8 = 32 KB
  const auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == AFA_DTYPE_BF16)
    launch_rotary<true>(layout, grid, smem, s, p);
  else
    launch_rotary<false>(layout, grid, smem, s, p);
  return ops_launched();
}
