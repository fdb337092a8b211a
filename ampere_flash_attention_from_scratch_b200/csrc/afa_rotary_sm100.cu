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
// those tokens in the same pass: one launch for q and k.
#include "ops_common.cuh"

namespace {

using namespace afa100;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows a thread has in flight: 8 loads of 16 bytes

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
  int32_t n_tokens, tokens;  // all of them, and of one CTA
  int32_t inverse;
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

// A thread turns 16 channels of a row: channels [8j, 8j + 8) of both halves, or
// 16 neighbouring ones when pairs are interleaved -- 8 pairs either way -- and
// copies 16 neighbouring ones behind rot_dim.
template <bool kBF16, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 table[];  // [tokens][half]: cosine, sine
  const int token0 = blockIdx.x * p.tokens;
  const int n_tok = min(p.tokens, p.n_tokens - token0);
  for (int i = threadIdx.x; i < n_tok * p.half; i += kThreads) {
    const int t = i / p.half, j = i - t * p.half;
    const int b = (token0 + t) / p.seq_len, n = (token0 + t) - b * p.seq_len;
    int axis = 0;
    while (axis < p.n_axes - 1 && j >= p.axis_end[axis]) ++axis;
    const double pos = load_position(p, axis * p.pos_s[0] + b * p.pos_s[1] + n * p.pos_s[2]);
    float2 cs = cos_sin(pos * static_cast<double>(p.inv_freq[j]));
    if (p.inverse) cs.y = -cs.y;
    table[i] = cs;
  }
  __syncthreads();

  const int per_row = p.head_dim >> 4;
  const int j = threadIdx.x % per_row;
  const int rows_step = kThreads / per_row;
  const bool turned = j < (p.half >> 3);
  // byte offsets of the thread's two 16-byte pieces within a row
  const int off0 = kInterleaved || !turned ? j * 32 : j * 16;
  const int off1 = kInterleaved || !turned ? off0 + 16 : off0 + p.half * 2;
  const int rows = n_tok * p.heads_all;
  if (threadIdx.x >= rows_step * per_row) return;
  for (int r0 = threadIdx.x / per_row; r0 < rows; r0 += rows_step * kUnroll) {
    uint4 x[kUnroll], y[kUnroll];
    char* dst[kUnroll];
    int tok[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = r0 + u * rows_step;
      dst[u] = nullptr;
      if (r < rows) {
        const int t = r / p.heads_all, h = r - t * p.heads_all;
        const int b = (token0 + t) / p.seq_len, n = (token0 + t) - b * p.seq_len;
        const int w = h >= p.n_heads;  // 0: q, 1: k
        const int hh = w ? h - p.n_heads : h;
        const char* src = p.in[w] + b * p.in_s[w][0] + n * p.in_s[w][1] + hh * p.in_s[w][2];
        dst[u] = p.out[w] + b * p.out_s[w][0] + n * p.out_s[w][1] + hh * p.out_s[w][2];
        tok[u] = t;
        x[u] = *reinterpret_cast<const uint4*>(src + off0);
        y[u] = *reinterpret_cast<const uint4*>(src + off1);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (dst[u] == nullptr) continue;
      if (turned) {
        const float2* cs = table + tok[u] * p.half + j * 8;
        uint32_t* xs = reinterpret_cast<uint32_t*>(&x[u]);
        uint32_t* ys = reinterpret_cast<uint32_t*>(&y[u]);
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t& w = i < 4 ? xs[i] : ys[i - 4];
            const float2 v = unpack2<kBF16>(w);
            const float2 c = cs[i];
            w = pack2<kBF16>(v.x * c.x - v.y * c.y, v.y * c.x + v.x * c.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 a = unpack2<kBF16>(xs[i]), b = unpack2<kBF16>(ys[i]);
            const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
            xs[i] = pack2<kBF16>(a.x * c0.x - b.x * c0.y, a.y * c1.x - b.y * c1.y);
            ys[i] = pack2<kBF16>(b.x * c0.x + a.x * c0.y, b.y * c1.x + a.y * c1.y);
          }
        }
      }
      *reinterpret_cast<uint4*>(dst[u] + off0) = x[u];
      *reinterpret_cast<uint4*>(dst[u] + off1) = y[u];
    }
  }
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
  if (tokens > INT32_MAX - 64 || heads > 65536) return AFA_ERR_TOO_LARGE;

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
  // Tokens a CTA: as many as give each thread kUnroll rows, unless the GPU would
  // then have fewer than four CTAs an SM.
  const int per_row = a->head_dim / 16;
  int64_t t = (int64_t{kUnroll} * (kThreads / per_row) + heads - 1) / heads;
  const int64_t fill = tokens / (4 * static_cast<int64_t>(sms));
  t = t > fill ? fill : t;
  t = t < 1 ? 1 : (t > 16 ? 16 : t);
  p.tokens = static_cast<int32_t>(t);
  const unsigned grid = static_cast<unsigned>((tokens + t - 1) / t);
  const size_t smem = static_cast<size_t>(t) * p.half * sizeof(float2);  // at most 16 * 256 * 8 = 32 KB
  const auto s = static_cast<cudaStream_t>(stream);
  if (a->dtype == AFA_DTYPE_BF16) {
    if (a->interleaved)
      rotary_kernel<true, true><<<grid, kThreads, smem, s>>>(p);
    else
      rotary_kernel<true, false><<<grid, kThreads, smem, s>>>(p);
  } else {
    if (a->interleaved)
      rotary_kernel<false, true><<<grid, kThreads, smem, s>>>(p);
    else
      rotary_kernel<false, false><<<grid, kThreads, smem, s>>>(p);
  }
  return ops_launched();
}
