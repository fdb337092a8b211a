// ops_common.cuh -- what the launchers and kernels of the cache operators and
// of the rotary positions (include/afa_sm100_ops.h) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "afa_sm100_ops.h"

namespace afa100 {

constexpr int kOpsMaxDevices = 64;

// Current device, its SM count and that it is compute capability 10.0; probed
// once per device.
inline int ops_device(int* dev_out, int* sm_count_out) {
  static std::mutex mu;
  static int sms[kOpsMaxDevices] = {};  // 0: not probed, -1: another architecture
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kOpsMaxDevices) {
    cudaGetLastError();
    return AFA_ERR_NO_DEVICE;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (sms[dev] == 0) {
    int major = 0, minor = 0, n = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return AFA_ERR_NO_DEVICE;
    }
    sms[dev] = major == 10 && minor == 0 ? n : -1;
  }
  if (sms[dev] < 0) return AFA_ERR_ARCH;
  *dev_out = dev;
  *sm_count_out = sms[dev];
  return AFA_OK;
}

inline int ops_launched() {
  if (cudaGetLastError() != cudaSuccess) return AFA_ERR_LAUNCH;
  return AFA_OK;
}

// A launch whose CTAs may take their places while the stream's kernel before
// it ends; the kernel calls after_previous() before it touches global memory.
// Calls in a row, plain -> so: rotary of 64 tokens 4.2 -> 2.8 us, a token
// written to 128 sequences and read back 8.3 -> 5.2, attention over 500 tokens
// 10.3 -> 8.3, over 32 x 256..8192 45.9 -> 41.9, over 8 x 131072 237 -> 231; 8
// prompts written and read back 70.4 -> 66.5, 131072 tokens read back 110.7 ->
// 109.3.  Among other work no case is slower either (8 x 131072 264 -> 262).
template <class... P, class... A>
inline cudaError_t ops_launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                              const A&... args) {
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Waits until the stream's earlier kernels have ended and their writes are
// seen, then lets the next one's CTAs in: in this order, so that whatever that
// one reads before its own wait is not written by kernels before this one.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

inline bool ops_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }

// Strides (batch, seq, head) of a 16-bit tensor whose rows are moved 16 bytes
// at a time; a stride of a size-1 dimension is never used.  Inputs may repeat
// (stride 0), outputs may not.
inline bool ops_strides_ok(const int64_t s[3], int64_t batch, int64_t seq, int64_t heads, bool output) {
  const int64_t ext[3] = {batch, seq, heads};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && (s[i] % 8 != 0 || s[i] < (output ? 8 : 0))) return false;
  return true;
}

// Two 16-bit values of a 32-bit word as fp32 and back.
template <bool kBF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kBF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}
template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// 32 bytes at a time: the row strides and addresses are multiples of 16, so where
// the address is not one of 32 they go as two halves.  kOnce: read by no other
// thread, so not kept in L1.  (Not by ld.global.nc either way: the kernel is on the
// GPU while the one before it still writes what it will read.)
template <bool kOnce>
__device__ __forceinline__ void load32(uint32_t (&v)[2][4], const char* p) {
  if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0u) {
    if constexpr (kOnce)
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[1][0]), "=r"(v[1][1]),
                     "=r"(v[1][2]), "=r"(v[1][3])
                   : "l"(p)
                   : "memory");
    else
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[1][0]), "=r"(v[1][1]),
                     "=r"(v[1][2]), "=r"(v[1][3])
                   : "l"(p)
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 h = *reinterpret_cast<const uint4*>(p + 16 * i);
      v[i][0] = h.x;
      v[i][1] = h.y;
      v[i][2] = h.z;
      v[i][3] = h.w;
    }
  }
}
__device__ __forceinline__ void store32(char* p, const uint32_t (&v)[2][4]) {
  if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0u) {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0][0]), "r"(v[0][1]), "r"(v[0][2]),
                 "r"(v[0][3]), "r"(v[1][0]), "r"(v[1][1]), "r"(v[1][2]), "r"(v[1][3]), "l"(p)
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<uint4*>(p + 16 * i) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
  }
}

// The kernels' report of a bad table entry or length (include/afa_sm100_ops.h).
__device__ __forceinline__ void report(int32_t* status, int32_t code) {
  if (status != nullptr) *static_cast<volatile int32_t*>(status) = code;
}

// A sequence's lengths as the cache kernels use them: new rows and the position
// of row 0, or no rows at all (reported) where they contradict each other.
struct NewRows {
  int count;
  int first;
};
__device__ __forceinline__ NewRows new_rows(const AfaCache4& c, int b, int seq_len) {
  const int kv = c.kv_lens[b];
  const int fresh = c.new_lens != nullptr ? c.new_lens[b] : seq_len;
  if (kv < 0 || static_cast<int64_t>(kv) > static_cast<int64_t>(c.max_pages) * c.page_size || fresh < 0 ||
      fresh > seq_len || fresh > kv) {
    report(c.status, AFA_DEV_BAD_LENGTH);
    return NewRows{0, 0};
  }
  return NewRows{fresh, kv - fresh};
}

inline int ops_log2(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// The cache argument's own checks, shared by the three cache operators.
inline int ops_check_cache(const AfaCache4* c) {
  if (c == nullptr) return AFA_ERR_INVALID_ARGUMENT;
  if (c->dtype != AFA_DTYPE_FP16 && c->dtype != AFA_DTYPE_BF16) return AFA_ERR_UNSUPPORTED_DTYPE;
  if (c->head_dim != 64 && c->head_dim != 128) return AFA_ERR_NO_KERNEL;
  if (c->cache == nullptr || c->page_table == nullptr || c->kv_lens == nullptr) return AFA_ERR_INVALID_ARGUMENT;
  if (c->n_pages <= 0 || c->max_pages <= 0 || c->batch <= 0 || c->n_kv_heads <= 0) return AFA_ERR_INVALID_ARGUMENT;
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
    return AFA_ERR_INVALID_ARGUMENT;
  if (!ops_aligned16(c->cache) || c->page_stride % 16 != 0) return AFA_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(c->page_table) & 3u) != 0u || (reinterpret_cast<uintptr_t>(c->kv_lens) & 3u) != 0u ||
      (reinterpret_cast<uintptr_t>(c->new_lens) & 3u) != 0u || (reinterpret_cast<uintptr_t>(c->status) & 3u) != 0u)
    return AFA_ERR_MISALIGNED;
  const int64_t page_bytes = int64_t{2} * c->n_kv_heads * c->page_size * afa_cache4_row_bytes(c->head_dim);
  if (c->n_pages > 1 && c->page_stride < page_bytes) return AFA_ERR_INVALID_ARGUMENT;
  if (c->batch > 1 && c->table_stride < 0) return AFA_ERR_INVALID_ARGUMENT;
  if (int64_t{1} * c->max_pages * c->page_size > INT32_MAX - 8192) return AFA_ERR_TOO_LARGE;
  return AFA_OK;
}

}  // namespace afa100
