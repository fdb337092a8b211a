// afa_fwd_sm100.cu -- C-ABI launcher of the sm_100a attention forward kernel
// (declared in include/afa_sm100.h).
//
// Replaces the launch half of the reference's torch binding
// (csrc/ampere_flash_attention.cu:35-136), its std::map kernel table
// (csrc/include/afa_preset_kernels.cuh:10-54) and the import-time shared-memory
// attribute setup (csrc/ampere_flash_attention.cu:143-150).  Differences, by
// design:
//   * no torch types: plain pointers, element strides and a cudaStream_t;
//   * the kernel table is keyed on (dtype, head_dim) -- the sm_100a kernel has
//     one tiling per head_dim, so the reference's Ampere tiling knobs do not
//     select anything here;
//   * the max-dynamic-smem attribute is set lazily per device on first use, so
//     processes that pick their device after loading the library work;
//   * every argument is validated before any CUDA call and every failure is a
//     return code; the launch itself is error-checked;
//   * beyond the reference: K/V length and head count of their own (GQA), a
//     causal mask and a log-sum-exp output (AfaFwdArgs extension fields).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "afa_fwd_kernel.cuh"
#include "afa_sm100.h"
#include "afa_sm100_ops.h"
#include "ops_sites.h"

namespace {

using afa100::FwdLayout;
using afa100::FwdParams;

// One (dtype, head_dim) preset: two kernel instances, [0] without and [1] with
// the causal mask (a template parameter, so the unmasked kernel carries none of
// the mask's per-tile work).
struct KernelEntry {
  int dtype;
  int head_dim;
  int stages;
  unsigned smem_bytes;
  cudaError_t (*set_smem_attr[2])();
  cudaError_t (*launch[2])(const FwdParams&, dim3, cudaStream_t);
};

// Per-device one-time setup of a kernel instance: raise its dynamic shared
// memory limit and verify that it is launched with exactly the register count
// the warpgroup register split (setmaxnreg) is sized for -- with fewer, the
// softmax warpgroups' setmaxnreg.inc could never be satisfied.
template <int kD, bool kBF16, int kStages, bool kCausal>
cudaError_t set_smem_attr_impl() {
  using L = FwdLayout<kD, kBF16, kStages>;
  cudaError_t e = cudaFuncSetAttribute(afa100::afa_fwd_sm100_kernel<kD, kBF16, kStages, kCausal>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(L::kSmemBytes));
  if (e != cudaSuccess) return e;
  cudaFuncAttributes attr{};
  e = cudaFuncGetAttributes(&attr, afa100::afa_fwd_sm100_kernel<kD, kBF16, kStages, kCausal>);
  if (e != cudaSuccess) return e;
  if (attr.numRegs != L::kLaunchRegs || attr.maxThreadsPerBlock < L::kThreads)
    return cudaErrorInvalidKernelImage;
  return cudaSuccess;
}

template <int kD, bool kBF16, int kStages, bool kCausal>
cudaError_t launch_impl(const FwdParams& p, dim3 grid, cudaStream_t stream) {
  using L = FwdLayout<kD, kBF16, kStages>;
  afa100::afa_fwd_sm100_kernel<kD, kBF16, kStages, kCausal>
      <<<grid, L::kThreads, L::kSmemBytes, stream>>>(p);
  return cudaGetLastError();
}

#define AFA_PRESET(DTYPE, HEAD_DIM, IS_BF16, STAGES)                                              \
  KernelEntry{DTYPE,                                                                             \
              HEAD_DIM,                                                                          \
              STAGES,                                                                            \
              FwdLayout<HEAD_DIM, IS_BF16, STAGES>::kSmemBytes,                                  \
              {&set_smem_attr_impl<HEAD_DIM, IS_BF16, STAGES, false>,                            \
               &set_smem_attr_impl<HEAD_DIM, IS_BF16, STAGES, true>},                            \
              {&launch_impl<HEAD_DIM, IS_BF16, STAGES, false>, &launch_impl<HEAD_DIM, IS_BF16, STAGES, true>}},

// Generated by csrc/generate_preset_kernels.py from
// afa_config.get_sm100_preset_configs().
const KernelEntry kKernels[] = {
#include "afa_preset_kernels.inc"
};
constexpr int kNumKernels = sizeof(kKernels) / sizeof(kKernels[0]);
constexpr int kMaxDevices = 64;

const KernelEntry* find_kernel(int dtype, int head_dim) {
  for (int i = 0; i < kNumKernels; ++i)
    if (kKernels[i].dtype == dtype && kKernels[i].head_dim == head_dim) return &kKernels[i];
  return nullptr;
}

int kernel_index(const KernelEntry* e) { return static_cast<int>(e - kKernels); }

struct DeviceState {
  bool probed = false;
  int cc = 0;
  int sm_count = 0;
  bool attr_set[kNumKernels][2] = {};
};
std::mutex g_mu;
DeviceState g_dev[kMaxDevices];

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::atomic<EncodeTiledFn> g_encode{nullptr};

// cuTensorMapEncodeTiled is fetched through the runtime's driver entry point so
// that this library does not link libcuda (it loads on machines without a GPU).
// Threads making their first call at the same time may each look it up; they
// store the same address.
int get_encode_fn(EncodeTiledFn* out) {
  EncodeTiledFn f = g_encode.load(std::memory_order_acquire);
  if (f == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || fn == nullptr) {
      cudaGetLastError();
      return AFA_ERR_TENSOR_MAP;
    }
    f = reinterpret_cast<EncodeTiledFn>(fn);
    g_encode.store(f, std::memory_order_release);
  }
  *out = f;
  return AFA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }

// Strides of size-1 dimensions are never used to address memory; they are
// ignored by the checks and normalised for the tensor map.
bool stride_ok(int64_t stride, int64_t extent) { return extent == 1 || (stride > 0 && stride % 8 == 0); }

// Encodes one Q/K/V/O tensor ([batch, seq, head, head_dim] with element
// strides s[0..2] and unit head_dim stride) as a 4-D tiled tensor map with dims
// ordered by increasing stride, box 64 head_dim elements x box_rows rows.  Sets
// *seq_inner when seq is dimension 1.
int encode_qkv(CUtensorMap* map, const void* ptr, const int64_t s[3], int B, int N, int H, int D,
               int dtype, bool* seq_inner, unsigned box_rows = 128u) {
  EncodeTiledFn enc = nullptr;
  int rc = get_encode_fn(&enc);
  if (rc != AFA_OK) return rc;
  const int64_t esz = 2;
  int64_t sb = s[0], sn = s[1], sh = s[2];
  bool si;
  if (H == 1)
    si = true;
  else if (N == 1)
    si = false;
  else
    si = sn < sh;
  // normalise unused strides so the nested-stride layout TMA expects holds
  if (si) {
    if (N == 1) sn = D;
    if (H == 1) sh = sn * N;
    if (B == 1) sb = sh * H;
  } else {
    if (H == 1) sh = D;
    if (N == 1) sn = sh * H;
    if (B == 1) sb = sn * N;
  }
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D),
                              static_cast<cuuint64_t>(si ? N : H),
                              static_cast<cuuint64_t>(si ? H : N), static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>((si ? sn : sh) * esz),
                                 static_cast<cuuint64_t>((si ? sh : sn) * esz),
                                 static_cast<cuuint64_t>(sb * esz)};
  const cuuint32_t box[4] = {64u, si ? box_rows : 1u, si ? 1u : box_rows, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUtensorMapDataType dt =
      dtype == AFA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = enc(map, dt, 4, const_cast<void*>(ptr), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return AFA_ERR_TENSOR_MAP;
  *seq_inner = si;
  return AFA_OK;
}

// K/V rows and heads after the zero-selects-default rule of the extension fields.
int kv_len(const AfaFwdArgs* a) { return a->seq_len_kv > 0 ? a->seq_len_kv : a->seq_len; }
int kv_heads(const AfaFwdArgs* a) { return a->n_kv_heads > 0 ? a->n_kv_heads : a->n_heads; }

int validate(const AfaFwdArgs* a) {
  if (a == nullptr) return AFA_ERR_INVALID_ARGUMENT;
  if (a->dtype != AFA_DTYPE_FP16 && a->dtype != AFA_DTYPE_BF16) return AFA_ERR_UNSUPPORTED_DTYPE;
  if (find_kernel(a->dtype, a->head_dim) == nullptr) return AFA_ERR_NO_KERNEL;
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->o == nullptr)
    return AFA_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->seq_len <= 0 || a->n_heads <= 0) return AFA_ERR_INVALID_ARGUMENT;
  if (a->seq_len_kv < 0 || a->n_kv_heads < 0 || (a->causal != 0 && a->causal != 1))
    return AFA_ERR_INVALID_ARGUMENT;
  const int n_kv = kv_len(a), h_kv = kv_heads(a);
  if (a->n_heads % h_kv != 0) return AFA_ERR_INVALID_ARGUMENT;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o))
    return AFA_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0u) return AFA_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(a->sched) & 7u) != 0u) return AFA_ERR_MISALIGNED;
  const int64_t ext_q[3] = {a->batch, a->seq_len, a->n_heads};
  const int64_t ext_kv[3] = {a->batch, n_kv, h_kv};
  const int64_t* all[4] = {a->q_strides, a->k_strides, a->v_strides, a->o_strides};
  for (int t = 0; t < 4; ++t) {
    const int64_t* ext = (t == 1 || t == 2) ? ext_kv : ext_q;
    for (int d = 0; d < 3; ++d)
      if (!stride_ok(all[t][d], ext[d])) return AFA_ERR_MISALIGNED;
  }
  // Work items and TMA coordinates are 32-bit.
  const int64_t n_q_pairs = (static_cast<int64_t>(a->seq_len) + 255) / 256;
  if (static_cast<int64_t>(a->batch) * a->n_heads * n_q_pairs > INT32_MAX) return AFA_ERR_TOO_LARGE;
  if (a->seq_len > (INT32_MAX - 512) || n_kv > (INT32_MAX - 512)) return AFA_ERR_TOO_LARGE;
  return AFA_OK;
}

// Scratch memory of afa_fwd_sm100_noalloc, for callers that may not allocate
// device memory: a static device array inside this library (one instance per
// device that loads it, kept until the process exits), used instead of
// caller-provided scheduler words.  In host code this name stands for a
// host-side shadow, not a device address, so it is never passed to a kernel:
// noalloc_scratch() asks the runtime for the device address.
static __device__ __align__(256) int32_t g_noalloc_scratch[AFA_NOALLOC_SCRATCH_BYTES / sizeof(int32_t)];

// Device address of g_noalloc_scratch on device `dev`, which must be the
// current device; looked up on the first call that needs it on that device
// (before any stream capture, as the header says) and kept.
int32_t* g_noalloc_ptr[kMaxDevices] = {};

int noalloc_scratch(int dev, int32_t** out) {
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_noalloc_ptr[dev] == nullptr) {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_noalloc_scratch) != cudaSuccess || ptr == nullptr) {
      cudaGetLastError();
      return AFA_ERR_LAUNCH;
    }
    g_noalloc_ptr[dev] = static_cast<int32_t*>(ptr);
  }
  *out = g_noalloc_ptr[dev];
  return AFA_OK;
}

// Bytes of scratch memory one call needs: the causal kernel's two scheduler
// words; nothing otherwise.
size_t scratch_bytes(const AfaFwdArgs* a) { return a->causal ? 2 * sizeof(int32_t) : 0; }

int fwd_impl(const AfaFwdArgs* a, void* stream, bool noalloc);

}  // namespace

extern "C" {

int afa_sm100_version(void) { return 300; }

int afa_fwd_sm100_threads(void) { return FwdLayout<128, false, 4>::kThreads; }

int afa_fwd_sm100_supported(int32_t dtype, int32_t head_dim) {
  return find_kernel(dtype, head_dim) != nullptr ? 1 : 0;
}

int afa_fwd_sm100_smem_bytes(int32_t dtype, int32_t head_dim) {
  const KernelEntry* e = find_kernel(dtype, head_dim);
  return e ? static_cast<int>(e->smem_bytes) : -1;
}

const char* afa_strerror(int code) {
  switch (code) {
    case AFA_OK: return "success";
    case AFA_ERR_INVALID_ARGUMENT: return "invalid argument (null pointer or non-positive size)";
    case AFA_ERR_UNSUPPORTED_DTYPE: return "Only fp16 and bf16 are supported";
    case AFA_ERR_NO_KERNEL: return "Kernel configuration was not found: no sm_100a kernel for this (dtype, head_dim)";
    case AFA_ERR_MISALIGNED: return "tensor base address or stride is not 16-byte aligned, or head_dim is not contiguous";
    case AFA_ERR_NO_DEVICE: return "no current CUDA device";
    case AFA_ERR_ARCH: return "the sm_100a kernel requires a compute capability 10.0 device (B200)";
    case AFA_ERR_TENSOR_MAP: return "cuTensorMapEncodeTiled rejected a tensor (layout not expressible as a TMA descriptor)";
    case AFA_ERR_LAUNCH: return "kernel launch failed";
    case AFA_ERR_DEVICE_TIMEOUT: return "a device-side bounded wait ran out; the kernel aborted";
    case AFA_ERR_TOO_LARGE: return "problem size exceeds 32-bit work-item / coordinate indexing";
    case AFA_ERR_SCRATCH_LIMIT: return "the call needs more scratch memory than it may use (afa_fwd_sm100_noalloc: AFA_NOALLOC_SCRATCH_BYTES; afa_cache4_fwd_sm100: workspace_bytes)";
    default: return "unknown error";
  }
}

const char* afa_status_string(int32_t status) {
  if (status == AFA_DEV_OK) return "ok";
  if (status == AFA_DEV_BAD_PAGE) return "cache: a page_table entry in use is not a page of the cache";
  if (status == AFA_DEV_BAD_LENGTH) return "cache: a sequence's kv_lens or new_lens is negative or too large";
  switch (status - AFA_DEV_TIMEOUT_BASE) {
    case afa100::kSiteLoadQEmpty: return "timeout: TMA producer waiting for a free Q buffer";
    case afa100::kSiteLoadKVEmpty: return "timeout: TMA producer waiting for a free K/V slot";
    case afa100::kSiteMmaQFull: return "timeout: MMA waiting for the Q tiles";
    case afa100::kSiteMmaKFull: return "timeout: MMA waiting for a K tile";
    case afa100::kSiteMmaVFull: return "timeout: MMA waiting for a V tile";
    case afa100::kSiteMmaP0: return "timeout: MMA waiting for P of Q tile 0";
    case afa100::kSiteMmaP1: return "timeout: MMA waiting for P of Q tile 1";
    case afa100::kSiteSoftmaxS: return "timeout: softmax waiting for S";
    case afa100::kSiteSoftmaxO: return "timeout: epilogue waiting for the final O";
    case afa100::kSiteMmaDrain: return "timeout: draining outstanding MMAs at exit";
    case afa100::kSiteLoadItem: return "timeout: TMA producer waiting for a free work-item slot";
    case afa100::kSiteReadItem: return "timeout: waiting for the next claimed work item";
    case afa100::kSiteCorrAlpha: return "timeout: correction warp waiting for row scale factors";
    case afa100::kSiteCorrStats: return "timeout: correction warp waiting for the final row sums";
    case afa100::kSiteMmaOFree: return "timeout: MMA waiting for the previous item's O to be read out";
    case afa100::kSiteWideQ: return "timeout: cache MMA waiting for the Q tile";
    case afa100::kSiteWideKFull: return "timeout: cache MMA waiting for a K tile";
    case afa100::kSiteWideVFull: return "timeout: cache MMA or softmax waiting for a V tile";
    case afa100::kSiteWideS: return "timeout: cache softmax or loads waiting for S";
    case afa100::kSiteWideP: return "timeout: cache MMA waiting for P";
    case afa100::kSiteWidePv: return "timeout: cache loads or epilogue waiting for O";
    case afa100::kSiteWideDrain: return "timeout: draining outstanding cache MMAs at exit";
    default: return "unknown device status";
  }
}

int afa_fwd_sm100(const AfaFwdArgs* a, void* stream) { return fwd_impl(a, stream, false); }

int afa_fwd_sm100_noalloc(const AfaFwdArgs* a, void* stream) { return fwd_impl(a, stream, true); }

}  // extern "C"

namespace {

// The launch path of both entry points.  `noalloc`: the scheduler words come
// from g_noalloc_scratch (cleared on `stream` before the launch) and
// a->sched must be NULL.
int fwd_impl(const AfaFwdArgs* a, void* stream, bool noalloc) {
  int rc = validate(a);
  if (rc != AFA_OK) return rc;
  if (noalloc) {
    if (a->sched != nullptr) return AFA_ERR_INVALID_ARGUMENT;
    if (scratch_bytes(a) > AFA_NOALLOC_SCRATCH_BYTES) return AFA_ERR_SCRATCH_LIMIT;
  }
  const KernelEntry* ke = find_kernel(a->dtype, a->head_dim);

  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return AFA_ERR_NO_DEVICE;
  }
  int sm_count = 0;
  {
    std::lock_guard<std::mutex> lock(g_mu);
    DeviceState& ds = g_dev[dev];
    if (!ds.probed) {
      int major = 0, minor = 0;
      if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
          cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess ||
          cudaDeviceGetAttribute(&ds.sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return AFA_ERR_NO_DEVICE;
      }
      ds.cc = major * 10 + minor;
      ds.probed = true;
    }
    if (ds.cc != 100) return AFA_ERR_ARCH;
    const int ki = kernel_index(ke);
    const int ci = a->causal;
    if (!ds.attr_set[ki][ci]) {
      if (ke->set_smem_attr[ci]() != cudaSuccess) {
        cudaGetLastError();
        return AFA_ERR_LAUNCH;
      }
      ds.attr_set[ki][ci] = true;
    }
    sm_count = ds.sm_count;
  }

  FwdParams p{};
  bool si_q = false, si_k = false, si_v = false;
  const int n_kv = kv_len(a), h_kv = kv_heads(a);
  rc = encode_qkv(&p.tm_q, a->q, a->q_strides, a->batch, a->seq_len, a->n_heads, a->head_dim,
                  a->dtype, &si_q);
  if (rc == AFA_OK)
    rc = encode_qkv(&p.tm_k, a->k, a->k_strides, a->batch, n_kv, h_kv, a->head_dim, a->dtype, &si_k);
  if (rc == AFA_OK)
    rc = encode_qkv(&p.tm_v, a->v, a->v_strides, a->batch, n_kv, h_kv, a->head_dim, a->dtype, &si_v);
  bool si_o = false;
  if (rc == AFA_OK && (FwdLayout<128, false, 4>::kCorr || FwdLayout<128, false, 4>::kOTma))  // O is TMA-stored
    rc = encode_qkv(&p.tm_o, a->o, a->o_strides, a->batch, a->seq_len, a->n_heads, a->head_dim, a->dtype,
                    &si_o, 32u);
  if (rc != AFA_OK) return rc;
  p.seq_inner_mask = (si_q ? 1u : 0u) | (si_k ? 2u : 0u) | (si_v ? 4u : 0u) | (si_o ? 8u : 0u);
  p.o = a->o;
  p.o_sb = a->o_strides[0];
  p.o_sn = a->o_strides[1];
  p.o_sh = a->o_strides[2];
  p.seq_len = a->seq_len;
  p.seq_len_kv = n_kv;
  p.n_heads = a->n_heads;
  p.kv_group = a->n_heads / h_kv;
  p.n_q_pairs = (a->seq_len + 255) / 256;
  p.n_kv = (n_kv + 127) / 128;
  p.n_work = a->batch * a->n_heads * p.n_q_pairs;
  const afa100::DivMagic dq = afa100::DivMagic::make(p.n_q_pairs), dh = afa100::DivMagic::make(a->n_heads);
  p.qp_mul = dq.mul;
  p.qp_shift = dq.shift;
  p.h_mul = dh.mul;
  p.h_shift = dh.shift;
  p.causal_off = n_kv - a->seq_len;
  p.lse = a->lse;
  p.sched = a->causal ? a->sched : nullptr;
  if (noalloc && scratch_bytes(a) > 0) {
    // Only what the kernel requires to start at zero -- the scheduler words --
    // is cleared, in stream order; nothing is allocated.
    int32_t* words = nullptr;
    rc = noalloc_scratch(dev, &words);
    if (rc != AFA_OK) return rc;
    if (cudaMemsetAsync(words, 0, scratch_bytes(a), static_cast<cudaStream_t>(stream)) != cudaSuccess) {
      cudaGetLastError();
      return AFA_ERR_LAUNCH;
    }
    p.sched = words;
  }
  const float scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt(static_cast<float>(a->head_dim));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = a->status;
  p.timeout_ns = a->timeout_ns != 0 ? a->timeout_ns : 4000000000ull;
  p.test_flags = a->test_flags;

  const int grid = p.n_work < sm_count ? p.n_work : sm_count;
  if (ke->launch[a->causal](p, dim3(static_cast<unsigned>(grid)), static_cast<cudaStream_t>(stream)) !=
      cudaSuccess) {
    cudaGetLastError();
    return AFA_ERR_LAUNCH;
  }
  return AFA_OK;
}

}  // namespace
