// mma_sync_beside_alu.cu -- cycles per warp instruction of what attention over
// the 4-bit cache is made of, on one SM sub-partition: three-input logic, fma and
// mma.sync.m16n8k16, each alone and mixed (whether they overlap), and mma.sync
// with e4m3 operands beside the fp16 form.  One CTA an SM with 4, 8 or 16 warps
// (1, 2 or 4 a sub-partition), independent chains, in-kernel clock64.
//
//   nvcc -gencode arch=compute_100a,code=sm_100a -O3 -std=c++17 -o mma_sync_beside_alu \
//        ampere_flash_attention_from_scratch_b200/microbench/mma_sync_beside_alu.cu && ./mma_sync_beside_alu
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

constexpr int kIters = 1000;
enum : unsigned { kLogic = 1, kFma = 2, kHalf = 4, kE4m3 = 8 };  // 32, 32, 4 and 4 of them an iteration

template <unsigned kWhat>
__global__ void kern(uint32_t* sink, unsigned long long* cyc) {
  uint32_t a[8];
  float f[8], d[4][4];
  for (int i = 0; i < 8; ++i) a[i] = threadIdx.x * 7 + i, f[i] = static_cast<float>(threadIdx.x + i);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) d[i][j] = 0.0f;
  const uint32_t m = threadIdx.x & 0x0f, x = threadIdx.x & 0x3;
  __syncthreads();
  const unsigned long long t0 = clock64();
  for (int it = 0; it < kIters; ++it) {
    // group by group, as the kernel's code comes
    if constexpr ((kWhat & kLogic) != 0) {
#pragma unroll
      for (int i = 0; i < 32; ++i) asm volatile("lop3.b32 %0, %0, %1, %2, 0x6a;" : "+r"(a[i & 7]) : "r"(m), "r"(x));
    }
    if constexpr ((kWhat & kFma) != 0) {
#pragma unroll
      for (int i = 0; i < 32; ++i) asm volatile("fma.rn.f32 %0, %0, %1, %1;" : "+f"(f[i & 7]) : "f"(1.0001f));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr ((kWhat & kHalf) != 0)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %4, %5}, {%4, %5}, {%0, %1, %2, %3};"
            : "+f"(d[r][0]), "+f"(d[r][1]), "+f"(d[r][2]), "+f"(d[r][3])
            : "r"(m), "r"(x));
      if constexpr ((kWhat & kE4m3) != 0)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %4, %5}, {%4, %5}, {%0, %1, %2, %3};"
            : "+f"(d[r][0]), "+f"(d[r][1]), "+f"(d[r][2]), "+f"(d[r][3])
            : "r"(m), "r"(x));
    }
  }
  const unsigned long long t1 = clock64();
  uint32_t s = 0;
  for (int i = 0; i < 8; ++i) s += a[i] + __float_as_uint(f[i]);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) s += __float_as_uint(d[i][j]);
  sink[blockIdx.x * blockDim.x + threadIdx.x] = s;
  if (blockIdx.x == 0 && threadIdx.x == 0) *cyc = t1 - t0;
}

template <unsigned kWhat>
void run(const char* name, int sms, uint32_t* sink, unsigned long long* cyc) {
  for (int warps = 1; warps <= 4; warps *= 2) {
    kern<kWhat><<<sms, warps * 128>>>(sink, cyc);
    kern<kWhat><<<sms, warps * 128>>>(sink, cyc);
    unsigned long long h = 0;
    const cudaError_t e = cudaMemcpy(&h, cyc, sizeof(h), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) {
      printf("%s: %s\n", name, cudaGetErrorString(e));
      return;
    }
    printf("%-30s %d warps a sub-partition: %6.1f cycles an iteration and warp\n", name, warps,
           static_cast<double>(h) / kIters / warps);
  }
}

int main() {
  int sms = 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, 0);
  uint32_t* sink;
  unsigned long long* cyc;
  cudaMalloc(&sink, sizeof(uint32_t) * sms * 512);
  cudaMalloc(&cyc, sizeof(unsigned long long));
  run<kLogic>("32 LOP3", sms, sink, cyc);
  run<kFma>("32 FFMA", sms, sink, cyc);
  run<kHalf>("4 HMMA.16816", sms, sink, cyc);
  run<kE4m3>("4 e4m3 m16n8k32", sms, sink, cyc);
  run<kLogic | kHalf>("32 LOP3 + 4 HMMA", sms, sink, cyc);
  run<kFma | kHalf>("32 FFMA + 4 HMMA", sms, sink, cyc);
  run<kLogic | kFma>("32 LOP3 + 32 FFMA", sms, sink, cyc);
  run<kLogic | kFma | kHalf>("32 LOP3 + 32 FFMA + 4 HMMA", sms, sink, cyc);
  cudaFree(sink);
  cudaFree(cyc);
  return 0;
}
