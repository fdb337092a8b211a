// afa_cache4_wide_kernel.cuh -- attention over the 4-bit cache for many query
// rows of a key/value head (several new tokens, wide groups, chunks of a prompt),
// on tcgen05.
//
// The mathematics is that of afa_cache4_fwd_sm100.cu: codes are multiplied as they
// are, steps and minima are applied to the scores and to the weights.  What
// bounds that kernel beyond 16 rows is the unpacking, which every 16 rows repeat,
// and mma.sync.  Here the codes of 64 tokens are spread once to fp16 in shared
// memory for 128 rows, the products run beside the other work as tcgen05.mma
// (M = 128 rows; padded rows cost nothing that is short), and one thread holds
// one row, so that a token's steps and minima are read once for 32 rows.  What is
// left is the softmax: about 15 instructions a row and token, and the broadcast of
// a token's eight steps and minima to a warp, 8 shared-memory wavefronts (55 % of
// the pipe; packed fp32 instructions therefore change nothing).
// Measured, in calls in a row: [1, 512 new of 131072 tokens, 32/8 heads, 128] bf16 2.85
// ms = 386 TFLOP/s; [16 x 1024..16384, 8 key/value heads x 128 rows, 128] fp16 232 us,
// where the other kernel takes 391.  Two CTAs an SM leave a thread 128 registers: 88
// bytes are spilled at head_dim 128, 8 at 64.
//
//   warps 0-3   softmax: thread = row = TMEM lane; warp 0 also issues the MMAs
//   warps 4-7   loads (cp.async ring), codes -> fp16 tiles, steps and minima
//
// A step of 64 tokens:  S_g = Q_g K_g^T for each group g of 64 channels (fp32, 64
// columns);  P_g = p s'_g (fp16, over S_g's first columns);  O_g += P_g (c' - 8).
// Two CTAs share an SM (256 of 512 columns each): one's products and waits run
// under the other's softmax.  A tile of at most 64 rows stands in the 128 lanes
// twice, and each copy takes half of a step's tokens (its P is zero for the
// others), so that every warp has work; the copies are joined at a piece's end.
//
// K's tile holds c 2^-24 and, for odd channels, c 2^-20 (masked bits, subnormal
// fp16), V's c - 8 and 16 (c - 8); within eight channels the order is 0 4 1 5 2 6 3 7,
// as the masks give it.  Q's tile has the same order with odd channels divided by 16.
#pragma once

#include <cmath>
#include <type_traits>

#include "afa_cache4_fwd_common.cuh"
#include "ops_sites.h"

namespace afa100 {

template <int kD>
struct WideLayout {
  static constexpr int kG = kD / 64;
  static constexpr int kRow = kD / 2 + kD / 16;
  static constexpr int kRows = 128;
  static constexpr int kTok = 64;  // tokens of a step
  static constexpr int kThreads = 256;
  static constexpr int kRing = 3;  // steps of the ring of raw rows
  static constexpr uint32_t kSideBytes = kTok * kRow;
  static constexpr uint32_t kRawBytes = 2 * kSideBytes;
  static constexpr uint32_t kQAtom = kRows * 128u, kKAtom = kTok * 128u;  // one group's tile
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffK = kOffQ + kG * kQAtom;
  static constexpr uint32_t kOffV = kOffK + kG * kKAtom;
  static constexpr uint32_t kOffRaw = kOffV + kG * kKAtom;
  static constexpr uint32_t kOffKs = kOffRaw + kRing * kRawBytes;      // [2][kTok][s of kG groups, m of kG groups]
  static constexpr uint32_t kOffVs = kOffKs + 2u * kTok * kG * 8u;     // [kTok], the same
  static constexpr uint32_t kOffMl = kOffVs + kTok * kG * 8u;  // [64]: reference and sum of the second copies of rows
  static constexpr uint32_t kOffSeen = kOffMl + 64u * 8u;  // [4]: a producer warp's largest step of the values
  static constexpr uint32_t kOffBar = kOffSeen + 16u;
  static constexpr int kBarQ = 0, kBarK = 1, kBarV = 2, kBarS = 3, kBarP = 4, kBarPv = 5, kBarDrain = 6, kBars = 7;
  static constexpr uint32_t kOffTmem = kOffBar + kBars * 8u;
  static constexpr uint32_t kOffAbort = kOffTmem + 4u;
  static constexpr uint32_t kSmem = kOffAbort + 4u + 1024u;  // slack for the tiles' alignment
  static constexpr uint32_t kTmemCols = 128u * kG;
  static constexpr uint32_t kColO = 64u * kG;
  static constexpr int kShare = kRows * (kD + 2);  // floats of a CTA's share of an item
};

// A bounded wait: false, with the site reported and every other role's waits cut
// short, when the phase has not completed by the deadline.
struct WideSync {
  volatile int* abort;
  int32_t* status;
  uint64_t timeout_ns;
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int site) const {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t deadline = globaltimer_ns() + timeout_ns;
    for (;;) {
      if (mbar_try_wait_suspend(bar, parity, 20000u)) return true;
      if (*abort != 0) return false;
      if (globaltimer_ns() > deadline) {
        report(status, AFA_DEV_TIMEOUT_BASE + site);
        *abort = 1;
        return false;
      }
    }
  }
};

// The last token (exclusive) any row of the tile sees.
__device__ __forceinline__ int wide_reach(const FwdParams4& p, const Item& it, int fresh) {
  if (!p.causal) return it.tokens;
  const int tile = it.which % p.row_tiles;
  const int last = min(p.rows, (tile + 1) * 128) - 1;
  return min(it.tokens, max(0, it.tokens - fresh + last / p.group + 1));
}

__device__ __forceinline__ int fresh_of(const FwdParams4& p, int b) {
  return p.c.new_lens != nullptr ? p.c.new_lens[b] : p.seq_len;
}

// A barrier of a role's four warps; whether `ok` holds for all of them.
template <int kBarrier>
__device__ __forceinline__ bool agree(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(all)
      : "r"(ok ? 1u : 0u), "n"(kBarrier)
      : "memory");
  return all != 0u;
}

// 32 columns from each of two places, with one wait.
__device__ __forceinline__ void tmem_ld32x2_sync(uint32_t a0, uint32_t a1, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : AFA_R8(r, 0), AFA_R8(r, 8), AFA_R8(r, 16), AFA_R8(r, 24), AFA_R8(r, 32), AFA_R8(r, 40), AFA_R8(r, 48),
        AFA_R8(r, 56)
      : "r"(a0), "r"(a1)
      : "memory");
}

// Eight columns of O and the minima's part as eight channels: the columns are
// channels 0 4 1 5 2 6 3 7, odd ones 16 times.
__device__ __forceinline__ void columns(float (&f)[8], const uint32_t (&x)[8], float m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float odd = i & 1 ? 0.0625f : 1.0f;
    f[i] = fmaf(__uint_as_float(x[2 * i]), odd, m);
    f[i + 4] = fmaf(__uint_as_float(x[2 * i + 1]), odd, m);
  }
}

// 16-byte chunk `c` of row `row` of a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int row, int c) {
  return tile + static_cast<uint32_t>(row) * 128u + (static_cast<uint32_t>(c ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t m, uint32_t x) {  // (w & m) | x
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(m), "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// ---------------------------------------------------------------------------
// Role: loads and tiles (warps 4-7)
// ---------------------------------------------------------------------------
template <int kD, bool kBF16>
__device__ __forceinline__ void wide_produce(const FwdParams4& p, Walk w, char* smem, uint32_t sbase, const WideSync& sy) {
  using L = WideLayout<kD>;
  const int tid = static_cast<int>(threadIdx.x) - 128, lane = tid & 31;
  auto bar = [&](int i) { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); };

  // Loads run ahead through the pieces.  Lane i holds the page of the i-th block
  // of 16 tokens from the last look-up on, eight steps' worth.
  Walk ahead = w;
  bool more = true;
  int end = 0, page = 0, block = 0;
  const char* side = nullptr;
  auto look_up = [&]() {
    block = 0;
    const int at = ahead.tok + lane * 16;
    if (at < end) page = p.c.page_table[ahead.it.b * p.c.table_stride + (at >> p.page_shift)];
  };
  auto settle = [&]() {
    for (;;) {
      end = min(ahead.tok_end, wide_reach(p, ahead.it, fresh_of(p, ahead.it.b)));
      if (ahead.tok < end) break;
      if (!(more = ahead.next(p, 0))) return;
    }
    side = static_cast<const char*>(p.c.cache) +
           static_cast<int64_t>(ahead.it.which / p.row_tiles) * 2 * p.c.page_size * L::kRow;
    look_up();
  };
  auto load = [&](uint32_t stage) {
    if (more) {
      constexpr int kChunks = L::kTok * L::kRow / 16;  // of a side
      constexpr int kPerBlock = L::kRow;               // 16 tokens
#pragma unroll
      for (int i = 0; i < (2 * kChunks + 127) / 128; ++i) {
        const int x = tid + i * 128;
        const int kv = x >= kChunks, o = x - kv * kChunks;
        const int blk = o / kPerBlock;  // 0..3, or 4 behind the last chunk
        int pg = __shfl_sync(0xffffffffu, page, (block + blk) & 31);
        if (x < 2 * kChunks && ahead.tok + blk * 16 < end) {
          uint32_t bytes = 16;
          if (static_cast<uint32_t>(pg) >= static_cast<uint32_t>(p.c.n_pages)) {
            report(p.c.status, AFA_DEV_BAD_PAGE);  // zeros in place of a page that does not exist
            pg = 0;
            bytes = 0;
          }
          const uint32_t at = (ahead.tok + blk * 16) & (p.c.page_size - 1);
          const char* src = far(far(side, pg, p.page_stride), at + (kv ? p.c.page_size : 0), L::kRow);
          cp_async16(sbase + L::kOffRaw + stage * L::kRawBytes + static_cast<uint32_t>(x) * 16u,
                     src + (o - blk * kPerBlock) * 16, bytes);
        }
      }
      ahead.tok += L::kTok;
      block += 4;
      if (ahead.tok >= end)
        settle();
      else if (block == 32)
        look_up();
    }
    cp_async_commit();
  };
  settle();
#pragma unroll 1
  for (int s = 0; s < L::kRing - 1; ++s) load(s);

  // A thread spreads kD / 2 channels of one token: a group, or half of one.
  const int token = tid & 63, part = tid >> 6;
  auto spread = [&](bool values, uint32_t stage, uint32_t tile, char* scales, int tok0, int stop) {
    const char* row = smem + L::kOffRaw + stage * L::kRawBytes + (values ? L::kSideBytes : 0u) + token * L::kRow;
    uint32_t code[kD / 16];
    if constexpr (kD == 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + part * 32 + i * 8);
        code[2 * i] = v.x;
        code[2 * i + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) code[i] = *reinterpret_cast<const uint32_t*>(row + part * 16 + i * 4);
    }
    const int g = kD == 128 ? part : 0;
    const uint32_t dst = tile + g * L::kKAtom;
    const int c0 = kD == 128 ? 0 : part * 4;
#pragma unroll
    for (int i = 0; i < kD / 16; ++i) {
      const uint32_t u = code[i], u8 = u >> 8;
      uint32_t v[4];
      if (values) {
        v[0] = hsub2(masked(u, 0x000f000fu, 0x64006400u), 0x64086408u);
        v[1] = hsub2(masked(u, 0x00f000f0u, 0x64006400u), 0x64806480u);
        v[2] = hsub2(masked(u8, 0x000f000fu, 0x64006400u), 0x64086408u);
        v[3] = hsub2(masked(u8, 0x00f000f0u, 0x64006400u), 0x64806480u);
      } else {
        v[0] = u & 0x000f000fu;
        v[1] = u & 0x00f000f0u;
        v[2] = u8 & 0x000f000fu;
        v[3] = u8 & 0x00f000f0u;
      }
      st_shared_v4(swizzled(dst, token, c0 + i), v[0], v[1], v[2], v[3]);
    }
    if (kD == 128 || part == 0) {
      float2 sm = unpack2<kBF16>(*reinterpret_cast<const uint32_t*>(row + kD / 2 + g * 4));
      if (tok0 + token >= stop) sm = make_float2(0.0f, 0.0f);  // not a token, or one no row sees: not loaded
      float* out = reinterpret_cast<float*>(scales) + token * 2 * L::kG;
      out[g] = sm.x;
      out[L::kG + g] = values ? fmaf(8.0f, sm.x, sm.y) : sm.y;
      if (values) {
        float big = fabsf(sm.x);
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
        if (lane == 0) reinterpret_cast<float*>(smem + L::kOffSeen)[tid >> 5] = big;
      }
    }
  };
  auto publish = [&](int b) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };

  uint32_t j = 0, stage = 0;  // step of the CTA, its ring slot
  bool ok = (p.test_flags & AFA_TEST_PRODUCER_IDLE) == 0u;
  int stop = min(w.tok_end, wide_reach(p, w.it, fresh_of(p, w.it.b)));
  bool left = true;
  for (;; ++j, w.tok += L::kTok) {
    while (left && w.tok >= stop) {
      left = w.next(p, 0);
      if (left) stop = min(w.tok_end, wide_reach(p, w.it, fresh_of(p, w.it.b)));
    }
    if (!left) break;
    cp_async_wait<L::kRing - 2>();
    // Every thread's part has landed, and the slot loaded next has been read.  A wait that ran out for one warp is
    // everyone's here: the four leave at the same barrier.
    ok = agree<1>(ok);
    if (!ok) break;
    load(stage == 0 ? L::kRing - 1 : stage - 1);
    if (j > 0) ok = __all_sync(0xffffffffu, sy.wait(bar(L::kBarS), (j - 1) & 1, kSiteWideS));
    if (ok) {
      spread(false, stage, sbase + L::kOffK, smem + L::kOffKs + (j & 1) * (L::kTok * L::kG * 8u), w.tok, stop);
      publish(L::kBarK);
      if (j > 0) ok = __all_sync(0xffffffffu, sy.wait(bar(L::kBarPv), (j - 1) & 1, kSiteWidePv));
    }
    if (ok) {
      spread(true, stage, sbase + L::kOffV, smem + L::kOffVs, w.tok, stop);
      publish(L::kBarV);
    }
    stage = stage + 1 == L::kRing ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------
// MMA issue (warp 0 between its shares of the softmax; converged, lane 0 issues)
// ---------------------------------------------------------------------------
template <int kD>
struct WideMma {
  using L = WideLayout<kD>;
  uint32_t sbase, tmem, leader;
  __device__ __forceinline__ uint32_t bar(int i) const { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); }
  // S_g = Q_g K_g^T
  __device__ __forceinline__ void scores() const {
    constexpr uint32_t kIdesc = idesc_f16_f32(128, L::kTok, false, false);
#pragma unroll
    for (int g = 0; g < L::kG; ++g) {
      const uint32_t a = sdesc_lo(sbase + L::kOffQ + g * L::kQAtom, 16), b = sdesc_lo(sbase + L::kOffK + g * L::kKAtom, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_f16_ss(tmem + g * 64u, a + k * 2u, b + k * 2u, kIdesc, k > 0 ? 1u : 0u, leader);
    }
    umma_commit(bar(L::kBarS), leader);
  }
  // O_g += P_g V_g
  __device__ __forceinline__ void values(bool first) const {
    constexpr uint32_t kIdesc = idesc_f16_f32(128, 64, false, true);
#pragma unroll
    for (int g = 0; g < L::kG; ++g) {
      const uint32_t b = sdesc_lo(sbase + L::kOffV + g * L::kKAtom, L::kKAtom);
#pragma unroll
      for (int k = 0; k < 4; ++k)  // 16 tokens a step: 8 columns of P, 16 rows of V
        umma_f16_ts(tmem + L::kColO + g * 64u, tmem + g * 64u + k * 8u, b + k * (16u * 128u >> 4), kIdesc,
                    !first || k > 0 ? 1u : 0u, leader);
    }
    umma_commit(bar(L::kBarPv), leader);
  }
  // Nothing of this CTA's may still run when its tensor memory goes.
  __device__ __forceinline__ void drain(const FwdParams4& p) const {
    umma_commit(bar(L::kBarDrain), leader);
    const uint64_t deadline = globaltimer_ns() + p.timeout_ns;
    while (!mbar_try_wait_suspend(bar(L::kBarDrain), 0, 20000u)) {
      if (globaltimer_ns() > deadline) {
        report(p.c.status, AFA_DEV_TIMEOUT_BASE + kSiteWideDrain);
        break;
      }
    }
  }
};

// ---------------------------------------------------------------------------
// Role: softmax (warps 0-3)
// ---------------------------------------------------------------------------
template <int kD, bool kBF16>
__device__ __forceinline__ void wide_softmax(const FwdParams4& p, Walk w, char* smem, uint32_t sbase, uint32_t tmem,
                                             const WideSync& sy) {
  using L = WideLayout<kD>;
  constexpr int kG = L::kG;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31;
  auto bar = [&](int i) { return sbase + L::kOffBar + 8u * static_cast<uint32_t>(i); };
  const uint32_t mine = tmem + (static_cast<uint32_t>(tid & ~31) << 16);  // this warp's lanes
  const bool issuer = tid < 32;
  const WideMma<kD> mma{sbase, tmem, tid == 0 ? 1u : 0u};
  auto wait = [&](int b, uint32_t parity, int site) {
    const bool done = __all_sync(0xffffffffu, sy.wait(bar(b), parity, site));
    tc_fence_after_sync();
    return done;
  };
  uint32_t j = 0, piece = 0;
  bool ok = true;
  do {
    const Item it = w.it;
    if (w.unit_end <= p.item_units) continue;  // only the cost of an item that another CTA works on
    const int head = it.which / p.row_tiles, tile = it.which - head * p.row_tiles;
    const bool starts = it.unit <= p.item_units, whole = starts && w.unit_end == it.units;
    const int fresh = fresh_of(p, it.b);
    const int stop = min(w.tok_end, wide_reach(p, it, fresh));
    const int tile_rows = min(128, p.rows - tile * 128);
    const bool twice = tile_rows <= 64;
    const int copy = twice ? tid >> 6 : 0;
    const int row = twice ? tid & 63 : tid, r = tile * 128 + row;
    const bool valid = row < tile_rows;
    const bool busy = __any_sync(0xffffffffu, valid);
    const int n = r / p.group, h = head * p.group + (r - n * p.group);

    // --- this row of Q -----------------------------------------------------------------------------------
    float a_of = 0.0f, qs[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) qs[g] = 0.0f;
    if (w.tok < stop) {
      const char* src = p.q + it.b * p.q_s[0] + n * p.q_s[1] + h * p.q_s[2];
      float big = 0.0f;
      if (valid) {
#pragma unroll 4
        for (int c = 0; c < kD / 8; ++c) {
          const uint4 v4 = *reinterpret_cast<const uint4*>(src + c * 16);
          const uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<kBF16>(v[i]);
            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
            sum += f.x + f.y;
          }
          if (kG == 1 || c < 8)
            qs[0] += sum;
          else
            qs[kG - 1] += sum;
        }
      }
      // 2^e with e = 13 - floor(log2(big)), from the exponent field; within fp32's normal range
      int e = big > 0.0f ? 13 + 127 - static_cast<int>(__float_as_uint(big) >> 23) : 0;
      e = e > 90 ? 90 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      a_of = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * 16777216.0f * p.scale_log2;
#pragma unroll
      for (int g = 0; g < kG; ++g) qs[g] *= p.scale_log2;
#pragma unroll 4
      for (int c = 0; c < kD / 8; ++c) {
        uint4 v4 = make_uint4(0, 0, 0, 0);
        if (valid) v4 = *reinterpret_cast<const uint4*>(src + c * 16);
        const float2 x0 = unpack2<kBF16>(v4.x), x1 = unpack2<kBF16>(v4.y), x2 = unpack2<kBF16>(v4.z), x3 = unpack2<kBF16>(v4.w);
        const float odd = up * 0.0625f;
        st_shared_v4(swizzled(sbase + L::kOffQ + (c / 8) * L::kQAtom, tid, c % 8), pack2<false>(x0.x * up, x2.x * up),
                     pack2<false>(x0.y * odd, x2.y * odd), pack2<false>(x1.x * up, x3.x * up),
                     pack2<false>(x1.y * odd, x3.y * odd));
      }
      fence_proxy_async_shared();
      tc_fence_before_sync();  // the epilogue's reads of O come before the MMAs that this lets go
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::kBarQ));
      if (issuer) {
        ok = wait(L::kBarQ, piece & 1, kSiteWideQ) && wait(L::kBarK, j & 1, kSiteWideKFull);
        if (ok) mma.scores();
      }
      ++piece;
    }

    // --- the walk over the tokens ------------------------------------------------------------------------
    // As in the other kernel: p = 2^(score + off).  The references are whole numbers here, so that a half of P already
    // written may be rescaled in place: exactly, but for products that leave fp16's normal range by it.
    float reference = -INFINITY, off = 0.0f, limit_s = -INFINITY, l = 0.0f, step_max = 0.0f, acc_m[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) acc_m[g] = 0.0f;
    const int limit = p.causal ? min(it.tokens, max(0, it.tokens - fresh + n + 1)) : it.tokens;
    bool first = true;
    for (; ok && w.tok < stop; w.tok += L::kTok, ++j) {
      // V's tile is filled after K's by the same threads, so its barrier stands for the steps and minima of both.
      // (K's own may be a phase ahead by now: it is refilled as soon as S is done.)
      ok = wait(L::kBarV, j & 1, kSiteWideVFull) && wait(L::kBarS, j & 1, kSiteWideS);
      if (!ok) break;
      if (busy) {
        const float* ks = reinterpret_cast<const float*>(smem + L::kOffKs + (j & 1) * (L::kTok * kG * 8u));
        const float* vs = reinterpret_cast<const float*>(smem + L::kOffVs);
        const float4 big = *reinterpret_cast<const float4*>(smem + L::kOffSeen);
        const float seen = kG == 2 ? fmaxf(fmaxf(big.x, big.y), fmaxf(big.z, big.w)) : fmaxf(big.x, big.y);
        bool grow = seen > step_max;
        // 32 tokens
        auto half = [&](auto masked_tag, const int c) {
          constexpr bool kMasked = decltype(masked_tag)::value;
          const int tok0 = w.tok + 32 * c;
          float v[32];
          float top = -INFINITY;
          {
            uint32_t s[32 * kG];
            if constexpr (kG == 2)
              tmem_ld32x2_sync(mine + c * 32u, mine + 64u + c * 32u, s);
            else
              tmem_ld32_sync(mine + c * 32u, s);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float* sm = ks + (32 * c + i) * 2 * kG;
              if constexpr (kG == 2) {
                const float4 f = *reinterpret_cast<const float4*>(sm);
                const float dot = fmaf(f.y, __uint_as_float(s[32 + i]), f.x * __uint_as_float(s[i]));
                v[i] = fmaf(a_of, dot, fmaf(f.w, qs[1], fmaf(f.z, qs[0], off)));
              } else {
                const float2 f = *reinterpret_cast<const float2*>(sm);
                v[i] = fmaf(a_of, f.x * __uint_as_float(s[i]), fmaf(f.y, qs[0], off));
              }
            }
          }
          if constexpr (kMasked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (tok0 + i >= limit) v[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) top = fmax3(top, v[i], v[i + 1]);

          // (as in the other kernel; a lane finds the size of one token, for all rows)
          if (__any_sync(0xffffffffu, grow || top > limit_s)) {
            const float* mine_vs = vs + (32 * c + lane) * 2 * kG;
            float size = kLeastSize;
#pragma unroll
            for (int g = 0; g < kG; ++g) size = size_of(size, mine_vs[g], mine_vs[kG + g]);
            float most = fmaxf(size, seen);
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
            if (most > step_max) step_max = power_above(most);
            const float limit = kRescale + kHeadroom - log2_of_power(step_max);
            size = lg2_approx(size);
            most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) most = fmaxf(most, v[i] + __shfl_sync(0xffffffffu, size, i));
            const bool none = reference == -INFINITY;
            const bool passes = most > (none ? -INFINITY : kRescale + kHeadroom);
            if (!none || passes) limit_s = limit;
            if (__any_sync(0xffffffffu, passes)) {
              const float now = passes ? ceilf(most - off) : reference;
              const float to = passes ? kHeadroom - now : off;
              const float move = to - off;
              // in two parts, since steps that grow by more than 2^126 leave weights that still count
              const float part = truncf(0.5f * move);
              const float by0 = none ? 1.0f : ex2_approx(part), by1 = none ? 1.0f : ex2_approx(move - part);
              reference = now;
              off = to;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += move;
              l = l * by0 * by1;
#pragma unroll
              for (int g = 0; g < kG; ++g) acc_m[g] = acc_m[g] * by0 * by1;
              if (__any_sync(0xffffffffu, by1 != 1.0f)) {
                // (rolled loops: a step's code has to stay in the instruction cache, 2851 us for the chunk above, else 2938)
                if (c == 1 && !twice) {  // this step's first half of P
                  tmem_wait_st();
#pragma unroll 1
                  for (int g = 0; g < kG; ++g) {
                    uint32_t x[16];
                    tmem_ld16_sync(mine + g * 64u, x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {  // (a factor may be below fp16's range where the product is not)
                      const float2 f = unpack2<false>(x[i]);
                      x[i] = pack2<false>(f.x * by0 * by1, f.y * by0 * by1);
                    }
                    tmem_st16(mine + g * 64u, x);
                  }
                }
                if (!first) {
#pragma unroll 1
                  for (int o = 0; o < kD; o += 16) {
                    uint32_t x[16];
                    tmem_ld16_sync(mine + L::kColO + o, x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * by0 * by1);
                    tmem_st16(mine + L::kColO + o, x);
                  }
                }
                tmem_wait_st();
              }
            }
            grow = false;
          }

          uint32_t pp[kG][16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = ex2_approx(v[i]), p1 = ex2_approx(v[i + 1]);
            l += p0 + p1;
            const float* sm = vs + (32 * c + i) * 2 * kG;
            float a[2 * kG], b[2 * kG];
            if constexpr (kG == 2) {
              const float4 f0 = *reinterpret_cast<const float4*>(sm), f1 = *reinterpret_cast<const float4*>(sm + 4);
              a[0] = f0.x, a[1] = f0.y, a[2] = f0.z, a[3] = f0.w;
              b[0] = f1.x, b[1] = f1.y, b[2] = f1.z, b[3] = f1.w;
            } else {
              const float4 f = *reinterpret_cast<const float4*>(sm);
              a[0] = f.x, a[1] = f.y, b[0] = f.z, b[1] = f.w;
            }
#pragma unroll
            for (int g = 0; g < kG; ++g) {
              float x0 = p0 * a[g], x1 = p1 * b[g], m0 = a[kG + g], m1 = b[kG + g];
              if constexpr (kMasked) {  // a masked token's s' and m' may be NaN
                if (tok0 + i >= limit) x0 = m0 = 0.0f;
                if (tok0 + i + 1 >= limit) x1 = m1 = 0.0f;
              }
              pp[g][i / 2] = pack2<false>(x0, x1);
              acc_m[g] = fmaf(p1, m1, fmaf(p0, m0, acc_m[g]));
            }
          }
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            tmem_st16(mine + g * 64u + c * 16u, pp[g]);
            if (twice) {  // the other copy's tokens
#pragma unroll
              for (int i = 0; i < 16; ++i) pp[g][i] = 0u;
              tmem_st16(mine + g * 64u + (c ^ 1) * 16u, pp[g]);
            }
          }
        };
        const int c_begin = twice ? copy : 0, c_end = twice ? copy + 1 : 2;
        const bool some_masked = __any_sync(0xffffffffu, w.tok + 32 * c_end > limit);
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          if (some_masked)
            half(std::true_type{}, c);
          else
            half(std::false_type{}, c);
        }
        tmem_wait_st();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::kBarP));
      if (issuer) {
        ok = wait(L::kBarP, j & 1, kSiteWideP);
        if (ok) mma.values(first);
        if (ok && w.tok + L::kTok < stop) {
          ok = wait(L::kBarK, (j + 1) & 1, kSiteWideKFull);
          if (ok) mma.scores();
        }
      }
      first = false;
    }

    // --- O -------------------------------------------------------------------------------------------------
    if (ok && !first) ok = wait(L::kBarPv, (j - 1) & 1, kSiteWidePv);
    // A wait that ran out for one warp is everyone's here: the four leave at the same barrier.
    ok = agree<2>(ok);
    if (!ok) break;
    float ref = reference == -INFINITY ? -INFINITY : -off;
    // Q's tile is free now and holds the second copies' rows of O: 16-byte piece c of row r at c ^ (r mod 8).
    auto second = [&](int c) {
      return reinterpret_cast<float4*>(smem + L::kOffQ + row * (kD * 4) + ((c & ~7) | ((c ^ row) & 7)) * 16);
    };
    float2* ml = reinterpret_cast<float2*>(smem + L::kOffMl);
    float by = 1.0f, by_second = 0.0f;
    if (twice) {
      if (copy == 1 && busy) {
        if (valid) ml[row] = make_float2(ref, l);
#pragma unroll 2
        for (int c = 0; c < kD / 8; ++c) {
          uint32_t x[8];
          if (!first) {
            tmem_ld8_sync(mine + L::kColO + c * 8u, x);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0u;
          }
          const float m = kG == 1 || c < 8 ? acc_m[0] : acc_m[kG - 1];
          float f[8];
          columns(f, x, m);
          if (valid) {
            *second(2 * c) = make_float4(f[0], f[1], f[2], f[3]);
            *second(2 * c + 1) = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
      }
      agree<2>(true);
      if (copy == 0 && valid) {
        const float2 s = ml[row];
        const float both = fmaxf(ref, s.x);
        by = both == -INFINITY ? 1.0f : ex2_approx(0.5f * (ref - both));  // squares of these, as above
        by_second = both == -INFINITY ? 1.0f : ex2_approx(0.5f * (s.x - both));
        l = fmaf(by_second, by_second * s.y, l * by * by);
        ref = both;
      }
    }
    if (busy && copy == 0) {
      const bool some = valid && n < fresh && !(l == 0.0f);
      const float inv = some ? 1.0f / l : 0.0f;
      float* share = p.ws + (static_cast<int64_t>(blockIdx.x) * 2 + (starts ? 1 : 0)) * L::kShare;
      char* dst = p.o + it.b * p.o_s[0] + n * p.o_s[1] + h * p.o_s[2];
#pragma unroll 2
      for (int c = 0; c < kD / 8; ++c) {
        uint32_t x[8];
        float f[8];
        if (!first) {
          tmem_ld8_sync(mine + L::kColO + c * 8u, x);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0u;
        }
        const float m = kG == 1 || c < 8 ? acc_m[0] : acc_m[kG - 1];
        columns(f, x, m);
        if (valid) {
          if (twice) {
            const float4 s0 = *second(2 * c), s1 = *second(2 * c + 1);
            const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = fmaf(by_second, by_second * s[i], f[i] * by * by);
          }
          if (whole) {
            uint4 out = make_uint4(0, 0, 0, 0);
            if (some)
              out = make_uint4(pack2<kBF16>(f[0] * inv, f[1] * inv), pack2<kBF16>(f[2] * inv, f[3] * inv),
                               pack2<kBF16>(f[4] * inv, f[5] * inv), pack2<kBF16>(f[6] * inv, f[7] * inv));
            *reinterpret_cast<uint4*>(dst + c * 16) = out;
          } else {
            float* at = share + row * kD + c * 8;
            *reinterpret_cast<float4*>(at) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(at + 4) = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
      }
      if (valid && whole && p.lse != nullptr)
        p.lse[(static_cast<int64_t>(it.b) * p.n_heads + h) * p.seq_len + n] =
            some ? (ref + log2f(l)) * 0.69314718055994531f : -INFINITY;
      if (valid && !whole) {
        share[L::kRows * kD + row * 2] = ref;
        share[L::kRows * kD + row * 2 + 1] = l;
      }
    }
    if (twice) agree<2>(true);  // the second copies have been read: Q's tile may be filled
  } while (ok && w.next(p, 0));
  if (issuer) mma.drain(p);
}

template <int kD, bool kBF16>
__global__ void __launch_bounds__(WideLayout<kD>::kThreads, 2) cache4_wide_kernel(const FwdParams4 p) {
  using L = WideLayout<kD>;
  extern __shared__ char smem_raw[];
  char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // the tiles' swizzle atoms are 1024 bytes
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kOffAbort);

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
    w.open(p, 0);
  }
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < L::kBars; ++i)
        mbar_init(sbase + L::kOffBar + 8u * i, i == L::kBarQ || i == L::kBarK || i == L::kBarV || i == L::kBarP ? 4u : 1u);
      *abort = 0;
      fence_mbarrier_init();
    }
    __syncwarp();
    tmem_alloc(sbase + L::kOffTmem, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::kOffTmem);
  const WideSync sy{abort, p.c.status, p.timeout_ns};
  if (warp < 4)
    wide_softmax<kD, kBF16>(p, w, smem, sbase, tmem, sy);
  else
    wide_produce<kD, kBF16>(p, w, smem, sbase, sy);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

}  // namespace afa100
