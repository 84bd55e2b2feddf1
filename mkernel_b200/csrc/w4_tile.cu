// The product with 4-bit weights for more than a few tokens, on the 5th-generation tensor cores.
//
// A CTA computes 128 rows of the matrix (two strips) for up to 128 tokens, D = W A^T with the weights as
// the 128-row operand.  That operand never exists in shared memory: the lanes that decode the codes
// write whole numbers (code - zero, times a power of two) into tensor memory, in the 16x256b form
// whose lanes are the layout's lanes, and the MMA takes its A operand from there.  So shared memory
// carries only the packed codes and the tokens.
//
// One step is one group of columns.  The sums of a group are exact products added in fp32 by the tensor
// core; the threads that own the accumulator's lanes (a lane is a row of the matrix) read it, multiply
// it by the row's scale in fp32 and add it to registers.  No weight is rounded to be multiplied.
//
// A step is little work and a long way: decoding, a barrier, the tensor core, a barrier, reading,
// rescaling are about 900 cycles one after another for eight warps that share it, when 310 would keep
// memory busy.  Hence 16 warps and several steps under way: up to 64 tokens, two sets of eight warps
// take turns at the steps (each with sums of its own, added at the end); for more, whose sums would not
// fit its registers, all 16 share every step.  Decoders run ahead of the rescaling by the operand
// buffers that tensor memory has room for beside the accumulators.
//
// Warps 0..15 decode and rescale (quadrant warp % 4 of the lanes; of a step, the other bits decide which part
// of the decoding and which of the tokens), warps 16 and 17 issue the MMAs, a thread of warp 18 (warps 18
// and 19 where rows are not aligned) copies a ring of stages (a block of 128 columns: codes of two strips,
// tokens in the 128-byte swizzle).
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/mkernel_b200.h"
#include "w4_product.cuh"

namespace mkb {

constexpr int kTileRows = 2 * kW4Strip;
constexpr int kTileCompute = 16;                   // warps
constexpr int kTileIssue = 2;
constexpr int kTileLoaders = 2;
constexpr int kTileThreads = (kTileCompute + kTileIssue + kTileLoaders) * 32;
constexpr int kTileControl = 1024;                 // bytes before the ring
constexpr int kTilePitch = kTileRows + 4;          // floats of a token's sums

__host__ __device__ constexpr int w4_tile_stages(int tokens) { return tokens <= 64 ? 8 : tokens <= 96 ? 6 : 5; }

// Accumulators (of `tokens` columns) and operand buffers (of at most 64) that share tensor memory's 512.
__host__ __device__ constexpr int w4_tile_sums(int tokens) { return tokens == 128 ? 2 : tokens == 96 ? 3 : 4; }
__host__ __device__ constexpr int w4_tile_operands(int tokens) { return tokens == 96 ? 3 : 4; }

struct TileWait {
  volatile uint32_t* abort;   // shared: some wait of this CTA has run out
  uint64_t limit_ns;
};

// False when the wait has run out, here or elsewhere in the CTA.
__device__ __noinline__ bool w4_slow_wait(const TileWait& c, uint32_t bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((it & 127u) == 0u) {
      if (*c.abort != 0u) return false;
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > c.limit_ns) {
        *c.abort = 1u;
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool w4_wait(const TileWait& c, uint32_t bar, uint32_t parity) {
  return ptx::mbar_try_wait(bar, parity) || w4_slow_wait(c, bar, parity);
}
// The same for a whole warp that goes on, or gives up, together.
__device__ __forceinline__ bool w4_wait_warp(const TileWait& c, uint32_t bar, uint32_t parity) {
  return __all_sync(~0u, w4_wait(c, bar, parity));
}

template <typename T, int TOKENS, int GROUP>
__global__ void __launch_bounds__(kTileThreads, 1) w4_tile_kernel(const __grid_constant__ W4Params p,
                                                                 const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kTokens = TOKENS;
  constexpr int kSets = TOKENS <= 64 ? 2 : 1;       // of warps, that take turns at the steps
  constexpr int kSubs = kSets == 2 ? 2 : 4;         // warps of a set on a quadrant
  constexpr int TH = TOKENS / kSubs;                // sums of a thread
  constexpr int kStages = w4_tile_stages(kTokens);
  constexpr int kSteps = kW4Block / GROUP;          // of a block
  constexpr int kSums = w4_tile_sums(kTokens), kOperands = w4_tile_operands(kTokens);
  constexpr uint32_t kUsed = kSums * kTokens + kOperands * (GROUP / 2), kCols = kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512, "tensor memory has 512 columns");
  constexpr int kXHalf = kTokens * 128;             // bytes of 64 columns of the tokens

  const W4Form& f = p.form;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw);
  // control words: full[8] empty[8] a_full[4] d_full[4] d_free[4] | tensor memory address, abort flag
  auto full = [&](int s) { return base + 8u * s; };
  auto empty = [&](int s) { return base + 64u + 8u * s; };
  auto a_full = [&](int i) { return base + 128u + 8u * i; };
  auto d_full = [&](int i) { return base + 160u + 8u * i; };
  auto d_free = [&](int i) { return base + 192u + 8u * i; };
  volatile uint32_t* const s_tmem = reinterpret_cast<volatile uint32_t*>(base_ptr + 224);
  volatile uint32_t* const s_abort = s_tmem + 1;
  const uint32_t ring = base + kTileControl;
  uint8_t* const ring_ptr = base_ptr + kTileControl;

  const int rank = blockIdx.x % p.split;
  const int unit = blockIdx.x / p.split;
  const int row_tile = unit / p.token_tiles, token0 = unit % p.token_tiles * kTokens;
  const int blocks = (f.blocks - rank + p.split - 1) / p.split;     // rank, rank + split, ...
  const int strip0 = 2 * row_tile;
  const bool two = strip0 + 1 < f.strips;

  if (warp == kTileCompute) {
    ptx::tmem_alloc(base + 224, kCols);
    ptx::tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(full(s), p.vec ? 1 : kTileLoaders * 32);
      // the warps that decode from it, and the issuing warps that multiply by it
      ptx::mbar_init(empty(s), GROUP == 128 ? kTileCompute / kSets + 1 : kTileCompute + kTileIssue);
    }
    for (int i = 0; i < kOperands; ++i) ptx::mbar_init(a_full(i), kTileCompute / kSets);
    for (int i = 0; i < kSums; ++i) {
      ptx::mbar_init(d_full(i), 1);
      ptx::mbar_init(d_free(i), kTileCompute / kSets);
    }
    *s_abort = 0u;
    ptx::fence_mbar_init();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const uint32_t tmem_a = tmem + kSums * kTokens;
  const TileWait wc{s_abort, p.wait_limit_ns};

  const size_t strip_bytes = (size_t)f.blocks * f.chunk_bytes;
  const uint8_t* const data = p.data + (size_t)strip0 * strip_bytes + (size_t)rank * f.chunk_bytes;
  if (warp >= kTileCompute + kTileIssue) {
    // what is read first may be asked into L2 before the kernel ahead has finished
    const int lt = threadIdx.x - (kTileCompute + kTileIssue) * 32;
    for (int b = 0; b < kStages && b < blocks; ++b)
      for (int o = lt * 128; o < f.chunk_bytes; o += kTileLoaders * 32 * 128)
        for (int i = 0; i <= (int)two; ++i)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(data + i * strip_bytes + (size_t)b * p.split * f.chunk_bytes + o));
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  float acc[TH];
  if (warp < kTileCompute) {
    // ---------------- decode, rescale ----------------
    const int set = kSets == 2 ? warp >> 3 : 0, quad = warp & 3, g = lane >> 2;
    const int sub = kSets == 2 ? (warp >> 2) & 1 : warp >> 2;
    const int strip = quad >> 1, tile0 = (quad & 1) * 2;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const int codes_at = kTokens * 256 + strip * f.chunk_bytes;
    // scale of the accumulator's lane, in 16-bit units behind the codes
    const int row = (quad & 1) * 32 + lane;
    const int scale_at = codes_at + kW4CodeBytes + ((row & 7) * 8 + (row >> 4) * 2 + ((row >> 3) & 1)) * 2;
    const int offset_at = codes_at + kW4CodeBytes + kSteps * 128 + g * 16;
#pragma unroll
    for (int i = 0; i < TH; ++i) acc[i] = 0.0f;
    // The parts of a step that a warp decodes: the quadrant's two tiles, the GROUP columns, cut into kSubs.
    // kWords words of a lane's four in kUnits tiles, 8 columns of tensor memory a word.
    constexpr int kUnits = GROUP == 128 && kSubs == 2 ? 2 : 1;
    constexpr int kWords = (GROUP == 32 ? 2 : 4) / (GROUP < 128 && kSubs == 4 ? 2 : 1);
    const int my_tile = kUnits == 2 ? 0 : sub & 1;
    const int my_half = GROUP == 128 ? (kSubs == 4 ? sub >> 1 : sub) : 0;      // of the step
    const int my_word = GROUP < 128 && kSubs == 4 ? (sub >> 1) * kWords : 0;   // of the step's part of a lane's words
    auto load_codes = [&](const uint8_t* stage, int gi, uint32_t (&c)[kUnits][kWords]) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int half = GROUP == 128 ? my_half : GROUP == 64 ? gi : gi >> 1;
        const int word = (GROUP == 32 ? (gi & 1) * 2 : 0) + my_word;
        const uint8_t* from = stage + codes_at + ((half * 4 + tile0 + my_tile + i) * 32 + lane) * 16 + word * 4;
        if constexpr (kWords == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(from);
          c[i][0] = v.x; c[i][1] = v.y; c[i][2] = v.z; c[i][3] = v.w;
        } else if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          c[i][0] = v.x; c[i][1] = v.y;
        } else {
          c[i][0] = *reinterpret_cast<const uint32_t*>(from);
        }
      }
    };

    constexpr int kAhead = kOperands / kSets - 1;   // steps that a set decodes before one is rescaled
    float scale[kAhead + 1];                        // of this step and the last ones
#pragma unroll
    for (int i = 0; i <= kAhead; ++i) scale[i] = 0.0f;
    bool ok = true;
    int sums = set;                                 // accumulator of the step that is rescaled next
    uint32_t parity = 0;
    constexpr int kBatch = TH % 16 == 0 ? 16 : 8;
    auto rescale = [&](float by) {
      if (!w4_wait_warp(wc, d_full(sums), parity)) return false;
      ptx::tc_fence_after();
#pragma unroll
      for (int c = 0; c < TH; c += kBatch) {
        float d[kBatch];
        ptx::tmem_ld<kBatch>(tmem + lane_base + sums * kTokens + sub * TH + c, d);
        ptx::tmem_ld_wait();
        if (c + kBatch == TH) {
          ptx::tc_fence_before();
          __syncwarp();
          if (kOperands > kSums && lane == 0) ptx::mbar_arrive(d_free(sums));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) acc[c + i] = fmaf(by, d[i], acc[c + i]);
      }
      sums += kSets;
      if (sums >= kSums) { sums -= kSums; parity ^= 1; }
      return true;
    };
    int operand = set, step = 0;                    // steps of this set
    // one step in two blocks, one in a block's two, two in its four; or every one
    for (int b = GROUP == 128 ? set : 0; ok && b < blocks; b += GROUP == 128 ? kSets : 1) {
      const int s = b % kStages;
      if (!w4_wait_warp(wc, full(s), (b / kStages) & 1)) { ok = false; break; }
      const uint8_t* stage = ring_ptr + s * p.stage_bytes;
      constexpr int kMine = GROUP == 128 ? 1 : kSteps / kSets;
#pragma unroll
      for (int j = 0; j < kMine; ++j, ++step) {
        const int gi = GROUP == 128 ? 0 : j * kSets + set;
        const uint32_t a_at = tmem_a + lane_base + operand * (GROUP / 2);
        uint32_t codes[kUnits][kWords];
        load_codes(stage, gi, codes);
#pragma unroll
        for (int i = kAhead; i > 0; --i) scale[i] = scale[i - 1];
        const uint16_t scale_bits = *reinterpret_cast<const uint16_t*>(stage + scale_at + gi * 128);
        // The last step that used this operand buffer has been rescaled, so the tensor core has left it.
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          uint32_t off0 = W4Traits<T>::kMinusEight, off1 = off0;
          if (f.zeros) {
            const uint32_t both = *reinterpret_cast<const uint32_t*>(stage + offset_at + gi * 128 + (tile0 + my_tile + i) * 4);
            off0 = __byte_perm(both, 0, 0x1010);
            off1 = __byte_perm(both, 0, 0x3232);
          }
          uint32_t r[kWords * 4];
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            uint32_t a[4];
            w4_decode<T>(codes[i][w], off0, off1, a);
            r[4 * w] = a[0]; r[4 * w + 1] = a[2]; r[4 * w + 2] = a[1]; r[4 * w + 3] = a[3];
          }
          ptx::tmem_st_16x256(a_at + ((uint32_t)((my_tile + i) * 16) << 16) + my_half * 32 + my_word * 8, r);
        }
        scale[0] = W4Traits<T>::to_float(scale_bits);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(a_full(operand));
          if (j == kMine - 1) ptx::mbar_arrive(empty(s));
        }
        operand += kSets;
        if (operand >= kOperands) operand -= kOperands;
        if (step >= kAhead && !rescale(scale[kAhead])) { ok = false; break; }
      }
    }
#pragma unroll
    for (int i = kAhead - 1; i >= 0; --i)
      if (ok && step > i) ok = rescale(scale[i]);
    if (!ok) {
#pragma unroll
      for (int i = 0; i < TH; ++i) acc[i] = __int_as_float(0x7fc00000);
    }
    ptx::tc_fence_before();
  } else if (warp < kTileCompute + kTileIssue) {
    // ---------------- MMA issue: the whole warp, one lane elected inside the statement ----------------
    // Two warps take turns at the steps: one would be the slowest part of the pipeline (a wait is 150
    // cycles, the instructions of a step 260, its commits 120).  They need not wait for the tokens: who
    // decoded the step has.
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc = (1u << 4) | (kType << 7) | (kType << 10) | ((kTokens >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t desc_hi = static_cast<uint32_t>(ptx::make_smem_desc_sw128(0, 16, 1024) >> 32);
    const int me = warp - kTileCompute;
    int operand = me, sums = me;
    uint32_t a_parity = 0, free_parity = 1;   // a fresh barrier has "completed" the phase before its first
    constexpr int kMine = GROUP == 128 ? 1 : kSteps / kTileIssue;
    for (int b = GROUP == 128 ? me : 0; b < blocks; b += GROUP == 128 ? kTileIssue : 1) {
      const int s = b % kStages;
      const uint32_t b_lo = static_cast<uint32_t>(ptx::make_smem_desc_sw128(ring + s * p.stage_bytes, 16, 1024));
      bool ok = true;
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int gi = GROUP == 128 ? 0 : j * kTileIssue + me;
        ok = w4_wait_warp(wc, a_full(operand), a_parity);
        // Decoders that run no further ahead than there are accumulators have emptied this one.
        if (kOperands > kSums) ok = ok && w4_wait_warp(wc, d_free(sums), free_parity);
        if (!ok) break;
        if (!p.vec) ptx::fence_proxy_async();   // the tokens were written by ordinary stores
        ptx::tc_fence_after();
        const uint32_t d = tmem + sums * kTokens, a = tmem_a + operand * (GROUP / 2);
        if constexpr (GROUP == 128) {
          ptx::umma_ts<4>(d, a, b_lo, desc_hi, idesc, 0);
          ptx::umma_ts<4>(d, a + 32, b_lo + (kXHalf >> 4), desc_hi, idesc, 1);
        } else if constexpr (GROUP == 64) {
          ptx::umma_ts<4>(d, a, b_lo + gi * (kXHalf >> 4), desc_hi, idesc, 0);
        } else {
          ptx::umma_ts<2>(d, a, b_lo + (gi >> 1) * (kXHalf >> 4) + (gi & 1) * 4, desc_hi, idesc, 0);
        }
        ptx::umma_commit_elect<1>(d_full(sums), 0);
        operand += kTileIssue;
        if (operand >= kOperands) { operand -= kOperands; a_parity ^= 1; }
        sums += kTileIssue;
        if (sums >= kSums) { sums -= kSums; free_parity ^= 1; }
      }
      if (!ok) break;
      ptx::umma_commit_elect<1>(empty(s), 0);
    }
  } else if (p.vec) {
    // ---------------- copies: one thread, tokens by tensor copies, codes by plain ones ----------------
    if (warp == kTileCompute + kTileIssue && lane == 0) {
      const uint32_t tx = kTokens * 256 + f.chunk_bytes * (two ? 2 : 1);
      for (int b = 0; b < blocks; ++b) {
        const int s = b % kStages;
        if (b >= kStages && !w4_wait(wc, empty(s), (b / kStages - 1) & 1)) break;
        const uint32_t stage = ring + s * p.stage_bytes;
        const uint8_t* chunk = data + (size_t)b * p.split * f.chunk_bytes;
        const int k = (rank + b * p.split) * kW4Block;
        ptx::mbar_expect_tx(full(s), tx);
        ptx::bulk_g2s(stage + kTokens * 256, chunk, f.chunk_bytes, full(s));
        if (two) ptx::bulk_g2s(stage + kTokens * 256 + f.chunk_bytes, chunk + strip_bytes, f.chunk_bytes, full(s));
        ptx::tma_load_2d(stage, &map, full(s), k, token0);
        ptx::tma_load_2d(stage + kXHalf, &map, full(s), k + 64, token0);
      }
    }
  } else {
    // ---------------- copies where rows of tokens start on no 16 bytes ----------------
    const int lt = threadIdx.x - (kTileCompute + kTileIssue) * 32, lw = lt >> 5;
    const int pieces = f.chunk_bytes / 16 * (two ? 2 : 1);
    // lane = 4 columns of a token, in the 128-byte swizzle
    const uint32_t unit = lane >> 1 & 7, low = (lane >> 4) * kXHalf + (lane & 1) * 8;
    const uint16_t* A = static_cast<const uint16_t*>(p.A);
    for (int b = 0; b < blocks; ++b) {
      const int s = b % kStages;
      if (b >= kStages && !w4_wait(wc, empty(s), (b / kStages - 1) & 1)) break;
      const uint32_t stage = ring + s * p.stage_bytes;
      const uint8_t* chunk = data + (size_t)b * p.split * f.chunk_bytes;
      for (int i = lt; i < pieces; i += kTileLoaders * 32) {
        const int o = i * 16;
        ptx::cp_async_16(stage + kTokens * 256 + o,
                         o < f.chunk_bytes ? chunk + o : chunk + strip_bytes + (o - f.chunk_bytes));
      }
      const long long k = (long long)(rank + b * p.split) * kW4Block + lane * 4;
#pragma unroll 4
      for (int m = lw; m < kTokens; m += kTileLoaders) {
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e[i] = token0 + m < p.M && k + i < f.K ? __ldg(A + (long long)(token0 + m) * p.lda + k + i) : 0u;
        *reinterpret_cast<uint2*>(ring_ptr + s * p.stage_bytes + low + m * 128 + ((unit ^ (m & 7)) << 4)) =
            make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
      }
      ptx::cp_async_commit();
      ptx::cp_async_wait<0>();
      ptx::mbar_arrive(full(s));
    }
    ptx::cp_async_commit();
    ptx::cp_async_wait<0>();
  }
  // a wait that ran out leaves MMAs that may still read the ring
  if (*s_abort != 0u) __nanosleep(50000);
  __syncthreads();
  if (warp == kTileCompute) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kCols);
  }

  // The sums, token by token, over the ring; the CTAs of a cluster then share the tokens.
  float* const red = reinterpret_cast<float*>(ring_ptr);
  if (warp < kTileCompute) {
    const int set = kSets == 2 ? warp >> 3 : 0, quad = warp & 3, sub = kSets == 2 ? (warp >> 2) & 1 : warp >> 2;
#pragma unroll
    for (int i = 0; i < TH; ++i) red[((set * kTokens) + sub * TH + i) * kTilePitch + quad * 32 + lane] = acc[i] * (1.0f / W4Traits<T>::kUnit);
  }
  if (p.split > 1) ptx::cluster_sync_all();
  else __syncthreads();
  // Four pairs of a token at a time: rows r .. r + 3 and r + 8 .. r + 11 of a tile.
  const int items = min(kTokens, p.M - token0) * (two ? 16 : 8);
  for (int e = rank * kTileThreads + threadIdx.x; e < items; e += p.split * kTileThreads) {
    const int token = two ? e >> 4 : e >> 3, quad = two ? e & 15 : e & 7;   // 8 quads of each strip
    const int r = (quad >> 3) * kW4Strip + (quad >> 1 & 3) * 16 + (quad & 1) * 4;
    const uint32_t at = ring + (token * kTilePitch + r) * 4;
    float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
    for (int c = 0; c < p.split; ++c) {
#pragma unroll
      for (int set = 0; set < kSets; ++set) {
        const uint32_t own = at + set * kTokens * kTilePitch * 4;
        const uint32_t a = p.split > 1 ? ptx::map_to_cta(own, c) : own;
        const float4 x = ptx::ld_cluster_f4(a), y = ptx::ld_cluster_f4(a + 32);
        u.x += x.x; u.y += x.y; u.z += x.z; u.w += x.w;
        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
      }
    }
    w4_epilogue4<T>(p, strip0 + (quad >> 3), (quad & 7) * 4, token0 + token, u, v);
  }
  if (p.split > 1) ptx::cluster_sync_all();   // nobody leaves while its shared memory is read
}

template <typename T, int TOKENS, int GROUP>
static int w4_tile_kernel_launch(const W4Params& p, const CUtensorMap& map, unsigned grid, cudaStream_t stream) {
  constexpr int kStages = w4_tile_stages(TOKENS);
  const int ring = kStages * p.stage_bytes, sums = (TOKENS <= 64 ? 2 : 1) * TOKENS * kTilePitch * 4;
  const int smem = 1024 + kTileControl + (ring > sums ? ring : sums);
  auto kern = w4_tile_kernel<T, TOKENS, GROUP>;
  static bool attr_set[64];
  int dev = 0;
  MKB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MKB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return w4_launch(kern, dim3(grid, 1, 1), kTileThreads, smem, p.split, stream, p, map);
}

template <typename T, int TOKENS>
static int w4_tile_group(const W4Params& p, const CUtensorMap& map, unsigned grid, cudaStream_t stream) {
  if (p.form.group == 32) return w4_tile_kernel_launch<T, TOKENS, 32>(p, map, grid, stream);
  if (p.form.group == 64) return w4_tile_kernel_launch<T, TOKENS, 64>(p, map, grid, stream);
  return w4_tile_kernel_launch<T, TOKENS, 128>(p, map, grid, stream);
}

template <typename T>
static int w4_tile_tokens(const W4Params& p, const CUtensorMap& map, int tokens, unsigned grid, cudaStream_t stream) {
  switch (tokens) {
    case 32: return w4_tile_group<T, 32>(p, map, grid, stream);
    case 64: return w4_tile_group<T, 64>(p, map, grid, stream);
    case 96: return w4_tile_group<T, 96>(p, map, grid, stream);
    default: return w4_tile_group<T, 128>(p, map, grid, stream);
  }
}

// Tokens as a tensor map: boxes of 64 columns (128 bytes, swizzled) of a CTA's tokens; columns behind K and
// rows behind M read as zeros.
static int w4_tile_map(CUtensorMap* map, const W4Params& p, int dtype, int tokens) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    const int rc = driver_entry("cuTensorMapEncodeTiled", &fn);
    if (rc != MK_OK) return rc;
    encode = reinterpret_cast<Encode>(fn);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)p.form.K, (cuuint64_t)p.M};
  const cuuint64_t strides[1] = {(cuuint64_t)p.lda * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)tokens}, ones[2] = {1, 1};
  const CUresult r =
      encode(map, dtype == MK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(p.A), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(MK_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return MK_OK;
}

int w4_tile_launch(W4Params& p, int dtype, int sms, cudaStream_t stream) {
  const W4Form& f = p.form;
  const long long row_tiles = (f.strips + 1) / 2;
  // Tokens to a CTA and CTAs to a cluster along K: whichever finishes first by a rough count of cycles,
  // 330 or 5 a token for a block, 4000 to start and end, 1500 more for a cluster.
  int tokens = 128;
  long long best = -1;
  for (int t = 32; t <= 128; t += 32)
    for (int split = 1; split <= 8 && split <= f.blocks; split *= 2) {
      const long long units = row_tiles * ((p.M + t - 1) / t) * split;
      const long long waves = (units + sms - 1) / sms;
      if (split > 1 && waves > 1) continue;
      const long long cost = waves * ((long long)((f.blocks + split - 1) / split) * (5 * t < 330 ? 330 : 5 * t) + 4000) +
                             (split > 1 ? 1500 : 0);
      if (best < 0 || cost < best) { best = cost; tokens = t; p.split = split; }
    }
  p.token_tiles = (p.M + tokens - 1) / tokens;
  p.stage_bytes = (tokens * 256 + 2 * f.chunk_bytes + 1023) / 1024 * 1024;
  p.vec = (reinterpret_cast<uintptr_t>(p.A) & 15) == 0 && p.lda % 8 == 0;
  CUtensorMap map = {};
  if (p.vec) {
    const int rc = w4_tile_map(&map, p, dtype, tokens);
    if (rc != MK_OK) return rc;
  }
  const long long grid = row_tiles * p.token_tiles * p.split;
  if (grid > 0x7fffffffLL) return set_error(MK_ERR_INVALID, "4-bit product: M=%d, N=%d is too large", p.M, f.N);
  return dtype == MK_BF16 ? w4_tile_tokens<__nv_bfloat16>(p, map, tokens, (unsigned)grid, stream)
                          : w4_tile_tokens<__half>(p, map, tokens, (unsigned)grid, stream);
}

}  // namespace mkb
