// The product with 4-bit weights for more than a few tokens, on the 5th-generation tensor cores.
//
// A CTA computes 128 rows of the matrix (two strips) for up to 256 tokens, D = W A^T with the weights as
// the 128-row operand.  That operand never exists in shared memory: the lanes that decode the codes
// write the weights into tensor memory, in the 16x256b form whose lanes are the layout's lanes, and the
// MMA takes its A operand from there.  So shared memory carries only the packed codes and the tokens.
//
// Here a weight is rounded to the 16-bit type before it is multiplied, (code - zero) * scale, exactly as
// mk_w4_dequantize gives it, and D stays in tensor memory from the first column to the last.  The
// few-token kernel rounds nothing; to do the same here the sums of every group must leave the tensor core to
// be scaled in fp32, which was built first and costs a tour through registers and two waits a group
// (256 tokens of 8192 x 8192 in groups of 64: 59 us that way, 29 this, or 1180 TFLOP/s).  What the rounding adds is
// smaller than the output's own (relative to the result 1.4e-3 in bf16, where that is 1.7e-3).  In the
// SwiGLU form two such sums are multiplied and it would be larger (2.1e-3), so there what the rounding left
// (REST) is multiplied as well, and nothing is lost.  The rule: rounding is taken where what it adds stays below
// the rounding of the output that follows in any case; MK_W4_EXACT takes the rest in the other forms too.
//
// Warps 0..15 decode, in two sets that take turns at the blocks of 128 columns (quadrant warp % 4 of the
// lanes, half of the columns by warp / 4 % 2), and at the end read the sums; warps 16 and 17 issue the
// MMAs; a thread each of warps 18 to 21 copies a ring of stages (a block: codes of two strips, tokens in the
// 128-byte swizzle).  A block is little work and a long way, from a barrier to the next whatever the tokens: in a
// grid of 128 CTAs it takes 324, 335, 516 and 841 ns for 32, 64, 128 and 256 tokens, of which its MMAs at the tensor
// core's rate are 92, 184, 368 and 736.  So what bounds a narrow product is how many blocks are under way, and up to
// 128 tokens two warps issue, every other block each, into sums of their own.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>
#include <type_traits>

#include "../../include/mkernel_b200.h"
#include "w4_product.cuh"

namespace mkb {

constexpr int kTileRows = 2 * kW4Strip;
constexpr int kTileCompute = 16;                   // warps, in two sets
constexpr int kTileSet = 8;
constexpr int kTileIssue = 2;
constexpr int kTileLoaders = 4;
constexpr int kTileThreads = (kTileCompute + kTileIssue + kTileLoaders) * 32;
constexpr int kTileControl = 1024;                 // bytes before the ring
constexpr int kTilePitch = kTileRows + 4;          // floats of a token's sums

// Up to 128 tokens two of everybody (sets of decoding warps, issuing warps with sums of their own, copying
// threads) take turns at the blocks; for 256, whose MMAs are long enough to hide the rest, all decoding
// warps share every block, and one warp issues.
// Who takes turns sees every other phase of a barrier only if the number of stages (or operand buffers) is odd,
// and could then take the phase before the last for the last: both numbers are multiples of the turns.
__host__ __device__ constexpr int w4_tile_turns(int tokens) { return tokens <= 128 ? 2 : 1; }
// Stages of the ring, and operand buffers (64 columns of tensor memory, or 128): what 227 KB and, beside the
// sums, 512 columns hold.
__host__ __device__ constexpr int w4_tile_stages(int tokens) { return tokens <= 64 ? 6 : tokens == 128 ? 4 : 3; }
__host__ __device__ constexpr int w4_tile_operands(int tokens, bool rest) { return rest ? 2 : w4_tile_stages(tokens); }

struct TileWait {
  volatile uint32_t* abort;   // shared: some wait of this CTA has run out, and the barrier that it was for
  uint64_t limit_ns;
};

// What a wait that ran out leaves behind: {code, CTA << 8 | kind of barrier, its offset, blocks of the CTA}, of the
// first CTA that met one since the words were cleared.
__device__ uint32_t w4_status_words[4];

// False when the wait has run out, here or elsewhere in the CTA.  `draining`: after that has happened, for what is
// still under way; runs out by itself alone.
__device__ __noinline__ bool w4_slow_wait(const TileWait& c, uint32_t bar, uint32_t parity, bool draining = false) {
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((it & 127u) == 0u) {
      if (!draining && *c.abort != 0u) return false;
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > c.limit_ns) {
        if (!draining) {
          c.abort[1] = bar;
          c.abort[0] = 1u;
        }
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

// Whether a copying thread is to stop here: never, but in the diagnostics build, where "debug_flags" can make a copy go
// missing (4: tokens, 8: codes; of block debug_flags >> 8 in the first CTA of each cluster) to see the waits for
// it run out.
__device__ __forceinline__ bool w4_copy_missing(const W4Params& p, int rank, bool tokens, int block) {
#ifdef MKB_DIAG
  return (p.debug_flags & (tokens ? 4 : 8)) != 0 && rank == 0 && block >= p.debug_flags >> 8;
#else
  return false;
#endif
}

template <typename T, int TOKENS, int GROUP, bool REST>
__global__ void __launch_bounds__(kTileThreads, 1)
    w4_tile_kernel(const __grid_constant__ W4Params p, const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kTokens = TOKENS;
  constexpr int kStages = w4_tile_stages(kTokens);
  constexpr int kOperands = w4_tile_operands(kTokens, REST), kOperand = REST ? 128 : 64;   // columns of one
  constexpr int kTurns = w4_tile_turns(kTokens), kSums = kTurns;
  static_assert(kStages % kTurns == 0 && kOperands % kTurns == 0, "no phase of a barrier is skipped");
  constexpr uint32_t kCols = 512;
  static_assert(kSums * kTokens + kOperand * kOperands <= kCols, "tensor memory has 512 columns");
  constexpr bool kOwn = kOperands < kStages;        // else an operand buffer is free when its stage is
  constexpr int kXHalf = kTokens * 128;             // bytes of 64 columns of the tokens

  const W4Form& f = p.form;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw);
  // control words: full[6] empty[6] a_full[6] a_empty[2] done | tensor memory address, abort flag, barrier, blocks
  // issued by the four copying threads
  auto full = [&](int s) { return base + 8u * s; };
  auto empty = [&](int s) { return base + 64u + 8u * s; };
  auto a_full = [&](int i) { return base + 128u + 8u * i; };
  auto a_empty = [&](int i) { return base + 192u + 8u * i; };
  const uint32_t done = base + 216u;
  volatile uint32_t* const s_tmem = reinterpret_cast<volatile uint32_t*>(base_ptr + 224);
  volatile uint32_t* const s_abort = s_tmem + 1;
  volatile uint32_t* const s_issued = s_tmem + 3;
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
      ptx::mbar_init(full(s), 2);
      ptx::mbar_init(empty(s), kTileCompute / kTurns + 1);
    }
    for (int i = 0; i < kOperands; ++i) {
      ptx::mbar_init(a_full(i), kTileCompute / kTurns);
      if (kOwn) ptx::mbar_init(a_empty(i), 1);
    }
    ptx::mbar_init(done, kSums);
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

  const int quad = warp & 3, half = warp >> 2 & 1;
  bool ok = true;
  if (warp < kTileCompute) {
    // ---------------- decode ----------------
    const int g = lane >> 2;
    const int strip = quad >> 1;
    constexpr int kGroups = kW4Block / GROUP;
    // of a stage: this lane's codes of two tiles, and the scales and zero points of its rows there
    constexpr int kTiles = kTurns;         // of the quadrant's two that a warp decodes
    const int tile0 = (quad & 1) * 2 + (kTiles == 1 ? warp / kTileSet : 0);
    const int codes_at = kTokens * 256 + strip * f.chunk_bytes + ((half * 4 + tile0) * 32 + lane) * 16;
    const int scales_at = kTokens * 256 + strip * f.chunk_bytes + kW4CodeBytes + g * 16 + tile0 * 4 +
                          (half * 64 / GROUP) * 128;
    const uint32_t a_at = tmem_a + ((uint32_t)(strip * 64 + tile0 * 16) << 16) + half * 32;
    for (int b = kTurns == 2 ? warp / kTileSet : 0; b < blocks; b += kTurns) {
      const int s = b % kStages, operand = b % kOperands;
      ok = w4_wait_warp(wc, full(s), (b / kStages) & 1);
      if (!ok) break;
      const uint8_t* stage = ring_ptr + s * p.stage_bytes;
      uint4 codes[kTiles];
      uint32_t scales[GROUP == 32 ? 2 : 1][kTiles], zeros[GROUP == 32 ? 2 : 1][kTiles];   // of rows g, g + 8
#pragma unroll
      for (int i = 0; i < kTiles; ++i) codes[i] = *reinterpret_cast<const uint4*>(stage + codes_at + i * 512);
#pragma unroll
      for (int gi = 0; gi < (GROUP == 32 ? 2 : 1); ++gi)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const uint8_t* from = stage + scales_at + gi * 128 + i * 4;
          scales[gi][i] = *reinterpret_cast<const uint32_t*>(from);
          zeros[gi][i] = f.zeros ? *reinterpret_cast<const uint32_t*>(from + kGroups * 128) : W4Traits<T>::kMinusEight;
        }
      if (kOwn && b >= kOperands) {
        ok = w4_wait_warp(wc, a_empty(operand), (b / kOperands - 1) & 1);
        if (!ok) break;
      }
      ptx::tc_fence_after();
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const uint32_t words[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
        uint32_t r[16], rest[16];
#pragma unroll
        for (int v = 0; v < 4; v += 2) {
          const int gi = GROUP == 32 ? v / 2 : 0;
          const uint32_t sc = scales[gi][i], z = zeros[gi][i];
          const W4Round<T> weights(__byte_perm(z, 0, 0x1010), __byte_perm(z, 0, 0x3232), __byte_perm(sc, 0, 0x1010),
                                   __byte_perm(sc, 0, 0x3232));
#pragma unroll
          for (int w = v; w < v + 2; ++w) {
            uint32_t a[4], b[4];
            weights.template get<REST>(words[w], a, b);
            r[4 * w] = a[0]; r[4 * w + 1] = a[2]; r[4 * w + 2] = a[1]; r[4 * w + 3] = a[3];
            if (REST) { rest[4 * w] = b[0]; rest[4 * w + 1] = b[2]; rest[4 * w + 2] = b[1]; rest[4 * w + 3] = b[3]; }
          }
        }
        ptx::tmem_st_16x256(a_at + operand * kOperand + ((uint32_t)(i * 16) << 16), r);
        if (REST) ptx::tmem_st_16x256(a_at + operand * kOperand + 64 + ((uint32_t)(i * 16) << 16), rest);
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(a_full(operand));
        ptx::mbar_arrive(empty(s));
      }
    }
    if (ok) w4_wait_warp(wc, done, 0);
  } else if (warp < kTileCompute + kTileIssue) {
    // ---------------- MMA issue: the whole warp, one lane elected inside the statement ----------------
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc = (1u << 4) | (kType << 7) | (kType << 10) | ((kTokens >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t desc_hi = static_cast<uint32_t>(ptx::make_smem_desc_sw128(0, 16, 1024) >> 32);
    const uint32_t b_lo0 = static_cast<uint32_t>(ptx::make_smem_desc_sw128(ring, 16, 1024));
    const int me = warp - kTileCompute;
    const uint32_t d = tmem + me * kTokens;
    for (int b = me; me < kSums && b < blocks; b += kSums) {
      const int s = b % kStages, operand = b % kOperands;
      // The tokens need no wait of their own: who decoded the block has waited for them.
      ok = w4_wait_warp(wc, a_full(operand), (b / kOperands) & 1);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t a = tmem_a + operand * kOperand, b_lo = b_lo0 + s * (p.stage_bytes >> 4);
      ptx::umma_ts(d, a, b_lo, desc_hi, idesc, b >= kSums ? 1u : 0u);
      ptx::umma_ts(d, a + 32, b_lo + (kXHalf >> 4), desc_hi, idesc, 1);
      if (REST) {
        ptx::umma_ts(d, a + 64, b_lo, desc_hi, idesc, 1);
        ptx::umma_ts(d, a + 96, b_lo + (kXHalf >> 4), desc_hi, idesc, 1);
      }
      if (kOwn) ptx::umma_commit_elect<1>(a_empty(operand), 0);
      ptx::umma_commit_elect<1>(empty(s), 0);
    }
    if (me < kSums) ptx::umma_commit_elect<1>(done, 0);   // given up or not: when what was issued has finished
  } else {
    // ---------------- copies: two threads for the codes, two for the tokens (tensor copies) ----------------
    const int me = warp - kTileCompute - kTileIssue;
    const bool tokens = me >= 2, active = lane == 0 && (me & 1) < kTurns;
    const uint32_t tx = tokens ? kTokens * 256 : f.chunk_bytes * (two ? 2 : 1);
    int b = me & 1;
    for (; active && b < blocks; b += kTurns) {
      const int s = b % kStages;
      if (b >= kStages && !w4_wait(wc, empty(s), (b / kStages - 1) & 1)) break;
      if (w4_copy_missing(p, rank, tokens, b)) break;
      const uint32_t stage = ring + s * p.stage_bytes;
      ptx::mbar_expect_tx(full(s), tx);
      if (tokens) {
        const int k = (rank + b * p.split) * kW4Block;
        ptx::tma_load_2d(stage, &map, full(s), k, token0);
        ptx::tma_load_2d(stage + kXHalf, &map, full(s), k + 64, token0);
      } else {
        const uint8_t* chunk = data + (size_t)b * p.split * f.chunk_bytes;
        ptx::bulk_g2s(stage + kTokens * 256, chunk, f.chunk_bytes, full(s));
        if (two) ptx::bulk_g2s(stage + kTokens * 256 + f.chunk_bytes, chunk + strip_bytes, f.chunk_bytes, full(s));
      }
    }
    if (active) s_issued[me] = b;
  }
  __syncthreads();
  // Every role has ended, and whether a wait ran out is settled.  Where one did, copies and MMAs may be under way: nobody
  // writes over the ring, or leaves, before they have finished (or the limit has passed once more for each).
  bool spoiled = *s_abort != 0u;
  if (spoiled) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < kStages; ++s) {
        // Phases of full(s) that each of the stage's two copying threads has started: equal, or one ahead by one.
        const uint32_t codes = s_issued[s % kTurns], tokens = s_issued[2 + s % kTurns];
        const uint32_t n = (codes + kStages - 1 - s) / kStages, m = (tokens + kStages - 1 - s) / kStages;
        if (n != m) ptx::mbar_arrive(full(s));       // in the place of the copy that was never started
        const uint32_t last = n > m ? n : m;
        if (last > 0) w4_slow_wait(wc, full(s), (last - 1) & 1, true);
      }
      w4_slow_wait(wc, done, 0, true);
      const uint32_t at = s_abort[1] - base;
      if (atomicCAS(&w4_status_words[0], 0u, 1u) == 0u) {
        w4_status_words[1] = blockIdx.x << 8 | at / 64;
        w4_status_words[2] = at;
        w4_status_words[3] = blocks;
        __threadfence();
      }
    }
    __syncthreads();
  }

  // The sums, token by token, over the ring; the CTAs of a cluster then share the tokens.
  float* const red = reinterpret_cast<float*>(ring_ptr);
  if (warp < kTileCompute && !spoiled) {
    ptx::tc_fence_after();
    constexpr int kEach = kTokens / 4, kBatch = kEach < 16 ? 8 : 16;
    const int c0 = (warp >> 2) * kEach;
#pragma unroll
    for (int c = 0; c < kEach; c += kBatch) {
      float d[kBatch];
      ptx::tmem_ld<kBatch>(tmem + ((uint32_t)(quad * 32) << 16) + c0 + c, d);
      ptx::tmem_ld_wait();
      if (kSums == 2 && blocks > 1) {   // the second sums are of the blocks 1, 3, ...
        float e[kBatch];
        ptx::tmem_ld<kBatch>(tmem + ((uint32_t)(quad * 32) << 16) + kTokens + c0 + c, e);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kBatch; ++i) d[i] += e[i];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        red[(c0 + c + i) * kTilePitch + quad * 32 + lane] = d[i];
    }
    ptx::tc_fence_before();
  }
  if (p.split > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp == kTileCompute) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kCols);
  }
  // Where a CTA of the cluster gave up there are no sums: NaN, whatever lies in the ring.
  for (int c = 0; p.split > 1 && c < p.split; ++c)
    spoiled |= ptx::ld_cluster_u32(ptx::map_to_cta(base + 228u, c)) != 0u;
  const float nothing = spoiled ? __int_as_float(0x7fc00000) : 0.0f;
  // Four pairs of a token at a time: rows r .. r + 3 and r + 8 .. r + 11 of a tile.
  const int items = min(kTokens, p.M - token0) * (two ? 16 : 8);
  for (int e = rank * kTileThreads + threadIdx.x; e < items; e += p.split * kTileThreads) {
    const int token = two ? e >> 4 : e >> 3, quad = two ? e & 15 : e & 7;   // 8 quads of each strip
    const int r = (quad >> 3) * kW4Strip + (quad >> 1 & 3) * 16 + (quad & 1) * 4;
    const uint32_t at = ring + (token * kTilePitch + r) * 4;
    float4 u = make_float4(nothing, nothing, nothing, nothing), v = u;
    for (int c = 0; c < p.split && !spoiled; ++c) {
      const uint32_t a = p.split > 1 ? ptx::map_to_cta(at, c) : at;
      const float4 x = ptx::ld_cluster_f4(a), y = ptx::ld_cluster_f4(a + 32);
      u.x += x.x; u.y += x.y; u.z += x.z; u.w += x.w;
      v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    w4_epilogue4<T>(p, strip0 + (quad >> 3), (quad & 7) * 4, token0 + token, u, v);
  }
  if (p.split > 1) ptx::cluster_sync_all();   // nobody leaves while its shared memory is read
}

template <typename T, int TOKENS, int GROUP, bool REST>
static int w4_tile_kernel_launch(const W4Params& p, const CUtensorMap& map, unsigned grid, cudaStream_t stream) {
  constexpr int kStages = w4_tile_stages(TOKENS);
  const int ring = kStages * p.stage_bytes, sums = TOKENS * kTilePitch * 4;
  // More than half of what an SM has, so that two CTAs never share one: the second would wait for the first's
  // tensor memory, and two clusters might so wait for one another.
  const int least = 120 * 1024, need = 1024 + kTileControl + (ring > sums ? ring : sums);
  const int smem = need > least ? need : least;
  auto kern = w4_tile_kernel<T, TOKENS, GROUP, REST>;
  static bool attr_set[64];
  int dev = 0;
  MKB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MKB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return w4_launch(kern, dim3(grid, 1, 1), kTileThreads, smem, p.split, stream, p, map);
}

template <typename T, int TOKENS, bool REST>
static int w4_tile_group(const W4Params& p, const CUtensorMap& map, unsigned grid, cudaStream_t stream) {
  if (p.form.group == 32) return w4_tile_kernel_launch<T, TOKENS, 32, REST>(p, map, grid, stream);
  if (p.form.group == 64) return w4_tile_kernel_launch<T, TOKENS, 64, REST>(p, map, grid, stream);
  return w4_tile_kernel_launch<T, TOKENS, 128, REST>(p, map, grid, stream);
}
template <typename T, int TOKENS>
static int w4_tile_rest(const W4Params& p, const CUtensorMap& map, bool rest, unsigned grid, cudaStream_t stream) {
  return rest ? w4_tile_group<T, TOKENS, true>(p, map, grid, stream) : w4_tile_group<T, TOKENS, false>(p, map, grid, stream);
}

template <typename T>
static int w4_tile_tokens(const W4Params& p, const CUtensorMap& map, int tokens, bool rest, unsigned grid,
                          cudaStream_t stream) {
  switch (tokens) {
    case 32: return w4_tile_rest<T, 32>(p, map, rest, grid, stream);
    case 64: return w4_tile_rest<T, 64>(p, map, rest, grid, stream);
    case 128: return w4_tile_rest<T, 128>(p, map, rest, grid, stream);
    default: return w4_tile_rest<T, 256>(p, map, rest, grid, stream);
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

// How many clusters of 2, 4 or 8 CTAs run at once on the current device: fewer than its SMs give room for, since
// the CTAs of one share a part of the chip (of 4: 33 on 148 SMs).  All instances take an SM to a CTA.
static int w4_tile_clusters(int split, int* out) {
  static int cached[64][9];
  int dev = 0;
  MKB_CUDA(cudaGetDevice(&dev));
  const bool keep = dev >= 0 && dev < 64;
  if (!keep || cached[dev][split] == 0) {
    auto kern = w4_tile_kernel<__nv_bfloat16, 64, 128, false>;
    const int smem = 200 * 1024;
    MKB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split, 1, 1);
    cfg.blockDim = dim3(kTileThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MKB_CUDA(cudaOccupancyMaxActiveClusters(out, kern, &cfg));
    if (keep) cached[dev][split] = *out;
    return MK_OK;
  }
  *out = cached[dev][split];
  return MK_OK;
}

// Tokens to a CTA and CTAs to a cluster along K: whichever finishes first by what a block and a start and end
// take in ns (at 32, 64, 128 and 256 tokens, in grids that leave the chip room; 1.5 us more for a cluster of two).
// Clusters only where all of them run at once: 64 tokens of 4608 x 4096 take 18.7 us in 36 clusters of 4, 10.5 in 36
// of 2.  Against all other cuts of 41 shapes: within 2 % of the best at 35, 10 % from it at most.
int w4_tile_plan(const W4Form& f, int M, bool rest, int sms, W4TilePlan* out) {
  const long long row_tiles = (f.strips + 1) / 2;
  const int block_ns[2][4] = {{280, 290, 370, 500}, {400, 540, 800, 1250}}, ends_ns[4] = {3000, 3000, 4500, 8000};
  out->tokens = 128;
  out->split = 1;
  long long best = -1;
  int clusters[9] = {};
  for (int split = 2; split <= 8; split *= 2) {
    const int rc = w4_tile_clusters(split, &clusters[split]);
    if (rc != MK_OK) return rc;
  }
  for (int i = 0; i < 4; ++i)
    for (int split = 1; split <= 8 && split <= f.blocks; split *= 2) {
      const int t = 32 << i;
      const long long units = row_tiles * (((long long)M + t - 1) / t);
      if (split > 1 && units > clusters[split]) continue;
      const long long waves = (units * split + sms - 1) / sms;
      const long long each = (long long)((f.blocks + split - 1) / split) * block_ns[rest][i] + ends_ns[i];
      const long long cost = waves * each + (split > 1 ? 750 * split : 0);
      if (best < 0 || cost < best) { best = cost; out->tokens = t; out->split = split; }
    }
  out->token_tiles = (int)(((long long)M + out->tokens - 1) / out->tokens);
  out->ctas = row_tiles * out->token_tiles * out->split;
  if (out->ctas > 0x7fffffffLL) return set_error(MK_ERR_INVALID, "4-bit product: M=%d, N=%d is too large", M, f.N);
  return MK_OK;
}

int w4_tile_launch(W4Params& p, int dtype, bool rest, int sms, cudaStream_t stream) {
  W4TilePlan pl;
  int rc = w4_tile_plan(p.form, p.M, rest, sms, &pl);
  if (rc != MK_OK) return rc;
  p.split = pl.split;
  p.token_tiles = pl.token_tiles;
  p.stage_bytes = (pl.tokens * 256 + 2 * p.form.chunk_bytes + 1023) / 1024 * 1024;
  CUtensorMap map;
  rc = w4_tile_map(&map, p, dtype, pl.tokens);
  if (rc != MK_OK) return rc;
  return dtype == MK_BF16 ? w4_tile_tokens<__nv_bfloat16>(p, map, pl.tokens, rest, (unsigned)pl.ctas, stream)
                          : w4_tile_tokens<__half>(p, map, pl.tokens, rest, (unsigned)pl.ctas, stream);
}

}  // namespace mkb

using namespace mkb;

extern "C" {

int mk_w4_status(uint32_t out4[4]) {
  uint32_t w[4] = {0, 0, 0, 0};
  MKB_CUDA(cudaMemcpyFromSymbol(w, w4_status_words, sizeof(w)));
  if (out4) memcpy(out4, w, sizeof(w));
  if (w[0] != 0)
    return set_error(MK_ERR_DEVICE_WAIT, "4-bit product: device wait expired: code=%u cta=%u role=%u detail=(%u,%u)", w[0],
                     w[1] >> 8, w[1] & 255u, w[2], w[3]);
  return MK_OK;
}

int mk_w4_status_clear(void* stream) {
  void* words = nullptr;
  MKB_CUDA(cudaGetSymbolAddress(&words, w4_status_words));
  MKB_CUDA(cudaMemsetAsync(words, 0, sizeof(w4_status_words), static_cast<cudaStream_t>(stream)));
  return MK_OK;
}

}  // extern "C"
