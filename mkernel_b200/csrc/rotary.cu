// Rotary positions on rows of heads: y = x with the first rotary_dim features of every head turned by
// position * inv_freq.  Nothing but one read and one write of every element, so bound by memory:
// 8192 rows of 40 heads of 128 in bf16 take 31.7 us, 5.3 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mkernel_b200.h"
#include "host_util.h"
#include "ptx.cuh"
#include "rotary.cuh"

namespace mkb {

struct RotaryParams {
  const void* x;
  void* y;
  long long x_row, x_head, y_row, y_head;   // strides in elements
  long long rows;
  int heads, head_dim, rotary_dim;
  int slots, turned;       // of a head; the first `turned` turn, the others copy
  int per_row;             // slots of a row
  int rows_each;           // rows of a CTA
  int rows_abreast;        // rows that its threads take at once
  float sign;
  RotaryArgs rotary;
};

constexpr int kRotaryThreads = 512;  // at most
constexpr int kRotaryAhead = 2;      // rows whose loads a thread has in flight
constexpr int kRotaryAngles = 2048;  // of a CTA (16 KB of shared memory)

template <typename T, int P> struct alignas(sizeof(T) * P) RotaryVec { T v[P]; };

// Written as data that passes through: 8192 rows of 40 heads of 128 take 31 us so, 35 without.
template <typename T, int P>
__device__ __forceinline__ void rotary_store(T* to, const RotaryVec<T, P>& v) {
  if constexpr (sizeof(v) == 16) __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&v));
  else *reinterpret_cast<RotaryVec<T, P>*>(to) = v;
}

// A slot is P pairs of features of a head: vector 0 and vector 1 of P elements each, which are the
// first and second features of the pairs, or, interleaved, the pairs one after another.  A CTA has some
// whole rows; a thread has one slot of one head and goes down the rows, several loads ahead, so that
// nothing but pointers changes from one to the next.  The rows' angles are worked out once by all
// threads (sine and cosine, in 64 bits up to the turn, cost as much as turning several heads) while the
// first rows are on their way, and found in shared memory for every head.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, 2) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using Vec = RotaryVec<T, P>;
  __shared__ __align__(16) float2 angles[kRotaryAngles];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long row0 = (long long)blockIdx.x * p.rows_each;
  const int rows = (int)min((long long)p.rows_each, p.rows - row0);
  const int pairs = p.rotary_dim / 2;
  const int abreast = p.rows_abreast;

  auto work_out_angles = [&] {
    for (int e = threadIdx.x; e < rows * pairs; e += blockDim.x) {
      const int r = rows == 1 ? 0 : e / pairs;
      float2 cs = rotary_cos_sin(rotary_position(p.rotary, row0 + r), p.rotary.inv_freq[e - r * pairs],
                                 p.rotary.scale);
      cs.y *= p.sign;
      angles[e] = cs;
    }
    __syncthreads();
  };
  const int first_row = abreast == 1 ? 0 : threadIdx.x / p.per_row;
  bool have_angles = false;
  for (int in_row = threadIdx.x - first_row * p.per_row; in_row < p.per_row || !have_angles; in_row += blockDim.x) {
    const bool mine = in_row < p.per_row && first_row < abreast;   // the last warp may have threads to spare
    const int h = in_row / p.slots, slot = in_row - h * p.slots;
    const bool turns = slot < p.turned;
    const int a = !turns ? p.rotary_dim + (slot - p.turned) * 2 * P : INTERLEAVED ? slot * 2 * P : slot * P;
    const int b = turns && !INTERLEAVED ? a + pairs : a + P;
    const bool second = b < p.head_dim;   // the last vector of a head's copied features may not exist
    const T* x = static_cast<const T*>(p.x) + (row0 + first_row) * p.x_row + h * p.x_head;
    T* y = static_cast<T*>(p.y) + (row0 + first_row) * p.y_row + h * p.y_head;
    const long long x_step = abreast * p.x_row, y_step = abreast * p.y_row;
    Vec u[kRotaryAhead], v[kRotaryAhead];
    int next = first_row;                 // row of the next load
    auto load = [&](int c) {
      if (mine && next < rows) {
        u[c] = *reinterpret_cast<const Vec*>(x + a);
        if (second) v[c] = *reinterpret_cast<const Vec*>(x + b);
      }
      x += x_step;
      next += abreast;
    };
#pragma unroll
    for (int c = 0; c < kRotaryAhead; ++c) load(c);
    if (!have_angles) {
      work_out_angles();
      have_angles = true;
    }
    if (!mine) continue;
    for (int r0 = first_row; r0 < rows; r0 += kRotaryAhead * abreast) {
#pragma unroll
      for (int c = 0; c < kRotaryAhead; ++c) {
        const int r = r0 + c * abreast;
        if (r >= rows) break;
        if (turns) {
          const float2* cs = angles + r * pairs + slot * P;
#pragma unroll
          for (int k = 0; k < P; ++k) {
            // pair k: elements k of both vectors, or elements 2 k and 2 k + 1 of the two in a row
            T& first = INTERLEAVED ? (2 * k < P ? u[c].v[2 * k % P] : v[c].v[2 * k % P]) : u[c].v[k];
            T& other = INTERLEAVED ? (2 * k + 1 < P ? u[c].v[(2 * k + 1) % P] : v[c].v[(2 * k + 1) % P]) : v[c].v[k];
            const float2 t = rotary_turn((float)first, (float)other, cs[k]);
            first = (T)t.x;
            other = (T)t.y;
          }
        }
        rotary_store(y + a, u[c]);
        if (second) rotary_store(y + b, v[c]);
        y += y_step;
        load(c);
      }
    }
  }
}

template <typename T, int P>
static int rotary_launch(RotaryParams& p, bool interleaved, bool in_place, int sms, cudaStream_t stream) {
  p.turned = p.rotary_dim / 2 / P;
  p.slots = p.turned + (in_place ? 0 : (p.head_dim - p.rotary_dim + 2 * P - 1) / (2 * P));
  const long long per_row = (long long)p.heads * p.slots;
  if (per_row > 1 << 30 || p.rotary_dim / 2 > kRotaryAngles)
    return set_error(MK_ERR_INVALID, "mk_rotary: heads of %d (%d turned) features, %d to a row, are too many", p.head_dim,
                     p.rotary_dim, p.heads);
  p.per_row = (int)per_row;
  // Rows abreast up to about 256 threads; rows of a CTA such that one wave of 1024 threads to an SM has them
  // all (with a CTA to each row its latency comes back with every wave: 8192 rows of 40 heads of 128 took 54
  // us, 4097 rows of 9 heads 7.7 with 600 threads), within what their angles leave room for.
  const int room = kRotaryAngles / (p.rotary_dim / 2);
  int abreast = per_row >= 256 ? 1 : (int)(256 / per_row);
  if (abreast > room) abreast = room;
  if (abreast > p.rows) abreast = (int)p.rows;
  long long threads = (abreast * per_row + 31) / 32 * 32;
  if (threads > kRotaryThreads) threads = kRotaryThreads;
  const long long wave = 1024 / threads * sms;
  long long rows_each = (p.rows + wave - 1) / wave;
  rows_each = (rows_each + abreast - 1) / abreast * abreast;
  if (rows_each > room) rows_each = room;
  p.rows_abreast = abreast;
  p.rows_each = (int)rows_each;
  const long long blocks = (p.rows + rows_each - 1) / rows_each;
  if (blocks > 0x7fffffffLL) return set_error(MK_ERR_INVALID, "mk_rotary: %lld rows are too many", p.rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option_pdl() ? 1 : 0;
  if (interleaved) MKB_CUDA(cudaLaunchKernelEx(&cfg, rotary_kernel<T, P, true>, p));
  else MKB_CUDA(cudaLaunchKernelEx(&cfg, rotary_kernel<T, P, false>, p));
  return MK_OK;
}

// The widest vectors that every address and part of a head is a multiple of: 16 bytes, 4, one element.
template <typename T>
static int rotary_type(RotaryParams& p, bool interleaved, bool in_place, int sms, cudaStream_t stream) {
  auto fits = [&](int elems) {
    const long long m = elems;
    return (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) % (m * sizeof(T)) == 0 &&
           p.x_row % m == 0 && p.x_head % m == 0 && p.y_row % m == 0 && p.y_head % m == 0 &&
           p.rotary_dim / 2 % m == 0 && p.head_dim % m == 0;
  };
  constexpr int kWide = 16 / sizeof(T), kWord = 4 / sizeof(T);
  if (fits(kWide)) return rotary_launch<T, kWide>(p, interleaved, in_place, sms, stream);
  if (kWord > 1 && fits(kWord)) return rotary_launch<T, kWord>(p, interleaved, in_place, sms, stream);
  return rotary_launch<T, 1>(p, interleaved, in_place, sms, stream);
}

}  // namespace mkb

using namespace mkb;

extern "C" int mk_rotary(const void* x, long long x_row, long long x_head, void* y, long long y_row,
                         long long y_head, long long rows, int heads, int head_dim, int rotary_dim, int dtype,
                         const void* positions, int pos64, const float* inv_freq, float scale, int interleaved,
                         int inverse, void* stream) {
  if (rows < 0 || heads < 0 || head_dim < 1)
    return set_error(MK_ERR_INVALID, "mk_rotary: bad shape [%lld, %d, %d]", rows, heads, head_dim);
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return set_error(MK_ERR_INVALID, "mk_rotary: rotary_dim=%d must be even and within head_dim=%d", rotary_dim,
                     head_dim);
  if (dtype < MK_BF16 || dtype > MK_FP32) return set_error(MK_ERR_INVALID, "mk_rotary: unknown dtype %d", dtype);
  if (rows == 0 || heads == 0) return MK_OK;
  if (!x || !y || !positions || !inv_freq) return set_error(MK_ERR_INVALID, "mk_rotary: null operand");
  const int size = dtype == MK_FP32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % size != 0 ||
      reinterpret_cast<uintptr_t>(positions) % (pos64 ? 8 : 4) != 0 || reinterpret_cast<uintptr_t>(inv_freq) % 4 != 0)
    return set_error(MK_ERR_INVALID, "mk_rotary: misaligned operand");
  if (x == y && (x_row != y_row || x_head != y_head))
    return set_error(MK_ERR_INVALID, "mk_rotary: in place needs equal strides");
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  RotaryParams p = {};
  p.x = x; p.y = y; p.x_row = x_row; p.x_head = x_head; p.y_row = y_row; p.y_head = y_head;
  p.rows = rows; p.heads = heads; p.head_dim = head_dim; p.rotary_dim = rotary_dim;
  p.sign = inverse ? -1.0f : 1.0f;
  p.rotary.positions = positions; p.rotary.pos64 = pos64 != 0; p.rotary.inv_freq = inv_freq; p.rotary.scale = scale;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool in_place = x == y;
  if (dtype == MK_BF16) return rotary_type<__nv_bfloat16>(p, interleaved != 0, in_place, sms, s);
  if (dtype == MK_FP16) return rotary_type<__half>(p, interleaved != 0, in_place, sms, s);
  return rotary_type<float>(p, interleaved != 0, in_place, sms, s);
}
