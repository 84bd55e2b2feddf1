// Rotary positions on rows of heads: y = x with the first rotary_dim features of every head turned by
// position * inv_freq.  Nothing but one read and one write of every element, so bound by memory.
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
  int slots, turned;       // of a row; the first `turned` turn, the rest copy
  int heads_each;          // heads that a thread walks
  float sign;
  RotaryArgs rotary;
};

constexpr int kRotaryThreads = 128;
constexpr int kRotaryAhead = 4;   // heads whose loads a thread has in flight

template <typename T, int P> struct alignas(sizeof(T) * P) RotaryVec { T v[P]; };

// A slot is P pairs of features: vector 0 and vector 1 of P elements each, which are the first and
// second features of the pairs, or, interleaved, the pairs one after another.  A thread has a slot
// of a row, takes its P angles once and walks heads_each heads; neighbouring threads have
// neighbouring slots.  Angles cost P sines and cosines (in 64 bits up to the turn), so the more heads
// share them the better, as long as there are enough threads to keep memory busy.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using Vec = RotaryVec<T, P>;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const unsigned long long e = (unsigned long long)blockIdx.x * kRotaryThreads + threadIdx.x;
  const unsigned long long total = (unsigned long long)p.rows * p.slots;
  if (e >= total) return;
  long long row;
  int slot;
  if (total <= 0xffffffffu) {
    row = (uint32_t)e / (uint32_t)p.slots;
    slot = (int)((uint32_t)e % (uint32_t)p.slots);
  } else {
    row = (long long)(e / p.slots);
    slot = (int)(e % p.slots);
  }
  const int h0 = blockIdx.y * p.heads_each;
  const int heads = min(p.heads_each, p.heads - h0);
  const T* x = static_cast<const T*>(p.x) + row * p.x_row + (long long)h0 * p.x_head;
  T* y = static_cast<T*>(p.y) + row * p.y_row + (long long)h0 * p.y_head;

  if (slot >= p.turned) {   // features that are copied; the last vector may not exist
    const int at = p.rotary_dim + (slot - p.turned) * 2 * P;
    const bool two = at + P < p.head_dim;
#pragma unroll kRotaryAhead
    for (int h = 0; h < heads; ++h, x += p.x_head, y += p.y_head) {
      *reinterpret_cast<Vec*>(y + at) = *reinterpret_cast<const Vec*>(x + at);
      if (two) *reinterpret_cast<Vec*>(y + at + P) = *reinterpret_cast<const Vec*>(x + at + P);
    }
    return;
  }
  const int a = INTERLEAVED ? slot * 2 * P : slot * P;
  const int b = INTERLEAVED ? a + P : a + p.rotary_dim / 2;
  float2 cs[P];
  const long long position = rotary_position(p.rotary, row);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    cs[i] = rotary_cos_sin(position, __ldg(p.rotary.inv_freq + slot * P + i), p.rotary.scale);
    cs[i].y *= p.sign;
  }
  for (int h = 0; h < heads; h += kRotaryAhead) {
    Vec u[kRotaryAhead], v[kRotaryAhead];
#pragma unroll
    for (int i = 0; i < kRotaryAhead; ++i)
      if (h + i < heads) {
        u[i] = *reinterpret_cast<const Vec*>(x + i * p.x_head + a);
        v[i] = *reinterpret_cast<const Vec*>(x + i * p.x_head + b);
      }
#pragma unroll
    for (int i = 0; i < kRotaryAhead; ++i)
      if (h + i < heads) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          // pair k: elements k of both vectors, or elements 2 k and 2 k + 1 of the two in a row
          T& first = INTERLEAVED ? (2 * k < P ? u[i].v[2 * k % P] : v[i].v[2 * k % P]) : u[i].v[k];
          T& second = INTERLEAVED ? (2 * k + 1 < P ? u[i].v[(2 * k + 1) % P] : v[i].v[(2 * k + 1) % P]) : v[i].v[k];
          const float2 r = rotary_turn((float)first, (float)second, cs[k]);
          first = (T)r.x;
          second = (T)r.y;
        }
        *reinterpret_cast<Vec*>(y + i * p.y_head + a) = u[i];
        *reinterpret_cast<Vec*>(y + i * p.y_head + b) = v[i];
      }
    x += kRotaryAhead * p.x_head;
    y += kRotaryAhead * p.y_head;
  }
}

template <typename T, int P>
static int rotary_launch(RotaryParams& p, bool interleaved, bool in_place, int sms, cudaStream_t stream) {
  p.turned = p.rotary_dim / 2 / P;
  p.slots = p.turned + (in_place ? 0 : (p.head_dim - p.rotary_dim + 2 * P - 1) / (2 * P));
  // As many heads to a thread as leave 512 threads to an SM: 8192 rows of 40 heads of 128 share an angle
  // among all 40, one token's are taken by a thread each.
  const long long threads = p.rows * p.slots;
  long long parts = (512LL * sms + threads - 1) / threads;
  if (parts > p.heads) parts = p.heads;
  p.heads_each = (int)((p.heads + parts - 1) / parts);
  parts = (p.heads + p.heads_each - 1) / p.heads_each;
  const long long blocks = (threads + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > 0x7fffffffLL || parts > 65535)
    return set_error(MK_ERR_INVALID, "mk_rotary: %lld rows of %d heads are too many", p.rows, p.heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)parts, 1);
  cfg.blockDim = dim3(kRotaryThreads, 1, 1);
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
