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

// Division of an int below 2^31 by a fixed positive int, as a multiplication (Granlund and Montgomery).
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(int divisor) : d((uint32_t)divisor), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct RotaryParams {
  const void* x;
  void* y;
  long long x_row, x_head, y_row, y_head;   // strides in elements
  long long rows;
  int heads, head_dim, rotary_dim;
  int turned;              // slots of a head that turn; the others copy
  int rows_each;           // rows of a CTA
  FastDiv slots, per_row;  // slots of a head; of a row
  float sign;
  RotaryArgs rotary;
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryAhead = 2;      // slots whose loads a thread has in flight
constexpr int kRotaryAngles = 2048;  // of a CTA (16 KB of shared memory)

template <typename T, int P> struct alignas(sizeof(T) * P) RotaryVec { T v[P]; };

// A slot is P pairs of features of a head: vector 0 and vector 1 of P elements each, which are the
// first and second features of the pairs, or, interleaved, the pairs one after another.  A CTA has a few
// whole rows.  Its threads ask for their first slots' features, then work out the rows' angles, each
// once (sine and cosine, in 64 bits up to the turn, cost as much as turning several heads), and
// find them in shared memory for every head.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using Vec = RotaryVec<T, P>;
  __shared__ __align__(16) float2 angles[kRotaryAngles];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long row0 = (long long)blockIdx.x * p.rows_each;
  const int rows = (int)min((long long)p.rows_each, p.rows - row0);
  const uint32_t items = rows * p.per_row.d;
  const int pairs = p.rotary_dim / 2;

  struct Item { const T* x; T* y; int a, b, angle; bool turns, second; };
  auto item = [&](uint32_t e) {
    const uint32_t r = p.per_row.div(e), in_row = e - r * p.per_row.d;
    const uint32_t h = p.slots.div(in_row);
    const int slot = (int)(in_row - h * p.slots.d);
    Item i;
    i.x = static_cast<const T*>(p.x) + (row0 + r) * p.x_row + h * p.x_head;
    i.y = static_cast<T*>(p.y) + (row0 + r) * p.y_row + h * p.y_head;
    i.turns = slot < p.turned;
    i.a = !i.turns ? p.rotary_dim + (slot - p.turned) * 2 * P : INTERLEAVED ? slot * 2 * P : slot * P;
    i.b = i.turns && !INTERLEAVED ? i.a + pairs : i.a + P;
    i.second = i.b < p.head_dim;        // the last vector of a head's copied features may not exist
    i.angle = (int)r * pairs + slot * P;
    return i;
  };
  auto load = [&](uint32_t e, Vec& u, Vec& v) {
    if (e >= items) return;
    const Item i = item(e);
    u = *reinterpret_cast<const Vec*>(i.x + i.a);
    if (i.second) v = *reinterpret_cast<const Vec*>(i.x + i.b);
  };

  Vec u[kRotaryAhead], v[kRotaryAhead];
#pragma unroll
  for (int c = 0; c < kRotaryAhead; ++c) load(threadIdx.x + c * kRotaryThreads, u[c], v[c]);
  for (int e = threadIdx.x; e < rows * pairs; e += kRotaryThreads) {
    const int r = rows == 1 ? 0 : e / pairs;
    float2 cs = rotary_cos_sin(rotary_position(p.rotary, row0 + r), __ldg(p.rotary.inv_freq + (e - r * pairs)),
                               p.rotary.scale);
    cs.y *= p.sign;
    angles[e] = cs;
  }
  __syncthreads();
  for (uint32_t e0 = threadIdx.x; e0 < items; e0 += kRotaryAhead * kRotaryThreads) {
#pragma unroll
    for (int c = 0; c < kRotaryAhead; ++c) {
      const uint32_t e = e0 + c * kRotaryThreads;
      if (e >= items) break;
      const Item i = item(e);
      if (i.turns) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          // pair k: elements k of both vectors, or elements 2 k and 2 k + 1 of the two in a row
          T& first = INTERLEAVED ? (2 * k < P ? u[c].v[2 * k % P] : v[c].v[2 * k % P]) : u[c].v[k];
          T& second = INTERLEAVED ? (2 * k + 1 < P ? u[c].v[(2 * k + 1) % P] : v[c].v[(2 * k + 1) % P]) : v[c].v[k];
          const float2 r = rotary_turn((float)first, (float)second, angles[i.angle + k]);
          first = (T)r.x;
          second = (T)r.y;
        }
      }
      *reinterpret_cast<Vec*>(i.y + i.a) = u[c];
      if (i.second) *reinterpret_cast<Vec*>(i.y + i.b) = v[c];
      load(e + kRotaryAhead * kRotaryThreads, u[c], v[c]);
    }
  }
}

template <typename T, int P>
static int rotary_launch(RotaryParams& p, bool interleaved, bool in_place, int sms, cudaStream_t stream) {
  p.turned = p.rotary_dim / 2 / P;
  const int slots = p.turned + (in_place ? 0 : (p.head_dim - p.rotary_dim + 2 * P - 1) / (2 * P));
  const long long per_row = (long long)p.heads * slots;
  if (per_row > 1 << 30 || p.rotary_dim / 2 > kRotaryAngles)
    return set_error(MK_ERR_INVALID, "mk_rotary: heads of %d (%d turned) features, %d to a row, are too many", p.head_dim,
                     p.rotary_dim, p.heads);
  // Rows of a CTA: enough to give every thread its first slots, and so many that one wave of four CTAs to an
  // SM has them all (8192 rows of 40 heads of 128: 54 us with a CTA to each row, whose latency comes
  // back with every wave); their angles must fit shared memory.
  long long rows_each = kRotaryAhead * kRotaryThreads / per_row;
  const long long wave = (p.rows + 4 * sms - 1) / (4 * sms);
  if (rows_each < wave) rows_each = wave;
  if (rows_each > kRotaryAngles / (p.rotary_dim / 2)) rows_each = kRotaryAngles / (p.rotary_dim / 2);
  if (rows_each < 1) rows_each = 1;
  p.rows_each = (int)rows_each;
  p.slots = FastDiv(slots);
  p.per_row = FastDiv((int)per_row);
  const long long blocks = (p.rows + rows_each - 1) / rows_each;
  if (blocks > 0x7fffffffLL) return set_error(MK_ERR_INVALID, "mk_rotary: %lld rows are too many", p.rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
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
