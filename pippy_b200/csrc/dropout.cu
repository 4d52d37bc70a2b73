// Dropout whose mask is computed from (seed, stream, element) in the forward and again in the backward: it is never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds turn a
// 128-bit counter and a 64-bit key into four 32-bit numbers.  Here the key is the seed and the counter is (element / 8,
// stream); a block's eight 16-bit halves, low half first, decide eight consecutive elements: an element stays if its
// number is at least `threshold`, so the probability is threshold / 65536 exactly and the factor 65536 / (65536 - threshold)
// keeps the expectation.  16 bits instead of 32 halve the arithmetic, which would otherwise be what bounds the kernel.
// Bound by bandwidth: 8192 x 4096 elements with residual 35 us, 5.8 TB/s; the backward, 4 bytes an element, 31.  Two groups of eight
// elements in flight in a thread took 37 and 32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

extern "C" void pb_count_launch(int n);

namespace pbd {

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

struct Args {
  const __nv_bfloat16* x;
  const __nv_bfloat16* residual;  // null: none
  __nv_bfloat16* y;
  long long n;
  const unsigned long long* seed_ptr;  // null: `seed`
  unsigned long long seed, stream;
  unsigned threshold;
  float factor;
};

// y = (residual +) (stays ? x * factor : 0), summed in fp32 and rounded once.  kVec: 16-byte accesses; the last, partial
// group of eight elements and unaligned tensors take the element-wise form.
template <bool kRes, bool kVec>
__global__ void __launch_bounds__(256) dropout_kernel(Args a) {
  const unsigned long long seed = a.seed_ptr ? *a.seed_ptr : a.seed;
  const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
  const long long groups = (a.n + 7) / 8;
  for (long long g = blockIdx.x * (long long)blockDim.x + threadIdx.x; g < groups; g += (long long)gridDim.x * blockDim.x) {
    const long long first = g * 8;
    const bool whole = kVec && first + 8 <= a.n;
    uint4 xv = make_uint4(0, 0, 0, 0), rv = xv;
    if (whole) {
      xv = __ldg(reinterpret_cast<const uint4*>(a.x + first));
      if (kRes) rv = __ldg(reinterpret_cast<const uint4*>(a.residual + first));
    }
    const uint4 w = philox(make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)a.stream, (uint32_t)(a.stream >> 32)), key);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    if (whole) {
      const __nv_bfloat162* xb = reinterpret_cast<const __nv_bfloat162*>(&xv);
      const __nv_bfloat162* rb = reinterpret_cast<const __nv_bfloat162*>(&rv);
      uint4 out;
      __nv_bfloat162* ob = reinterpret_cast<__nv_bfloat162*>(&out);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(xb[i]);
        float lo = (word[i] & 0xffffu) >= a.threshold ? f.x * a.factor : 0.f;
        float hi = (word[i] >> 16) >= a.threshold ? f.y * a.factor : 0.f;
        if (kRes) {
          const float2 r = __bfloat1622float2(rb[i]);
          lo += r.x;
          hi += r.y;
        }
        ob[i] = __floats2bfloat162_rn(lo, hi);
      }
      *reinterpret_cast<uint4*>(a.y + first) = out;
    } else {
      for (int e = 0; e < 8 && first + e < a.n; ++e) {
        const uint32_t number = (word[e >> 1] >> ((e & 1) * 16)) & 0xffffu;
        float v = number >= a.threshold ? __bfloat162float(a.x[first + e]) * a.factor : 0.f;
        if (kRes) v += __bfloat162float(a.residual[first + e]);
        a.y[first + e] = __float2bfloat16_rn(v);
      }
    }
  }
}

}  // namespace pbd

extern "C" {

// x, residual (may be null), y: n contiguous bf16 values.  threshold 0..65535: an element is dropped with probability
// threshold / 65536.  seed_ptr (device, 8 bytes) takes precedence over `seed`.
int pb_dropout(const void* x, const void* residual, void* y, long long n, const long long* seed_ptr, long long seed,
               long long stream_id, int threshold, void* stream_) {
  using namespace pbd;
  if (n < 0 || threshold < 0 || threshold > 65535) return -1;
  if (n == 0) return 0;
  Args a;
  a.x = reinterpret_cast<const __nv_bfloat16*>(x);
  a.residual = reinterpret_cast<const __nv_bfloat16*>(residual);
  a.y = reinterpret_cast<__nv_bfloat16*>(y);
  a.n = n;
  a.seed_ptr = reinterpret_cast<const unsigned long long*>(seed_ptr);
  a.seed = (unsigned long long)seed;
  a.stream = (unsigned long long)stream_id;
  a.threshold = (unsigned)threshold;
  a.factor = 65536.f / (float)(65536 - threshold);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  long long blocks = ((n + 7) / 8 + 255) / 256;
  if (blocks > 148 * 32) blocks = 148 * 32;
  const unsigned grid = (unsigned)blocks;
  if (residual) {
    if (vec) dropout_kernel<true, true><<<grid, 256, 0, stream>>>(a);
    else dropout_kernel<true, false><<<grid, 256, 0, stream>>>(a);
  } else {
    if (vec) dropout_kernel<false, true><<<grid, 256, 0, stream>>>(a);
    else dropout_kernel<false, false><<<grid, 256, 0, stream>>>(a);
  }
  pb_count_launch(1);
  return (int)cudaGetLastError();
}

}  // extern "C"
