// Global 2-norm of a list of gradients and clipping (C ABI include/stew_step.h):
//   norm = sqrt(sum src^2) / divisor,   dst = src (1 / divisor) min(1, max_norm / (norm + 1e-6))
//
// Two launches over the same work split: the list is cut into chunks of GC_CHUNK values, chunk c
// goes to CTA c mod grid.  The first writes one 64-bit sum of squares per CTA; every CTA of the
// second adds those sums up in the same order (so all of them use the same bits), forms the
// factor and scales its chunks.  The tensors' pointers travel in the kernel's parameters, so a
// call needs no copy to the device and can be captured; longer lists take several launches.
// The squares are summed in 64 bits: a 32-bit sum overflows from |g| = 1.8e19 and loses the small
// gradients of a long list.
#include <math.h>

#include <cuda_bf16.h>

#include "common.cuh"
#include "stew_step.h"

namespace nf4b {

constexpr int GC_MAX = 512;        // gradients of one launch (16 KB of kernel parameters)
constexpr int GC_CHUNK = 4096;     // values of one unit of work
constexpr int GC_THREADS = 256;
constexpr int GC_MAX_CTAS = 148 * 4;

struct GcItem {
  const void* src;
  void* dst;
  int64_t numel;
  int32_t dtype;
  int32_t chunk0;  // chunks of the gradients before this one
};
struct GcList {
  GcItem it[GC_MAX];
  int32_t n, chunks;
};

// The gradient that holds chunk c.
__device__ __forceinline__ int gc_find(const GcList& l, int c) {
  int lo = 0, hi = l.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.it[mid].chunk0 <= c) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float gc_get(const void* p, int64_t i, int dt) {
  if (dt == NF4B_F32) return static_cast<const float*>(p)[i];
  if (dt == NF4B_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void gc_put(void* p, int64_t i, int dt, float v) {
  if (dt == NF4B_F32) static_cast<float*>(p)[i] = v;
  else if (dt == NF4B_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// The CTA's sum, in a fixed order, in thread 0.
__device__ __forceinline__ double gc_cta_sum(double v) {
  __shared__ double s[GC_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < GC_THREADS / 32; ++i) t += s[i];
  return t;
}

__global__ void __launch_bounds__(GC_THREADS) grad_norm_kernel(const __grid_constant__ GcList l, double* __restrict__ part) {
  double acc = 0.0;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const GcItem& it = l.it[gc_find(l, c)];
    const int64_t i0 = int64_t(c - it.chunk0) * GC_CHUNK, i1 = min64(it.numel, i0 + GC_CHUNK);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += GC_THREADS) {
      const double v = gc_get(it.src, i, it.dtype);
      acc = fma(v, v, acc);
    }
  }
  acc = gc_cta_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(GC_THREADS)
    grad_scale_kernel(const __grid_constant__ GcList l, const double* __restrict__ part, int parts, float max_norm,
                      const float* __restrict__ divisor, float* __restrict__ norm_out) {
  __shared__ float s_factor;
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += GC_THREADS) acc += part[i];
  acc = gc_cta_sum(acc);
  if (threadIdx.x == 0) {
    const double div = divisor ? double(*divisor) : 1.0;
    const double norm = sqrt(acc) / fabs(div);
    const double q = double(max_norm) / (norm + 1e-6);
    s_factor = float((q >= 1.0 ? 1.0 : q) / div);  // a NaN norm stays one
    if (blockIdx.x == 0 && norm_out) *norm_out = float(norm);
  }
  __syncthreads();
  const float f = s_factor;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const GcItem& it = l.it[gc_find(l, c)];
    if (it.dst == nullptr || (it.dst == it.src && f == 1.f)) continue;
    const int64_t i0 = int64_t(c - it.chunk0) * GC_CHUNK, i1 = min64(it.numel, i0 + GC_CHUNK);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += GC_THREADS)
      gc_put(it.dst, i, it.dtype, gc_get(it.src, i, it.dtype) * f);
  }
}

}  // namespace nf4b

using namespace nf4b;

extern "C" int64_t nf4b_clip_grads_work_bytes(int32_t n) {
  if (n < 0) return -1;
  return (int64_t(n) / GC_MAX + 1) * GC_MAX_CTAS * 8;
}

extern "C" int nf4b_clip_grads(const nf4b_grad* grads, int32_t n, float max_norm, const float* divisor, float* norm,
                               void* work, int64_t work_bytes, void* stream) {
  NF4B_RETURN_IF(n < 0 || !(max_norm >= 0.f), NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!norm || !work || (n > 0 && !grads), NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(work, 8) || !aligned(norm, 4) || !aligned(divisor, 4), NF4B_ERR_ALIGNMENT);
  NF4B_RETURN_IF(work_bytes < nf4b_clip_grads_work_bytes(n), NF4B_ERR_INVALID_ARG);
  for (int i = 0; i < n; ++i) {
    const nf4b_grad& g = grads[i];
    NF4B_RETURN_IF(g.numel < 0 || (g.numel > 0 && !g.src), NF4B_ERR_INVALID_ARG);
    NF4B_RETURN_IF(g.dtype != NF4B_F32 && g.dtype != NF4B_F16 && g.dtype != NF4B_BF16, NF4B_ERR_UNSUPPORTED);
    NF4B_RETURN_IF(g.numel > (int64_t(1) << 40), NF4B_ERR_UNSUPPORTED);
    const uintptr_t al = g.dtype == NF4B_F32 ? 4 : 2;
    NF4B_RETURN_IF(!aligned(g.src, al) || !aligned(g.dst, al), NF4B_ERR_ALIGNMENT);
  }
  int st = check_device();
  if (st != NF4B_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  double* part = static_cast<double*>(work);
  GcList l;
  int parts = 0;
  // pass 0 measures, pass 1 scales: the same lists, so the same split
  for (int pass = 0; pass < 2; ++pass) {
    int at = 0;
    int first = 0;
    do {
      l.n = 0;
      int64_t chunks = 0;
      for (; at < n && l.n < GC_MAX; ++at) {
        const nf4b_grad& g = grads[at];
        if (g.numel == 0) continue;
        l.it[l.n++] = GcItem{g.src, g.dst, g.numel, g.dtype, int32_t(chunks)};
        chunks += (g.numel + GC_CHUNK - 1) / GC_CHUNK;
        NF4B_RETURN_IF(chunks > 0x7FFFFFFF, NF4B_ERR_UNSUPPORTED);
      }
      l.chunks = int32_t(chunks);
      const unsigned grid = unsigned(chunks < 1 ? 1 : (chunks < GC_MAX_CTAS ? chunks : GC_MAX_CTAS));
      if (pass == 0) {
        grad_norm_kernel<<<grid, GC_THREADS, 0, s>>>(l, part + parts);
        parts += int(grid);
      } else {
        grad_scale_kernel<<<grid, GC_THREADS, 0, s>>>(l, part, parts, max_norm, divisor, first++ == 0 ? norm : nullptr);
      }
      st = launch_status("gradient clipping launch");
      if (st != NF4B_OK) return st;
    } while (at < n);
  }
  return NF4B_OK;
}
