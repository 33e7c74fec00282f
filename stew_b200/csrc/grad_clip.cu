// Global 2-norm of a list of gradients and clipping (C ABI include/stew_step.h):
//   norm = sqrt(sum src^2) / |divisor|,   dst = src (1 / divisor) min(1, max_norm / (norm + 1e-6))
//
// Two launches: the list is cut into chunks of 16 KB, every CTA takes a contiguous run of them.  The first
// launch writes one 64-bit sum of squares per CTA; every CTA of the second adds those sums up in the same
// order (so all of them use the same bits), forms the factor and scales its run.  The tensors' pointers
// travel in the kernel's parameters, so a call needs no copy to the device and can be captured; longer lists
// take several launches.
//
// Bound by memory: the list is read twice and written once (a list under the limit, in place, is read
// once).  187 M bf16 values, out of place: 190 us, 5.9 TB/s of 6.5 measured for a copy.  Scaling from the
// end of each run (to find what the first launch read last in the L2), stores that leave the L2 first and
// fetching a chunk ahead all measured the same.  A step's 112 adapters (8.7 MB fp32, in the L2): 8.5 us.
//
// Squares are summed in 64 bits: a 32-bit sum overflows from |g| = 1.8e19 and drifts over a long
// list.  A 16-bit value's square is exact in 32 bits, so two of them are added there (one
// rounding, 2^-24) and the pair goes to the 64-bit sum, where no square can over- or underflow
// (vectors outside [2^-50, 2^60) take 64 bits from the start): half the 64-bit conversions.
#include <math.h>

#include <type_traits>

#include <cuda_bf16.h>

#include "common.cuh"
#include "stew_step.h"

namespace nf4b {

constexpr int GC_SMALL = 64;       // gradients of a launch: 2 KB of kernel parameters,
constexpr int GC_LARGE = 512;      // or 16 KB
constexpr int GC_CHUNK = 16384;    // bytes of one chunk
constexpr int GC_THREADS = 256;
constexpr int GC_VECS = GC_CHUNK / 16 / GC_THREADS;  // 16-byte loads a thread has in flight
// CTAs of a launch: what fits on the 148 SMs at once (the scaling kernel keeps more in registers)
constexpr int GC_NORM_CTAS = 148 * 4, GC_SCALE_CTAS = 148 * 3;

struct GcItem {
  const void* src;
  void* dst;
  int64_t numel;
  int32_t dtype;
  int32_t chunk0;  // chunks of the gradients before this one
};
template <int CAP>
struct GcList {
  GcItem it[CAP];
  int32_t n, chunks;
};

// The gradient that holds chunk c.
template <int CAP>
__device__ __forceinline__ int gc_find(const GcList<CAP>& l, int c) {
  int lo = 0, hi = l.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.it[mid].chunk0 <= c) lo = mid; else hi = mid;
  }
  return lo;
}

// This CTA's run of chunks.
__device__ __forceinline__ int gc_first(int chunks, unsigned cta) { return int(int64_t(chunks) * cta / gridDim.x); }

template <typename T>
__device__ __forceinline__ float gc_to_f(T v);
template <>
__device__ __forceinline__ float gc_to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float gc_to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float gc_to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T gc_from_f(float v);
template <>
__device__ __forceinline__ float gc_from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half gc_from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 gc_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Squares of one 16-byte vector.
template <typename T>
__device__ __forceinline__ double gc_squares(uint4 v) {
  constexpr int V = 16 / sizeof(T);
  const T* x = reinterpret_cast<const T*>(&v);
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = gc_to_f(x[i]);
  double acc = 0.0;
  bool pairs = sizeof(T) == 2;
  if (sizeof(T) == 2) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, fabsf(f[i]));
    pairs = m == 0.f || (m >= 0x1p-50f && m < 0x1p60f);
  }
  if (pairs) {  // (a NaN beside finite values stays in the sums)
#pragma unroll
    for (int i = 0; i < V; i += 2) acc += double(fmaf(f[i], f[i], f[i + 1] * f[i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) acc = fma(double(f[i]), double(f[i]), acc);
  }
  return acc;
}

// Values before the next 16-byte boundary of p (at most n).
template <typename T>
__device__ __forceinline__ int gc_head(const T* p, int n) {
  return min(n, int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / int(sizeof(T)));
}

// Squares of n values (at most a chunk): whole vectors between the 16-byte boundaries, the few
// values outside them one by one.
template <typename T>
__device__ __forceinline__ double gc_norm_chunk(const T* p, int n) {
  constexpr int V = 16 / sizeof(T);
  const int head = gc_head(p, n), nv = (n - head) / V;
  const uint4* body = reinterpret_cast<const uint4*>(p + head);
  uint4 v[GC_VECS];
#pragma unroll
  for (int k = 0; k < GC_VECS; ++k) {
    const int i = threadIdx.x + k * GC_THREADS;
    v[k] = i < nv ? body[i] : make_uint4(0, 0, 0, 0);
  }
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < GC_VECS; ++k) acc += gc_squares<T>(v[k]);
  const int rest = n - nv * V;
  if (threadIdx.x < rest) {
    const double x = gc_to_f(p[threadIdx.x < head ? threadIdx.x : threadIdx.x + nv * V]);
    acc = fma(x, x, acc);
  }
  return acc;
}

template <typename T>
__device__ __forceinline__ void gc_scale_chunk(const T* src, T* dst, int n, float f) {
  constexpr int V = 16 / sizeof(T);
  if (((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) != 0) {
    // boundaries that do not coincide: one value at a time
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += GC_THREADS) dst[i] = gc_from_f<T>(gc_to_f(src[i]) * f);
    return;
  }
  const int head = gc_head(src, n), nv = (n - head) / V;
  const uint4* from = reinterpret_cast<const uint4*>(src + head);
  uint4* to = reinterpret_cast<uint4*>(dst + head);
  uint4 v[GC_VECS];
#pragma unroll
  for (int k = 0; k < GC_VECS; ++k) {
    const int i = threadIdx.x + k * GC_THREADS;
    if (i < nv) v[k] = from[i];
  }
#pragma unroll
  for (int k = 0; k < GC_VECS; ++k) {
    const int i = threadIdx.x + k * GC_THREADS;
    T* x = reinterpret_cast<T*>(&v[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = gc_from_f<T>(gc_to_f(x[e]) * f);
    if (i < nv) to[i] = v[k];
  }
  const int rest = n - nv * V;
  if (threadIdx.x < rest) {
    const int i = threadIdx.x < head ? threadIdx.x : threadIdx.x + nv * V;
    dst[i] = gc_from_f<T>(gc_to_f(src[i]) * f);
  }
}

// The same with a factor that fp32 holds only with less precision, or not at all.
template <typename T>
__device__ __forceinline__ void gc_scale_chunk_wide(const T* src, T* dst, int n, double f) {
  for (int i = threadIdx.x; i < n; i += GC_THREADS) dst[i] = gc_from_f<T>(float(double(gc_to_f(src[i])) * f));
}

// Calls f(typed src, typed dst, count) for chunk c of gradient `it`.
template <typename F>
__device__ __forceinline__ void gc_chunk(const GcItem& it, int c, F f) {
  auto go = [&](auto* tag) {
    using T = typename std::remove_pointer<decltype(tag)>::type;
    constexpr int64_t N = GC_CHUNK / sizeof(T);
    const int64_t i0 = int64_t(c - it.chunk0) * N;
    T* dst = static_cast<T*>(it.dst);
    f(static_cast<const T*>(it.src) + i0, dst == nullptr ? nullptr : dst + i0, int(min64(N, it.numel - i0)));
  };
  if (it.dtype == NF4B_F32) go(static_cast<float*>(nullptr));
  else if (it.dtype == NF4B_F16) go(static_cast<__half*>(nullptr));
  else go(static_cast<__nv_bfloat16*>(nullptr));
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

template <int CAP>
__global__ void __launch_bounds__(GC_THREADS, GC_NORM_CTAS / 148)
    grad_norm_kernel(const __grid_constant__ GcList<CAP> l, double* __restrict__ part) {
  grid_dep_wait();  // programmatic launch: no global access before the wait
  double acc = 0.0;
  const int c0 = gc_first(l.chunks, blockIdx.x), c1 = gc_first(l.chunks, blockIdx.x + 1);
  int g = c0 < c1 ? gc_find(l, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    while (g + 1 < l.n && l.it[g + 1].chunk0 <= c) ++g;
    gc_chunk(l.it[g], c, [&](auto* src, auto*, int n) { acc += gc_norm_chunk(src, n); });
  }
  acc = gc_cta_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int CAP>
__global__ void __launch_bounds__(GC_THREADS, GC_SCALE_CTAS / 148)
    grad_scale_kernel(const __grid_constant__ GcList<CAP> l, const double* __restrict__ part, int parts, float max_norm,
                      const float* __restrict__ divisor, float* __restrict__ norm_out) {
  grid_dep_wait();  // programmatic launch: no global access before the wait
  __shared__ double s_factor;
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += GC_THREADS) acc += part[i];
  acc = gc_cta_sum(acc);
  if (threadIdx.x == 0) {
    const double div = divisor ? double(*divisor) : 1.0;
    const double norm = sqrt(acc) / fabs(div);
    const double q = double(max_norm) / (norm + 1e-6);
    s_factor = (q >= 1.0 ? 1.0 : q) / div;  // a NaN norm stays one
    if (blockIdx.x == 0 && norm_out) *norm_out = float(norm);
  }
  __syncthreads();
  const double wide = s_factor;
  const float f = float(wide);
  // outside fp32's normal range (gradients of 1e30 and a limit of 1e-10, a divisor of 1e-39) the results may still
  // be inside
  const bool normal = wide == 0.0 || !(fabs(wide) < 0x1p-126 || (isinf(f) && !isinf(wide)));
  const int c0 = gc_first(l.chunks, blockIdx.x), c1 = gc_first(l.chunks, blockIdx.x + 1);
  int g = c0 < c1 ? gc_find(l, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    while (g + 1 < l.n && l.it[g + 1].chunk0 <= c) ++g;
    const GcItem& it = l.it[g];
    if (it.dst == nullptr || (it.dst == it.src && f == 1.f)) continue;
    gc_chunk(it, c, [&](auto* src, auto* dst, int n) {
      if (normal) gc_scale_chunk(src, dst, n, f);
      else gc_scale_chunk_wide(src, dst, n, wide);
    });
  }
}

// One pass over the list, in launches of up to CAP gradients: pass 0 measures, pass 1 scales.
template <int CAP>
static int gc_pass(int pass, const nf4b_grad* grads, int n, float max_norm, const float* divisor, float* norm, double* part,
                   int* parts, cudaStream_t s) {
  GcList<CAP> l;
  int at = 0, done = 0;
  do {
    l.n = 0;
    int64_t chunks = 0;
    for (; at < n && l.n < CAP; ++at) {
      const nf4b_grad& g = grads[at];
      if (g.numel == 0) continue;
      l.it[l.n++] = GcItem{g.src, g.dst, g.numel, g.dtype, int32_t(chunks)};
      const int64_t per = GC_CHUNK / (g.dtype == NF4B_F32 ? 4 : 2);
      chunks += (g.numel + per - 1) / per;
      NF4B_RETURN_IF(chunks > 0x7FFFFFFF, NF4B_ERR_UNSUPPORTED);
    }
    l.chunks = int32_t(chunks);
    const int64_t most = pass == 0 ? GC_NORM_CTAS : GC_SCALE_CTAS;
    const unsigned grid = unsigned(chunks < 1 ? 1 : (chunks < most ? chunks : most));
    if (pass == 0) {
      NF4B_CUDA_TRY(launch_pdl(grad_norm_kernel<CAP>, dim3(grid), dim3(GC_THREADS), size_t(0), s, l, part + *parts));
      *parts += int(grid);
    } else {
      NF4B_CUDA_TRY(launch_pdl(grad_scale_kernel<CAP>, dim3(grid), dim3(GC_THREADS), size_t(0), s, l, part, *parts,
                               max_norm, divisor, done++ == 0 ? norm : nullptr));
    }
    const int st = launch_status("gradient clipping launch");
    if (st != NF4B_OK) return st;
  } while (at < n);
  return NF4B_OK;
}

}  // namespace nf4b

using namespace nf4b;

extern "C" int64_t nf4b_clip_grads_work_bytes(int32_t n) {
  if (n < 0) return -1;
  return (int64_t(n) / GC_LARGE + 1) * GC_NORM_CTAS * 8;
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
  int parts = 0;
  for (int pass = 0; pass < 2; ++pass) {
    st = n <= GC_SMALL ? gc_pass<GC_SMALL>(pass, grads, n, max_norm, divisor, norm, part, &parts, s)
                       : gc_pass<GC_LARGE>(pass, grads, n, max_norm, divisor, norm, part, &parts, s);
    if (st != NF4B_OK) return st;
  }
  return NF4B_OK;
}
