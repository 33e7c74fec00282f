// Attention over packed token rows, forward and backward (C ABI include/stew_step.h):
//   s_ij = scale q_i.k_j,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - do_i.o_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// over the pairs (i, j) of one sequence inside the window i - left <= j <= i + right.
//
// One warp owns one (token, head): forward and dq walk the token's keys, dk/dv walk the queries
// that see the key, over every query head of its group.  A lane holds head_dim / 32 consecutive
// features (rounded up to 4); all sums are fp32 in registers and in a fixed order.
#include <math.h>

#include <cuda_bf16.h>

#include "common.cuh"
#include "stew_step.h"

namespace nf4b {

constexpr int AT_MAX_DIM = 128;
constexpr int AT_WARPS = 4;

template <typename T>
__device__ __forceinline__ float at_to_f(T v);
template <>
__device__ __forceinline__ float at_to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float at_to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T at_from_f(float v);
template <>
__device__ __forceinline__ __half at_from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 at_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four features of a lane (zeros behind head_dim).
template <typename T>
__device__ __forceinline__ void at_load(const T* row, int lane, int head_dim, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = lane * 4 + i < head_dim ? at_to_f(row[lane * 4 + i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void at_store(T* row, int lane, int head_dim, const float (&f)[4], float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane * 4 + i < head_dim) row[lane * 4 + i] = at_from_f<T>(f[i] * s);
}
__device__ __forceinline__ float at_dot(const float (&a)[4], const float (&b)[4]) {
  float s = fmaf(a[0], b[0], fmaf(a[1], b[1], fmaf(a[2], b[2], a[3] * b[3])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// The sequence [a, b) that holds token t; false behind the last one.  cu's values are clamped
// to [0, tokens], so nothing outside the tensors is ever addressed.
__device__ __forceinline__ bool at_sequence(const nf4b_attn& p, int64_t t, int64_t& a, int64_t& b) {
  auto at = [&](int i) { return i == 0 ? int64_t(0) : max(int64_t(0), min64(p.cu[i], p.tokens)); };
  if (p.rows == 0 || t >= at(p.rows)) return false;
  int lo = 0, hi = p.rows;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at(mid) <= t) lo = mid; else hi = mid;
  }
  a = at(lo);
  b = at(hi);
  return true;
}

template <typename T>
__global__ void __launch_bounds__(32 * AT_WARPS) attn_fwd_kernel(const nf4b_attn p, T* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * AT_WARPS + (threadIdx.x >> 5);
  if (w >= p.tokens * p.heads) return;
  const int64_t t = w / p.heads;
  const int h = int(w - t * p.heads), hk = h / (p.heads / p.kv_heads);
  int64_t a, b;
  float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.f;
  if (at_sequence(p, t, a, b)) {
    float q[4];
    at_load(static_cast<const T*>(p.q) + t * p.q_stride + h * p.q_head_stride, lane, p.head_dim, q);
    const int64_t j0 = p.left < 0 ? a : max(a, t - p.left), j1 = p.right < 0 ? b : min64(b, t + p.right + 1);
    for (int64_t j = j0; j < j1; ++j) {
      float k[4], v[4];
      at_load(static_cast<const T*>(p.k) + j * p.k_stride + hk * p.k_head_stride, lane, p.head_dim, k);
      at_load(static_cast<const T*>(p.v) + j * p.v_stride + hk * p.v_head_stride, lane, p.head_dim, v);
      const float s = at_dot(q, k) * p.scale;
      const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
      const float c = expf(m - mu), e = expf(s - mu);
      l = l * c + e;
      m = mn;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(e, v[i], o[i] * c);
    }
  }
  at_store(out + (t * p.heads + h) * p.head_dim, lane, p.head_dim, o, l == 0.f ? 0.f : 1.f / l);
  if (lane == 0) lse[int64_t(h) * p.tokens + t] = l == 0.f ? -INFINITY : m + logf(l);
}

// dq, and delta_i = do_i.o_i for the dk/dv kernel.
template <typename T>
__global__ void __launch_bounds__(32 * AT_WARPS)
    attn_dq_kernel(const nf4b_attn p, const T* __restrict__ out, const float* __restrict__ lse, const T* __restrict__ dout,
                   T* __restrict__ dq, float* __restrict__ delta) {
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * AT_WARPS + (threadIdx.x >> 5);
  if (w >= p.tokens * p.heads) return;
  const int64_t t = w / p.heads;
  const int h = int(w - t * p.heads), hk = h / (p.heads / p.kv_heads);
  int64_t a, b;
  float g[4] = {0, 0, 0, 0}, dl = 0.f;
  const int64_t off = (t * p.heads + h) * p.head_dim;
  if (at_sequence(p, t, a, b)) {
    float q[4], o[4], d[4];
    at_load(static_cast<const T*>(p.q) + t * p.q_stride + h * p.q_head_stride, lane, p.head_dim, q);
    at_load(out + off, lane, p.head_dim, o);
    at_load(dout + off, lane, p.head_dim, d);
    dl = at_dot(o, d);
    const float le = lse[int64_t(h) * p.tokens + t];
    const int64_t j0 = p.left < 0 ? a : max(a, t - p.left), j1 = p.right < 0 ? b : min64(b, t + p.right + 1);
    for (int64_t j = j0; j < j1; ++j) {
      float k[4], v[4];
      at_load(static_cast<const T*>(p.k) + j * p.k_stride + hk * p.k_head_stride, lane, p.head_dim, k);
      at_load(static_cast<const T*>(p.v) + j * p.v_stride + hk * p.v_head_stride, lane, p.head_dim, v);
      const float e = le == -INFINITY ? 0.f : expf(at_dot(q, k) * p.scale - le);
      const float ds = e * (at_dot(d, v) - dl);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = fmaf(ds, k[i], g[i]);
    }
  }
  at_store(dq + off, lane, p.head_dim, g, p.scale);
  if (lane == 0) delta[int64_t(h) * p.tokens + t] = dl;
}

template <typename T>
__global__ void __launch_bounds__(32 * AT_WARPS)
    attn_dkv_kernel(const nf4b_attn p, const float* __restrict__ lse, const T* __restrict__ dout,
                    const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv) {
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * AT_WARPS + (threadIdx.x >> 5);
  if (w >= p.tokens * p.kv_heads) return;
  const int64_t j = w / p.kv_heads;
  const int hk = int(w - j * p.kv_heads), grp = p.heads / p.kv_heads;
  int64_t a, b;
  float gk[4] = {0, 0, 0, 0}, gv[4] = {0, 0, 0, 0};
  if (at_sequence(p, j, a, b)) {
    float k[4], v[4];
    at_load(static_cast<const T*>(p.k) + j * p.k_stride + hk * p.k_head_stride, lane, p.head_dim, k);
    at_load(static_cast<const T*>(p.v) + j * p.v_stride + hk * p.v_head_stride, lane, p.head_dim, v);
    const int64_t i0 = p.right < 0 ? a : max(a, j - p.right), i1 = p.left < 0 ? b : min64(b, j + p.left + 1);
    for (int h = hk * grp; h < (hk + 1) * grp; ++h) {
      for (int64_t i = i0; i < i1; ++i) {
        float q[4], d[4];
        at_load(static_cast<const T*>(p.q) + i * p.q_stride + h * p.q_head_stride, lane, p.head_dim, q);
        at_load(dout + (i * p.heads + h) * p.head_dim, lane, p.head_dim, d);
        const float le = lse[int64_t(h) * p.tokens + i];
        const float e = le == -INFINITY ? 0.f : expf(at_dot(q, k) * p.scale - le);
        const float ds = e * (at_dot(d, v) - delta[int64_t(h) * p.tokens + i]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          gv[x] = fmaf(e, d[x], gv[x]);
          gk[x] = fmaf(ds, q[x], gk[x]);
        }
      }
    }
  }
  const int64_t off = (j * p.kv_heads + hk) * p.head_dim;
  at_store(dk + off, lane, p.head_dim, gk, p.scale);
  at_store(dv + off, lane, p.head_dim, gv, 1.f);
}

static bool attn_strides_ok(int64_t stride, int64_t head_stride, const nf4b_attn& a, int heads) {
  return (a.tokens == 1 || stride >= a.head_dim) && (heads == 1 || head_stride >= a.head_dim) && stride % 8 == 0 &&
         head_stride % 8 == 0 && stride < (int64_t(1) << 38) && head_stride < (int64_t(1) << 38);
}

// Checks the call and writes its normalised form (window bounds cut to the token count, so that
// index + bound stays in 32 bits).
static int attn_checks(const nf4b_attn* in, nf4b_attn* a) {
  NF4B_RETURN_IF(in == nullptr, NF4B_ERR_INVALID_ARG);
  *a = *in;
  NF4B_RETURN_IF(a->tokens < 0 || a->rows < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->head_dim <= 0,
                 NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(a->heads % a->kv_heads != 0, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!(a->scale > 0.f) || !isfinite(a->scale), NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(a->dtype != NF4B_F16 && a->dtype != NF4B_BF16, NF4B_ERR_UNSUPPORTED);
  NF4B_RETURN_IF(a->head_dim % 8 != 0 || a->head_dim > AT_MAX_DIM, NF4B_ERR_UNSUPPORTED);
  NF4B_RETURN_IF(a->tokens > 0x3FFFFFFF || a->rows > 0x3FFFFFFF || a->heads > 65535, NF4B_ERR_UNSUPPORTED);
  if (a->tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!a->q || !a->k || !a->v || !a->cu, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cu, 4), NF4B_ERR_ALIGNMENT);
  NF4B_RETURN_IF(!attn_strides_ok(a->q_stride, a->q_head_stride, *a, a->heads) ||
                     !attn_strides_ok(a->k_stride, a->k_head_stride, *a, a->kv_heads) ||
                     !attn_strides_ok(a->v_stride, a->v_head_stride, *a, a->kv_heads),
                 NF4B_ERR_ALIGNMENT);
  a->left = a->left < 0 || a->left >= a->tokens ? -1 : a->left;
  a->right = a->right < 0 || a->right >= a->tokens ? -1 : a->right;
  return NF4B_OK;
}

}  // namespace nf4b

using namespace nf4b;

extern "C" int nf4b_attn_fwd(const nf4b_attn* args, void* out, float* lse, void* stream) {
  nf4b_attn a;
  int st = attn_checks(args, &a);
  if (st != NF4B_OK) return st;
  if (a.tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!out || !lse, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(out, 16) || !aligned(lse, 16), NF4B_ERR_ALIGNMENT);
  st = check_device();
  if (st != NF4B_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t warps = a.tokens * a.heads;
  NF4B_RETURN_IF(warps / AT_WARPS >= 0x7FFFFFFF, NF4B_ERR_UNSUPPORTED);
  const unsigned grid = unsigned((warps + AT_WARPS - 1) / AT_WARPS);
  if (a.dtype == NF4B_F16)
    attn_fwd_kernel<__half><<<grid, 32 * AT_WARPS, 0, s>>>(a, static_cast<__half*>(out), lse);
  else
    attn_fwd_kernel<__nv_bfloat16><<<grid, 32 * AT_WARPS, 0, s>>>(a, static_cast<__nv_bfloat16*>(out), lse);
  return launch_status("attn_fwd_kernel launch");
}

extern "C" int64_t nf4b_attn_bwd_work_bytes(int64_t tokens, int32_t rows, int32_t heads, int32_t kv_heads) {
  if (tokens < 0 || rows < 0 || heads <= 0 || kv_heads <= 0 || tokens > 0x3FFFFFFF || rows > 0x3FFFFFFF ||
      heads > 65535 || heads % kv_heads != 0)
    return -1;
  return (tokens * heads * 4 + 15) / 16 * 16;
}

template <typename T>
static int attn_bwd_launch(const nf4b_attn& a, const void* out, const float* lse, const void* dout, void* dq, void* dk,
                           void* dv, float* delta, cudaStream_t s) {
  const unsigned gq = unsigned((a.tokens * a.heads + AT_WARPS - 1) / AT_WARPS);
  const unsigned gk = unsigned((a.tokens * a.kv_heads + AT_WARPS - 1) / AT_WARPS);
  attn_dq_kernel<T><<<gq, 32 * AT_WARPS, 0, s>>>(a, static_cast<const T*>(out), lse, static_cast<const T*>(dout),
                                                 static_cast<T*>(dq), delta);
  attn_dkv_kernel<T><<<gk, 32 * AT_WARPS, 0, s>>>(a, lse, static_cast<const T*>(dout), delta, static_cast<T*>(dk),
                                                  static_cast<T*>(dv));
  return launch_status("attn backward launch");
}

extern "C" int nf4b_attn_bwd(const nf4b_attn* args, const void* out, const float* lse, const void* dout, void* dq,
                             void* dk, void* dv, void* work, int64_t work_bytes, void* stream) {
  nf4b_attn a;
  int st = attn_checks(args, &a);
  if (st != NF4B_OK) return st;
  if (a.tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!out || !lse || !dout || !dq || !dk || !dv || !work, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(out, 16) || !aligned(lse, 16) || !aligned(dout, 16) || !aligned(dq, 16) || !aligned(dk, 16) ||
                     !aligned(dv, 16) || !aligned(work, 16),
                 NF4B_ERR_ALIGNMENT);
  const int64_t need = nf4b_attn_bwd_work_bytes(a.tokens, a.rows, a.heads, a.kv_heads);
  NF4B_RETURN_IF(need < 0, NF4B_ERR_UNSUPPORTED);
  NF4B_RETURN_IF(work_bytes < need, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(a.tokens * a.heads / AT_WARPS >= 0x7FFFFFFF, NF4B_ERR_UNSUPPORTED);
  st = check_device();
  if (st != NF4B_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* delta = static_cast<float*>(work);
  return a.dtype == NF4B_F16 ? attn_bwd_launch<__half>(a, out, lse, dout, dq, dk, dv, delta, s)
                             : attn_bwd_launch<__nv_bfloat16>(a, out, lse, dout, dq, dk, dv, delta, s);
}
