// Attention over packed token rows, forward and backward (C ABI include/stew_step.h):
//   s_ij = scale q_i.k_j,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - do_i.o_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// over the pairs (i, j) of one sequence inside the window i - left <= j <= i + right.
//
// One warp owns one (token, head): forward and dq walk the token's keys, dk/dv walk the queries
// that see the key, over every query head of its group.  A lane holds head_dim / 32 consecutive
// features (rounded up to 4); all sums are fp32 in registers and in a fixed order.
#include <mutex>

#include "attn_common.cuh"

namespace nf4b {

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

// ------------------------------------------------------------------- forward
// One CTA per (128-token query tile, head); two CTAs on an SM, so one's softmax runs beside the
// other's MMAs.  The scores S = Q K^T and the output O live in TMEM (128 + 64 DC columns), the
// probabilities overwrite the scores as 16-bit values and are the A operand of P V straight from
// TMEM; Q, K and V are TMA tiles in shared memory (V's is read as an MN-major operand, so nothing
// is transposed).
//   warps 0-3  softmax: one thread per query row
//   warp 4     TMA: Q, then K and V tiles through a ring of AT_RING slots
//   warp 5     TMEM allocation, MMA issue
// One pass over the keys with a running maximum m and sum l (Milakov and Gimelshein's online
// softmax); O is rescaled only when the maximum has grown by more than 2^8, else P may exceed 1
// (by at most 2^8, far inside fp16's range) and l with it -- the quotient is the same.
template <int DC>
struct AttnFwdSmem {
  static constexpr int TILE = DC * AT_BOX;
  static constexpr int RING = DC == 1 ? 4 : 2;
  static constexpr int Q = 0;
  static constexpr int KV = TILE;
  static constexpr int BAR = KV + RING * TILE;
  // full[RING], empty[RING], q_full, s_full, p_ready, o_full, staged
  static constexpr int NBAR = 2 * RING + 5;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int ALLOC = MISC + 16 + 1024;  // slack to align the base to 1024 B
};
constexpr int AT_FWD_THREADS = 192;
constexpr float AT_LAZY = 8.f;  // log2 growth of the maximum that O tolerates unscaled

template <typename T, int DC>
__global__ void __launch_bounds__(AT_FWD_THREADS, 2)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p, T* __restrict__ out,
                    float* __restrict__ lse) {
  using L = AttnFwdSmem<DC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* empty = full + L::RING;
  uint64_t* q_full = empty + L::RING;
  uint64_t* s_full = q_full + 1;
  uint64_t* p_ready = s_full + 1;
  uint64_t* o_full = p_ready + 1;
  uint64_t* staged = o_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  grid_dep_wait();  // programmatic launch: no global access before the wait
  // the last slots first: a causal sequence's last tiles see the most keys
  const int slot = p.slots - 1 - int(blockIdx.x / p.heads);
  const int h = blockIdx.x % p.heads, hk = h / (p.heads / p.kv_heads);
  const AttnTile t = at_find(p, slot);
  if (t.i0 >= t.len) return;
  if (t.tail) {
    const int n = min(AT_TILE, t.len - t.i0), vec = p.head_dim / 8;
    for (int i = threadIdx.x; i < n * vec; i += AT_FWD_THREADS) {
      const int64_t row = t.a + t.i0 + i / vec;
      *reinterpret_cast<uint4*>(out + (row * p.heads + h) * p.head_dim + (i % vec) * 8) = make_uint4(0, 0, 0, 0);
    }
    if (threadIdx.x < n) lse[int64_t(h) * p.tokens + t.a + t.i0 + threadIdx.x] = -INFINITY;
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::RING; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(s_full, 1);
    mbar_init(p_ready, 128);
    mbar_init(o_full, 1);
    mbar_init(staged, 1);
    fence_barrier_init();
    *abort_flag = 0;
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  if (warp == 4 && lane == 0) {
    prefetch_tma_desc(&tm_q);
    prefetch_tma_desc(&tm_k);
    prefetch_tma_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_o = tmem + AT_TILE;

  // the tile's keys [j_lo, j_hi] (relative to a), in tiles of 128 from a multiple of 128 on
  const int i_last = min(t.i0 + AT_TILE, t.len) - 1;
  const int j_lo = p.left < 0 ? 0 : max(0, t.i0 - p.left);
  const int j_hi = p.right < 0 ? t.len - 1 : min(t.len - 1, i_last + p.right);
  const int jt0 = j_lo >> 7, nt = (j_hi >> 7) - jt0 + 1;

  if (warp == 4) {
    // ---------------------------------------------------------------- TMA
    int issued = 0;
    bool ok = true;
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, L::TILE);
      for (int c = 0; c < DC; ++c) tma_load_3d(sbase + L::Q + c * AT_BOX, &tm_q, q_full, c * 64, h, t.a + t.i0);
    }
    uint32_t st_phase = 0;
    for (int x = 0; ok && x < 2 * nt; ++x, ++issued) {
      const int s = x % L::RING;
      const bool is_v = x & 1;
      const int j0 = (jt0 + (x >> 1)) * AT_TILE;
      ok = at_wait(&empty[s], ((x / L::RING) & 1) ^ 1, abort_flag, 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      const bool ragged = is_v && j0 + AT_TILE > t.len;
      if (lane == 0) {
        uint64_t* bar = ragged ? staged : &full[s];
        mbar_arrive_expect_tx(bar, L::TILE);
        for (int c = 0; c < DC; ++c)
          tma_load_3d(sbase + L::KV + s * L::TILE + c * AT_BOX, is_v ? &tm_v : &tm_k, bar, c * 64, hk, t.a + j0);
      }
      if (ragged) {
        ok = __all_sync(0xffffffffu, at_wait(staged, st_phase, abort_flag, 2));
        if (!ok) at_drain(staged, st_phase);
        st_phase ^= 1;
        at_zero_rows<DC>(smem + L::KV + s * L::TILE, t.len - j0);
        if (lane == 0) mbar_arrive(&full[s]);
      }
    }
    // an abandoned CTA's loads must have landed before its shared memory goes
    if (*abort_flag && lane == 0) {
      at_drain(q_full, 0);
      for (int x = max(0, issued - L::RING); x < issued; ++x) at_drain(&full[x % L::RING], (x / L::RING) & 1);
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0) {
      const int kd = (p.head_dim + 15) / 16;               // K steps of the scores
      const uint32_t id_s = at_idesc<T>(AT_TILE, false);
      const uint32_t id_o = at_idesc<T>(kd * 16, true);    // N = head_dim rounded up to 16
      const uint64_t dq = smem_desc_sw128(sbase + L::Q, 16, 1024);
      const uint64_t dk0 = smem_desc_sw128(sbase + L::KV, 16, 1024);
      const uint64_t dv0 = smem_desc_sw128(sbase + L::KV, AT_BOX, 1024);
      bool ok = at_wait(q_full, 0, abort_flag, 3);
      auto scores = [&](int x) {  // x: ring position of the K tile
        const int s = x % L::RING;
        ok = ok && at_wait(&full[s], (x / L::RING) & 1, abort_flag, 4);
        if (!ok) return;
        tc_fence_after();
        const uint64_t dk = dk0 + uint64_t(s * (L::TILE >> 4));
        for (int k = 0; k < kd; ++k) {
          const uint64_t off = uint64_t((k >> 2) * (AT_BOX >> 4) + (k & 3) * 2);
          umma_f16(t_s, dq + off, dk + off, id_s, k > 0);
        }
        umma_commit(&empty[s]);
        umma_commit(s_full);
      };
      scores(0);
      for (int i = 0; ok && i < nt; ++i) {
        const int x = 2 * i + 1, s = x % L::RING;
        ok = at_wait(&full[s], (x / L::RING) & 1, abort_flag, 5) && at_wait(p_ready, i & 1, abort_flag, 6);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = dv0 + uint64_t(s * (L::TILE >> 4));
#pragma unroll
        for (int k = 0; k < AT_TILE / 16; ++k)
          umma_f16_ts(t_o, t_s + k * 8, dv + uint64_t(k * (2048 >> 4)), id_o, i > 0 || k > 0);
        umma_commit(&empty[s]);
        // the next scores overwrite P: MMAs of one thread run in order
        if (i + 1 < nt) scores(x + 1);
      }
      umma_commit(o_full);
      at_drain(o_full, 0);  // nothing in flight when TMEM and shared memory go
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const uint32_t lane_off = uint32_t(warp * 32) << 16;
    const int i = t.i0 + threadIdx.x;  // this thread's query row, relative to a
    const float sl2 = p.scale * AT_LOG2E;
    const int see_lo = p.left < 0 ? 0 : i - p.left;
    const int see_hi = p.right < 0 ? t.len - 1 : min(t.len - 1, i + p.right);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int it = 0; it < nt; ++it) {
      const int j0 = (jt0 + it) * AT_TILE;
      ok = at_wait(s_full, it & 1, abort_flag, 7);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + lane_off + c * 32, s[c]);
      tmem_ld_wait();
      // tiles that the window or the sequence's end cuts (the same for the whole CTA)
      if (j0 + AT_TILE > t.len || (p.right >= 0 && j0 + AT_TILE - 1 > t.i0 + p.right) ||
          (p.left >= 0 && j0 < t.i0 + AT_TILE - 1 - p.left)) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (j0 + c < see_lo || j0 + c > see_hi) s[c >> 5][c & 31] = 0xff800000u;  // -inf
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c >> 5][c & 31]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // also where nothing was visible before (m = -inf: the factor is 0, and so are O and l)
      const bool grow = (top - m) * sl2 > AT_LAZY;
      if (it > 0 && __any_sync(0xffffffffu, grow)) {
        const float f = grow ? at_exp2((m - top) * sl2) : 1.f;
        l *= f;
#pragma unroll 1
        for (int c = 0; c < p.head_dim; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + lane_off + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st_32x32b_x32(t_o + lane_off + c, o);
        }
      }
      if (it == 0 || grow) m = top;
      const float neg = m == -INFINITY ? 0.f : -m * sl2;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const int e = c * 64 + 2 * k;
          const float a = at_exp2(fmaf(__uint_as_float(s[e >> 5][e & 31]), sl2, neg));
          const float b = at_exp2(fmaf(__uint_as_float(s[e >> 5][(e & 31) + 1]), sl2, neg));
          sum[k & 3] += a + b;
          pk[k] = at_pack<T>(a, b);  // the MMA's operand type; l keeps the 32-bit values
        }
        tmem_st_32x32b_x32(t_s + lane_off + c * 32, pk);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_ready);
    }
    if (__all_sync(0xffffffffu, ok)) ok = at_wait(o_full, 0, abort_flag, 8);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t row = t.a + i;
      T* o_row = out + (row * p.heads + h) * p.head_dim;
#pragma unroll
      for (int c = 0; c < DC * 2; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + lane_off + c * 32, o);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint4 v;
          uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = at_pack<T>(__uint_as_float(o[k * 8 + 2 * e]) * inv, __uint_as_float(o[k * 8 + 2 * e + 1]) * inv);
          if (i < t.len && c * 32 + k * 8 < p.head_dim) *reinterpret_cast<uint4*>(o_row + c * 32 + k * 8) = v;
        }
      }
      if (i < t.len) lse[int64_t(h) * p.tokens + row] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, 256);
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
  // CTAs of a launch
  NF4B_RETURN_IF(at_slots(a->tokens, a->rows) * a->heads > 0x7FFFFFFF, NF4B_ERR_UNSUPPORTED);
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

// [tokens][heads][head_dim] as 64-feature boxes of 128 tokens of one head, 128-byte swizzle, zeros
// outside the tensor.
static int attn_tmap(CUtensorMap* m, const nf4b_attn& a, const void* base, int heads, int64_t stride, int64_t head_stride) {
  const uint64_t dims[3] = {uint64_t(a.head_dim), uint64_t(heads), uint64_t(a.tokens)};
  const uint64_t strides[2] = {uint64_t(head_stride) * 2, uint64_t(stride) * 2};
  const uint32_t box[3] = {64, 1, AT_TILE};
  return make_tmap_tiled(m, a.dtype == NF4B_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

static AttnParams attn_params(const nf4b_attn& a) {
  return AttnParams{a.cu,       int32_t(a.tokens), a.rows,  a.heads, a.kv_heads,
                    a.head_dim, a.left,            a.right, int32_t(at_slots(a.tokens, a.rows)), a.scale};
}

// Dynamic shared memory of a kernel, set once per device.
template <typename K>
static int attn_smem(K kernel, int bytes, bool (&done)[64]) {
  static std::mutex mu;
  int dev = 0;
  NF4B_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return NF4B_ERR_DEVICE;
  std::lock_guard<std::mutex> lock(mu);
  if (!done[dev]) {
    NF4B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return NF4B_OK;
}

template <typename T, int DC>
static int attn_fwd_launch(const nf4b_attn& a, void* out, float* lse, cudaStream_t s) {
  CUtensorMap q, k, v;
  int st = attn_tmap(&q, a, a.q, a.heads, a.q_stride, a.q_head_stride);
  if (st == NF4B_OK) st = attn_tmap(&k, a, a.k, a.kv_heads, a.k_stride, a.k_head_stride);
  if (st == NF4B_OK) st = attn_tmap(&v, a, a.v, a.kv_heads, a.v_stride, a.v_head_stride);
  static bool done[64] = {false};
  if (st == NF4B_OK) st = attn_smem(attn_fwd_kernel<T, DC>, AttnFwdSmem<DC>::ALLOC, done);
  if (st != NF4B_OK) return st;
  const AttnParams p = attn_params(a);
  NF4B_CUDA_TRY(launch_pdl(attn_fwd_kernel<T, DC>, dim3(unsigned(p.slots) * unsigned(a.heads)), dim3(AT_FWD_THREADS),
                           size_t(AttnFwdSmem<DC>::ALLOC), s, q, k, v, p, static_cast<T*>(out), lse));
  return launch_status("attn_fwd_kernel launch");
}

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
  const bool wide = a.head_dim > 64;
  if (a.dtype == NF4B_F16)
    return wide ? attn_fwd_launch<__half, 2>(a, out, lse, s) : attn_fwd_launch<__half, 1>(a, out, lse, s);
  return wide ? attn_fwd_launch<__nv_bfloat16, 2>(a, out, lse, s) : attn_fwd_launch<__nv_bfloat16, 1>(a, out, lse, s);
}

extern "C" int nf4b_attn_error_flag(int* value, int reset) {
  NF4B_RETURN_IF(value == nullptr, NF4B_ERR_INVALID_ARG);
  NF4B_CUDA_TRY(cudaMemcpyFromSymbol(value, g_attn_error, sizeof(int)));
  if (reset) {
    const int zero = 0;
    NF4B_CUDA_TRY(cudaMemcpyToSymbol(g_attn_error, &zero, sizeof(int)));
  }
  return NF4B_OK;
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
