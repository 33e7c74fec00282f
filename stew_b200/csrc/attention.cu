// Attention over packed token rows, forward and backward (C ABI include/stew_step.h):
//   s_ij = scale q_i.k_j,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - do_i.o_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// over the pairs (i, j) of one sequence inside the window i - left <= j <= i + right.
//
// Every product runs on tcgen05 over tiles of 128 or 64 tokens that TMA brings in; a ragged tile's rows of
// other sequences are zeroed in shared memory where a product sums over them, and masked elsewhere.
// Sums and softmax statistics are fp32 (TMEM, registers), in a fixed order.
#include <cstdlib>
#include <mutex>
#include <type_traits>

#include "attn_common.cuh"

namespace nf4b {

// ------------------------------------------------------------------- forward
// One CTA per (128-token query tile, head), over key tiles of 64 tokens; two CTAs on an SM, so one's
// softmax runs beside the other's MMAs.  TMEM (256 columns): two buffers of scores S = Q K^T, 64
// columns each, and the output O.  The scores of tile i + 1 are computed while the softmax of tile i
// runs; its probabilities overwrite its own scores as 16-bit values and are the A operand of P V
// straight from TMEM.  Q, K and V are TMA tiles in shared memory (V's is read as an MN-major operand,
// so nothing is transposed).
//   warps 0-3  softmax: one thread per query row
//   warp 4     TMA: Q, then K and V tiles through a ring of slots
//   warp 5     TMEM allocation, MMA issue
// One pass over the keys with a running maximum m and sum l (Milakov and Gimelshein's online
// softmax, with the known refinement that O is rescaled only when the maximum has grown by more than a
// threshold, here 2^8: else exp(s - m) may exceed 1, and l with it -- the quotient is the same).
// fp16: P holds 2^7 exp(s - m), at most 2^15 (l and O carry the factor, lse drops it), so that fp16's
// subnormals begin at 2^-21 of the row's maximum and zeros at 2^-32.  l sums P before its rounding: without
// the factor 65,536 keys at 2^-25.1 of the maximum, 1.8e-3 of the row's weight, were in l and not in O.
// Measured, 12 query / 2 key-value heads of 128, fp16: 16,384 causal tokens 780-830 us over boxes, 993-1,058 TFLOP/s
// (the power cap: cuBLAS sustains 1,371); 1,170 tokens in 4 rows 11.7 us, bound by a key tile's chain (scores,
// exponentials, product: about 1.1 us).  128-key tiles with one buffer of scores: 909 us; two query tiles per
// CTA that share K and V: 813.
constexpr int AT_KEYS = 64;                  // keys of a tile
constexpr int AT_KBOX = AT_KEYS * 128;       // bytes of its 64-feature TMA box
template <int DC>
struct AttnFwdSmem {
  static constexpr int QTILE = DC * AT_BOX;
  static constexpr int TILE = DC * AT_KBOX;
  static constexpr int RING = DC == 1 ? 10 : 4;
  static constexpr int Q = 0;
  static constexpr int KV = QTILE;
  static constexpr int BAR = KV + RING * TILE;
  // full[RING], empty[RING], q_full, s_full[2], p_ready[2], o_done, o_full
  static constexpr int NBAR = 2 * RING + 7;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int ALLOC = MISC + 16 + 1024;  // slack to align the base to 1024 B
};
static_assert(AttnFwdSmem<2>::ALLOC <= 115712 && AttnFwdSmem<1>::ALLOC <= 115712, "two CTAs on an SM");
constexpr int AT_FWD_THREADS = 192;
constexpr float AT_LAZY = 8.f;  // log2 growth of the maximum that O tolerates unscaled
// log2 of the factor that the forward's P carries
template <typename T>
constexpr float at_fwd_shift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

template <typename T, int DC>
__global__ void __launch_bounds__(AT_FWD_THREADS, 2)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p, T* __restrict__ out,
                    T* __restrict__ rest, float* __restrict__ lse) {
  using L = AttnFwdSmem<DC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* empty = full + L::RING;
  uint64_t* q_full = empty + L::RING;
  uint64_t* s_full = q_full + 1;    // [buffer]
  uint64_t* p_ready = s_full + 2;   // [buffer]
  uint64_t* o_done = p_ready + 2;   // a phase per P V (at most one behind where it is waited for)
  uint64_t* o_full = o_done + 1;    // after the last
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const AttnWait aw{abort_flag, p.wait_cycles};
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 128) {
    prefetch_tma_desc(&tm_q);
    prefetch_tma_desc(&tm_k);
    prefetch_tma_desc(&tm_v);
  }
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
      const int64_t off = (row * p.heads + h) * p.head_dim + (i % vec) * 8;
      *reinterpret_cast<uint4*>(out + off) = make_uint4(0, 0, 0, 0);
      if (rest != nullptr) *reinterpret_cast<uint4*>(rest + off) = make_uint4(0, 0, 0, 0);
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
    }
    mbar_init(o_done, 1);
    mbar_init(o_full, 1);
    fence_barrier_init();
    *abort_flag = 0;
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // scores at [0, 128), O behind them
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  // the tile's keys [j_lo, j_hi] (relative to a), in tiles of 64 from a multiple of 64 on
  const int i_last = min(t.i0 + AT_TILE, t.len) - 1;
  const int j_lo = p.left < 0 ? 0 : max(0, t.i0 - p.left);
  const int j_hi = p.right < 0 ? t.len - 1 : min(t.len - 1, i_last + p.right);
  const int jt0 = j_lo / AT_KEYS, nt = j_hi / AT_KEYS - jt0 + 1;

  if (warp == 4) {
    // ---------------------------------------------------------------- TMA
    int issued = 0;
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, L::QTILE);
      for (int c = 0; c < DC; ++c) tma_load_3d(sbase + L::Q + c * AT_BOX, &tm_q, q_full, c * 64, h, t.a + t.i0);
      for (int x = 0; x < 2 * nt; ++x, ++issued) {
        const int s = x % L::RING;
        if (!at_wait(&empty[s], ((x / L::RING) & 1) ^ 1, aw, 1)) break;
        mbar_arrive_expect_tx(&full[s], L::TILE);
        for (int c = 0; c < DC; ++c)
          tma_load_3d(sbase + L::KV + s * L::TILE + c * AT_KBOX, x & 1 ? &tm_v : &tm_k, &full[s], c * 64, hk,
                      t.a + (jt0 + (x >> 1)) * AT_KEYS);
      }
      // The loads must have landed before the CTA's shared memory goes.  Whoever gives up may do so after the
      // last of them was issued: always waited for (a finished CTA's have been).
      at_drain(q_full, 0);
      for (int x = max(0, issued - L::RING); x < issued; ++x) at_drain(&full[x % L::RING], (x / L::RING) & 1);
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA
    const uint32_t lead = elect_one();
    const int kd = (p.head_dim + 15) / 16;               // K steps of the scores
    const uint32_t id_s = at_idesc<T>(AT_KEYS, false);
    const uint32_t id_o = at_idesc<T>(kd * 16, true);    // N = head_dim rounded up to 16
    const uint64_t dq = smem_desc_sw128(sbase + L::Q, 16, 1024);
    const uint64_t dk0 = smem_desc_sw128(sbase + L::KV, 16, 1024);
    const uint64_t dv0 = smem_desc_sw128(sbase + L::KV, AT_KBOX, 1024);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      ok = __all_sync(0xffffffffu, ok && at_wait(bar, parity, aw, where));
      return ok;
    };
    auto arrived = [&](int x) { return wait(&full[x % L::RING], (x / L::RING) & 1, 4); };
    auto scores = [&](int i) {
      const uint64_t dk = dk0 + uint64_t((2 * i) % L::RING * (L::TILE >> 4));
#pragma unroll
      for (int k = 0; k < DC * 4; ++k)
        if (k < kd)
          at_mma_ss(lead, tmem + (i & 1) * AT_KEYS, dq + uint64_t((k >> 2) * (AT_BOX >> 4) + (k & 3) * 2),
                    dk + uint64_t((k >> 2) * (AT_KBOX >> 4) + (k & 3) * 2), id_s, k > 0);
      at_commit(lead, &s_full[i & 1]);
      at_commit(lead, &empty[(2 * i) % L::RING]);
    };
    wait(q_full, 0, 3);
    for (int i = 0; ok && i < 2 && i < nt; ++i) {
      if (!arrived(2 * i)) break;
      tc_fence_after();
      scores(i);
    }
    for (int i = 0; ok && i < nt; ++i) {
      const int sv = (2 * i + 1) % L::RING;
      if (!arrived(2 * i + 1) || (i + 2 < nt && !arrived(2 * i + 4)) || !wait(&p_ready[i & 1], (i >> 1) & 1, 6)) break;
      tc_fence_after();
      const uint64_t dv = dv0 + uint64_t(sv * (L::TILE >> 4));
      const int j0 = (jt0 + i) * AT_KEYS;
#pragma unroll
      for (int k = 0; k < AT_KEYS / 16; ++k)
        if (j0 + k * 16 < t.len)  // nothing behind the sequence's end
          at_mma_ts(lead, tmem + AT_TILE, tmem + (i & 1) * AT_KEYS + k * 8, dv + uint64_t(k * (2048 >> 4)), id_o,
                    i > 0 || k > 0);
      at_commit(lead, o_done);
      at_commit(lead, &empty[sv]);
      // the scores of tile i + 2 overwrite P of tile i: MMAs of one thread run in order
      if (i + 2 < nt) scores(i + 2);
    }
    // nothing in flight when TMEM and shared memory go
    at_commit(lead, o_full);
    at_drain(o_full, 0);
  } else {
    // ---------------------------------------------------------------- softmax
    const int w0 = warp * 32;
    const uint32_t lane_off = uint32_t(w0) << 16;
    const uint32_t t_s = tmem + lane_off, t_o = tmem + lane_off + AT_TILE;
    const int i = t.i0 + threadIdx.x;  // this thread's query row, relative to a
    const float sl2 = p.scale * AT_LOG2E;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    const int see_lo = p.left < 0 ? 0 : i - p.left;
    const int see_hi = p.right < 0 ? t.len - 1 : min(t.len - 1, i + p.right);
    const int lo_max = p.left < 0 ? 0 : t.i0 + w0 + 31 - p.left;  // what all rows of the warp see
    const int hi_min = p.right < 0 ? t.len - 1 : min(t.len - 1, t.i0 + w0 + p.right);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int it = 0; it < nt; ++it) {
      const int j0 = (jt0 + it) * AT_KEYS, b = it & 1;
      ok = at_wait(&s_full[b], (it >> 1) & 1, aw, 7);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint32_t s[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(t_s + b * AT_KEYS + c * 32, s[c]);
      tmem_ld_wait();
      if (j0 < lo_max || j0 + AT_KEYS - 1 > hi_min)
        at_hide(see_lo - j0, see_hi - j0, [&](int c) { s[c >> 5][c & 31] = 0xff800000u; });  // -inf
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < AT_KEYS; c += 2)
        mx[(c >> 1) & 3] = fmaxf(mx[(c >> 1) & 3], fmaxf(__uint_as_float(s[c >> 5][c & 31]), __uint_as_float(s[c >> 5][(c & 31) + 1])));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // also where nothing was visible before (m = -inf: the factor is 0, and so are O and l)
      const bool grow = (top - m) * sl2 > AT_LAZY;
      if (it > 0 && __any_sync(0xffffffffu, grow)) {
        const float f = grow ? at_exp2((m - top) * sl2) : 1.f;
        l *= f;
        ok = at_wait(o_done, (it - 1) & 1, aw, 9);  // the products so far
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < p.head_dim; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st_32x32b_x32(t_o + c, o);
        }
      }
      if (it == 0 || grow) m = top;
      const float neg = m == -INFINITY ? 0.f : fmaf(-m, sl2, at_fwd_shift<T>());
      const uint64_t negx2 = f2_pack(neg, neg);
      uint64_t sum[2] = {0, 0};
      uint32_t pk[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const int e = 2 * k;
        const float2 x = f2_unpack(f2_fma(f2_pack_u(s[e >> 5][e & 31], s[e >> 5][(e & 31) + 1]), sl2x2, negx2));
        const float u = at_exp2(x.x), v = at_exp2(x.y);
        sum[k & 1] = f2_add(sum[k & 1], f2_pack(u, v));
        pk[k] = at_pack<T>(u, v);  // the MMA's operand type; l keeps the 32-bit values
      }
      tmem_st_32x32b_x32(t_s + b * AT_KEYS, pk);
      const float2 l2 = f2_unpack(f2_add(sum[0], sum[1]));
      l += l2.x + l2.y;
      if (j0 + AT_KEYS > t.len) {  // the ragged last tile: V's rows behind the sequence's end
        const int x = 2 * it + 1;
        ok = at_wait(&full[x % L::RING], (x / L::RING) & 1, aw, 2);
        if (!__all_sync(0xffffffffu, ok)) break;
        at_zero_rows<DC, AT_KEYS, 128>(smem + L::KV + (x % L::RING) * L::TILE, t.len - j0, threadIdx.x);
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[b]);
    }
    if (__all_sync(0xffffffffu, ok)) ok = at_wait(o_full, 0, aw, 8);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t row = t.a + t.i0 + w0;
      // every MMA is done: the Q tile's memory is free
      at_store_rows<T, DC * 64>(t_o, smem + L::Q + w0 * DC * 128, out + (row * p.heads + h) * p.head_dim,
                                int64_t(p.heads) * p.head_dim, t.len - t.i0 - w0, p.head_dim, inv);
      if (rest != nullptr)
        at_store_rows<T, DC * 64, true>(t_o, smem + L::Q + w0 * DC * 128, rest + (row * p.heads + h) * p.head_dim,
                                        int64_t(p.heads) * p.head_dim, t.len - t.i0 - w0, p.head_dim, inv);
      if (i < t.len) lse[int64_t(h) * p.tokens + row + lane] = l == 0.f ? -INFINITY : m * p.scale + logf(l * (1.f / float(1 << int(at_fwd_shift<T>()))));
    }
    __syncwarp();
    tmem_st_wait();  // (a warp that gave up may have stores under way)
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, 256);
  if (*abort_flag) {  // a wait ran out somewhere: no row of the tile is an answer
    const int n = min(AT_TILE, t.len - t.i0);
    const int64_t off = (int64_t(t.a + t.i0) * p.heads + h) * p.head_dim, stride = int64_t(p.heads) * p.head_dim;
    at_poison_rows(out + off, stride, n, p.head_dim, threadIdx.x, AT_FWD_THREADS);
    if (rest != nullptr) at_poison_rows(rest + off, stride, n, p.head_dim, threadIdx.x, AT_FWD_THREADS);
    if (threadIdx.x < n) lse[int64_t(h) * p.tokens + t.a + t.i0 + threadIdx.x] = __int_as_float(0x7fffffff);
  }
}

// ------------------------------------------------------------------ backward
// Two launches.  The first (attn_prep_kernel) writes, per (head, token), the row's log-sum-exp in
// log2 units and delta = do.o (o with what its rounding left, where the forward kept that), and zeros behind
// the last sequence.  The second's persistent CTAs work on two
// kinds of units with one structure, a resident pair of 128-token tiles X, Y against a ring of tile pairs
// A, B (D = head_dim):
//   keys    : X = K, Y = V of a key tile; A = Q, B = dO over the query tiles of the group's heads (or a share
//             of them):  S^T = X A^T, dP^T = Y B^T, dV += P^T B, dK += dS^T A
//   queries : X = Q, Y = dO of a query tile and head; A = K, B = V over its key tiles:
//             S = X A^T, dP = Y B^T, dQ += dS A
// S and dP are recomputed by both kinds (7 products instead of 5): that buys dQ, dK and dV summed in
// TMEM in a fixed order, with no fp32 dQ buffer in memory and no atomics on values.  P and dS overwrite S and
// dP in TMEM as 16-bit values and are the A operands of the second products from there.
//   warps 0-7  elementwise: thread (row = TMEM lane, half of the columns)
//   warp 8     takes units, TMA; for key tiles also the query rows' (lse, delta) into shared memory
//   warp 9     TMEM allocation, MMA issue
// Measured, heads as above: 8,192 causal tokens 660-695 us over boxes, 741-780 TFLOP/s of the formula's five products
// (the power cap again); 1,170 tokens in 4 rows 33 us with six shares a key tile (one: 62).  A key tile's step takes
// about 2,900 clocks, of them 1,150 exponentials and 1,250 other elementwise work and waits in one chain,
// beside 2,048 of MMAs; a launch per unit instead of persistent CTAs: 43 us and 694.
//
// Fine units keep dS as two 16-bit values, its rounding and what that leaves, each with its product (at_fine()).
//
// fp16 range: dS is rounded to the operand type with a power-of-two scale 2^k that puts the largest
// |dO||V| + |delta| of the tiles a unit meets (the prep launch's maxima) at 2^14, and P with 2^8:
// gradients of any size keep fp16's 11 bits, where unscaled products of small gradients would fall
// into its subnormals (rows share their unit's scale: beside rows with gradients 2^20 times larger they still
// do).  The whole sequence's maxima would do for one scale, but their scan grows with the sequence under a
// window: 262,144 tokens, window 128, 14 heads of 64 on 2: 6,962 us against 2,046.  bf16 has fp32's range and
// is not scaled.
constexpr int AT_BWD_THREADS = 320;
constexpr int AT_PREP_THREADS = 256;

template <typename T>
constexpr float at_p_shift() { return std::is_same<T, __half>::value ? 8.f : 0.f; }

// The backward's scratch.
struct AttnWork {
  float2* row;    // [heads][tokens]: lse log2(e), delta
  float2* tile;   // [heads][slots]: max |dO_i|, max |delta_i| of a query tile
  float* vmax;    // [kv_heads][slots]: max |V_j| of a key tile
  unsigned* next;     // the next unit of work
  unsigned* tickets;  // [slots][kv_heads]: warps of a key tile's shares that are done
  float* parts;       // [slots][kv_heads][split]: their sums
};

__device__ __forceinline__ float at_half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA per (128-token tile, head), half a warp per row; reads O and dO.  Further CTAs per (tile, key/value
// head) read V.
template <typename T>
__global__ void __launch_bounds__(AT_PREP_THREADS)
    attn_prep_kernel(const __grid_constant__ AttnParams p, const T* __restrict__ out, const T* __restrict__ rest,
                     const T* __restrict__ dout,
                     const float* __restrict__ lse, const T* __restrict__ v, int64_t v_stride, int64_t v_head_stride,
                     AttnWork w, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv) {
  grid_dep_wait();  // programmatic launch: no global access before the wait
  const int per_slot = p.heads + p.kv_heads;
  const int slot = int(blockIdx.x / per_slot), h = blockIdx.x % per_slot, hk = h - p.heads;
  const bool keys = hk >= 0;
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) *w.next = 0;
    if (keys) w.tickets[slot * p.kv_heads + hk] = 0;
  }
  const AttnTile t = at_find(p, slot);
  if (t.i0 >= t.len) return;
  constexpr bool SCALED = at_p_shift<T>() != 0.f;
  constexpr int STEP = AT_PREP_THREADS / 16, N = AT_TILE / STEP;  // rows a thread works on: r0 + k STEP
  const int n = min(AT_TILE, t.len - t.i0);
  const int sub = threadIdx.x & 15, f = sub * 8, r0 = threadIdx.x >> 4;  // this thread's 8 features, first row
  const int64_t row0 = t.a + t.i0 + r0;
  auto live = [&](int k) { return r0 + k * STEP < n && f < p.head_dim; };
  if (t.tail) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    for (int k = 0; k < N; ++k) {
      if (!live(k)) continue;
      if (keys) {
        const int64_t off = ((row0 + k * STEP) * p.kv_heads + hk) * p.head_dim + f;
        *reinterpret_cast<uint4*>(dk + off) = z;
        *reinterpret_cast<uint4*>(dv + off) = z;
      } else {
        *reinterpret_cast<uint4*>(dq + ((row0 + k * STEP) * p.heads + h) * p.head_dim + f) = z;
      }
    }
    return;
  }
  if (keys && !SCALED) return;
  uint4 x4[N], y4[N], d4[N];  // every load under way before the first sum
  float l[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    x4[k] = y4[k] = d4[k] = make_uint4(0, 0, 0, 0);
    l[k] = 0.f;
    const int64_t row = row0 + k * STEP;
    if (!live(k)) continue;
    if (keys) {
      x4[k] = *reinterpret_cast<const uint4*>(v + row * v_stride + hk * v_head_stride + f);
    } else {
      const int64_t off = (row * p.heads + h) * p.head_dim + f;
      x4[k] = *reinterpret_cast<const uint4*>(out + off);
      d4[k] = *reinterpret_cast<const uint4*>(dout + off);
      if (rest != nullptr) y4[k] = *reinterpret_cast<const uint4*>(rest + off);
      if (sub == 0) l[k] = lse[int64_t(h) * p.tokens + row];
    }
  }
  float m_norm = 0.f, m_dl = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&x4[k]);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&y4[k]);
    const uint32_t* d = reinterpret_cast<const uint32_t*>(keys ? &x4[k] : &d4[k]);
    float dot = 0.f, nd = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = at_unpack<T>(x[i]), c = at_unpack<T>(y[i]), b = at_unpack<T>(d[i]);
      dot = fmaf(a.x + c.x, b.x, fmaf(a.y + c.y, b.y, dot));
      nd = fmaf(b.x, b.x, fmaf(b.y, b.y, nd));
    }
    if (!keys) {
      dot = at_half_warp_sum(dot);
      // a row without weight (lse = -inf) must give p = 0
      if (r0 + k * STEP < n && sub == 0)
        w.row[int64_t(h) * p.tokens + row0 + k * STEP] = make_float2(l[k] == -INFINITY ? INFINITY : l[k] * AT_LOG2E, dot);
      m_dl = fmaxf(m_dl, fabsf(dot));
    }
    if (SCALED) m_norm = fmaxf(m_norm, at_half_warp_sum(nd));
  }
  if (!SCALED) return;
  __shared__ float s_max[2][AT_PREP_THREADS / 16];
  if (sub == 0) {
    s_max[0][r0] = m_norm;
    s_max[1][r0] = m_dl;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float m = 0.f, e = 0.f;
    for (int i = 0; i < AT_PREP_THREADS / 16; ++i) {
      m = fmaxf(m, s_max[0][i]);
      e = fmaxf(e, s_max[1][i]);
    }
    if (keys) w.vmax[int64_t(hk) * p.slots + slot] = sqrtf(m);
    else w.tile[int64_t(h) * p.slots + slot] = make_float2(sqrtf(m), e);
  }
}

// Whole warp: the exponent k of a unit's dS scale, from the tiles it meets: nd query tiles from slot d0 on of
// heads [h0, h0 + nh), nv key tiles from slot v0 on of key/value head hk.  (Any k is right that overflows
// nothing: the sums are scaled back in fp32.  Only a unit's own tiles are read, so that under a window the
// scan does not grow with the sequence.)
__device__ __forceinline__ int at_ds_exponent(const AttnParams& p, const AttnWork& w, int h0, int nh, int d0, int nd, int hk,
                                              int v0, int nv) {
  const int lane = threadIdx.x & 31;
  float m_do = 0.f, m_dl = 0.f, m_v = 0.f;
  for (int i = lane; i < nh * nd; i += 32) {
    const int g = i / nd;
    const float2 x = w.tile[int64_t(h0 + g) * p.slots + d0 + i - g * nd];
    m_do = fmaxf(m_do, x.x);
    m_dl = fmaxf(m_dl, x.y);
  }
  for (int i = lane; i < nv; i += 32) m_v = fmaxf(m_v, w.vmax[int64_t(hk) * p.slots + v0 + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m_do = fmaxf(m_do, __shfl_xor_sync(0xffffffffu, m_do, o));
    m_dl = fmaxf(m_dl, __shfl_xor_sync(0xffffffffu, m_dl, o));
    m_v = fmaxf(m_v, __shfl_xor_sync(0xffffffffu, m_v, o));
  }
  const float m = fmaf(m_do, m_v, m_dl);  // |dS| = p |dP - delta| <= |dO||V| + |delta|
  if (!(m > 0.f) || !(m < INFINITY)) return 0;
  const int e = int((__float_as_uint(m) >> 23) & 255u) - 127;
  return min(max(14 - e, -100), 100);
}
__device__ __forceinline__ float at_pow2(int k) { return __uint_as_float(uint32_t(k + 127) << 23); }

template <int DC>
struct AttnBwdSmem {
  static constexpr int TILE = DC * AT_BOX;
  static constexpr int X = 0;
  static constexpr int Y = TILE;
  static constexpr int A = 2 * TILE;
  static constexpr int B = 4 * TILE;
  static constexpr int OUT = 6 * TILE;             // 2 KB per elementwise warp: rows on their way out
  static constexpr int AUX = OUT + 8 * 2048;       // [2][128] -lse, [2][128] -delta (scaled)
  static constexpr int UNIT = AUX + 4 * AT_TILE * 4;  // [2] AttnUnit, and the last 4 taken
  static constexpr int BAR = UNIT + 6 * 64;
  // a_full[2], a_empty[2], b_full[2], b_empty[2], aux_empty[2], unit_full[2], unit_empty[2], xy_full,
  // xy_empty, s_full, p_ready, dp_full, ds_ready, acc_full, acc_empty, drained, exp_full[2]
  static constexpr int NBAR = 25;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int ALLOC = MISC + 16 + 1024;  // slack to align the base to 1024 B
};
static_assert(AttnBwdSmem<2>::ALLOC <= 232448, "shared memory budget");

// TMEM columns (512): S | P, dP | dS, and the two sums.
constexpr int AT_TM_S = 0, AT_TM_DP = 128, AT_TM_DV = 256, AT_TM_DX = 384;

struct AttnBwdMaps {
  CUtensorMap q, k, v, dout;
};

// One unit of work: a key tile and a share of its group's heads, a query tile and a head, or a piece of the
// sum over a key tile's shares.
enum { AT_UNIT_QUERIES = 0, AT_UNIT_KEYS = 1, AT_UNIT_JOIN = 2, AT_UNIT_END = 3 };
constexpr int AT_PIECES = 4;  // pieces of that sum
struct AttnUnit {
  int kind, a, len, i0;  // the resident tile: tokens a + [i0, i0 + 128) of a sequence of len
  int h, hk, rank;       // head of X and Y; key/value head; the share of a key tile, or the piece of a sum
  int yt0, nt, n;        // the ring's first tile, its tiles per head, ring items
  int h0;                // first query head of a key tile's share
  int join;              // the key tile's number among those that are shared
  int fine;              // dS as two 16-bit values
};
static_assert(sizeof(AttnUnit) <= 64, "one slot of the unit ring");

// Whether dS goes into dQ and dK with what its rounding leaves: sequences of one tile, windows of 128, and
// batches whose sequences have 256 tokens or fewer on average (the tokens behind the last one do not count).  The
// ds of a row sum to zero, so over a few tokens their roundings stay in the sums: with two to ten tokens a
// sequence dq and dk were 1.50 to 1.56 times as far off the 64-bit result as values rounded once, with the rest
// 1.05 to 1.14 times; over some hundred tokens it was 1.43.  It costs a second dS product: a backward of 1,170
// tokens in 4 rows 33 -> 36 us where all of them take it, of 8,192 670 -> 820.  The choice is a unit's own, so
// that a short sequence's gradients do not depend on what is packed beside it: that took 1,170 tokens from 32 to
// 33 us, a window of 255 over 8,192 from 90.5 to 94.5, 8,192 causal ones from 666 to 676 (against a kernel of
// each kind, chosen for the whole call).
__device__ __forceinline__ bool at_fine(const AttnParams& p, int len) {
  return len <= AT_TILE || (p.left >= 0 && p.right >= 0 && p.left + p.right < AT_TILE) ||
         (at_start(p, p.rows) + 255) >> 8 <= p.rows;
}

// Whole warp: unit number `at` of the order (below n_all), false for one without tokens.
struct AttnUnits {
  unsigned n_keys, n_main, n_all;
  __device__ AttnUnits(const AttnParams& p, int split) {
    n_keys = unsigned(p.slots) * unsigned(p.kv_heads) * unsigned(split);
    n_main = n_keys + unsigned(p.slots) * unsigned(p.heads);
    n_all = n_main + (split > 1 ? unsigned(p.slots) * unsigned(p.kv_heads) * AT_PIECES : 0u);
  }
};
__device__ __forceinline__ bool at_unit(const AttnParams& p, const AttnUnits& order, int split, unsigned at, AttnUnit& u, int& slot) {
  const int grp = p.heads / p.kv_heads;
  if (at < order.n_keys) {
    u.kind = AT_UNIT_KEYS;
    u.rank = int(at % unsigned(split));
    u.join = int(at / unsigned(split));
  } else if (at < order.n_main) {
    u.kind = AT_UNIT_QUERIES;
    u.rank = u.join = 0;
    slot = p.slots - 1 - int((at - order.n_keys) / unsigned(p.heads));
    u.h = int((at - order.n_keys) % unsigned(p.heads));
    u.hk = u.h / grp;
    u.h0 = 0;
  } else {
    u.kind = AT_UNIT_JOIN;
    u.rank = int((at - order.n_main) % AT_PIECES);
    u.join = int((at - order.n_main) / AT_PIECES);
  }
  if (u.kind != AT_UNIT_QUERIES) {
    slot = int(unsigned(u.join) / unsigned(p.kv_heads));
    u.h = u.hk = int(unsigned(u.join) % unsigned(p.kv_heads));
    u.h0 = u.h * grp + u.rank * (grp / split);
  }
  const AttnTile t = at_find(p, slot);
  if (t.tail || t.i0 >= t.len) {  // rows behind the last sequence: the prep launch's
    u.kind = AT_UNIT_END;
    return false;
  }
  u.a = t.a;
  u.len = t.len;
  u.i0 = t.i0;
  const bool keys = u.kind == AT_UNIT_KEYS;
  const int back = keys ? p.right : p.left, ahead = keys ? p.left : p.right;  // the window seen from X's side
  const int last = min(t.i0 + AT_TILE, t.len) - 1;
  const int lo = back < 0 ? 0 : max(0, t.i0 - back), hi = ahead < 0 ? t.len - 1 : min(t.len - 1, last + ahead);
  u.yt0 = lo >> 7;
  u.nt = (hi >> 7) - u.yt0 + 1;
  u.n = keys ? u.nt * (grp / split) : u.nt;
  u.fine = at_fine(p, t.len);
  return true;
}

// A share's sums: groups of four features of [dK | dV], by rows.
template <int DC>
__device__ __forceinline__ float4* at_part(float* parts, int join, int split, int rank) {
  return reinterpret_cast<float4*>(parts) + (int64_t(join) * split + rank) * (DC * 32) * AT_TILE;
}

// Persistent: every CTA takes units from a counter, the longest kind first (key tiles with a group's heads;
// of a causal sequence the first key tiles, which the most queries see, and the last query tiles; then the
// sums over shares), so that the next unit's tiles are on their way and its first scores done while this
// unit's sums are stored.  A sum waits for its shares; they come before it in the order, so each has been
// taken by a CTA that runs and does not wait for it (no unit belongs to a CTA before that CTA takes it: one
// that found no room yet holds nothing up).
template <typename T, int DC>
__global__ void __launch_bounds__(AT_BWD_THREADS, 1)
    attn_bwd_kernel(const __grid_constant__ AttnBwdMaps maps, const __grid_constant__ AttnParams p, const AttnWork w,
                    const int split, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv) {
  using L = AttnBwdSmem<DC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* a_full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* a_empty = a_full + 2;
  uint64_t* b_full = a_empty + 2;
  uint64_t* b_empty = b_full + 2;
  uint64_t* aux_empty = b_empty + 2;
  uint64_t* unit_full = aux_empty + 2;
  uint64_t* unit_empty = unit_full + 2;
  uint64_t* xy_full = unit_empty + 2;
  uint64_t* xy_empty = xy_full + 1;
  uint64_t* s_full = xy_empty + 1;
  uint64_t* p_ready = s_full + 1;
  uint64_t* dp_full = p_ready + 1;
  uint64_t* ds_ready = dp_full + 1;
  uint64_t* acc_full = ds_ready + 1;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drained = acc_empty + 1;
  uint64_t* exp_full = drained + 1;  // [2]: a unit's exponent of the dS scale, which comes after the unit
  float* aux_lse = reinterpret_cast<float*>(smem + L::AUX);
  float* aux_dl = aux_lse + 2 * AT_TILE;
  AttnUnit* units = reinterpret_cast<AttnUnit*>(smem + L::UNIT);
  AttnUnit* taken = units + 2;  // [4]: the last units this CTA took
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const AttnWait aw{abort_flag, p.wait_cycles};
  int* exponent = reinterpret_cast<int*>(smem + L::MISC + 8);  // [2]
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int grp = p.heads / p.kv_heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&a_full[i], 2);  // the tile, and the producer once the rows' (lse, delta) are there
      mbar_init(&a_empty[i], 1);
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], 1);
      mbar_init(&aux_empty[i], 8);
      mbar_init(&unit_full[i], 1);
      mbar_init(&unit_empty[i], 9);
      mbar_init(&exp_full[i], 1);
    }
    mbar_init(xy_full, 1);
    mbar_init(xy_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(p_ready, 256);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 256);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 256);
    mbar_init(drained, 1);
    fence_barrier_init();
    for (int i = 0; i < 4; ++i) taken[i].kind = AT_UNIT_END;
    *abort_flag = 0;
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 256) {
    prefetch_tma_desc(&maps.q);
    prefetch_tma_desc(&maps.k);
    prefetch_tma_desc(&maps.v);
    prefetch_tma_desc(&maps.dout);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_dep_wait();  // programmatic launch: no global access before the wait

  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) {  // whole warp
    ok = __all_sync(0xffffffffu, ok && at_wait(bar, parity, aw, where));
    return ok;
  };

  if (warp == 8) {
    // ---------------------------------------------------------------- units and TMA
    const AttnUnits order(p, split);
    unsigned loads = 0, issued = 0, aux = 0;  // ring items so far, also those under way
    int k = 0, tiles = 0;         // units so far; those of them with tiles
    // the row starts into the L1 while the first unit's number is on its way
    for (int i = lane * 32; i <= p.rows && i < 1024; i += 1024) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.cu + i));
    for (;; ++k) {
      // the next unit that is not empty
      AttnUnit u;
      u.kind = AT_UNIT_END;
      int slot = 0;
      for (;;) {
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(w.next, 1u);
        at = __shfl_sync(0xffffffffu, at, 0);
        if (at >= order.n_all || at_unit(p, order, split, at, u, slot)) break;
      }
      if (lane == 0) taken[k & 3] = u;
      const bool keys = u.kind == AT_UNIT_KEYS, main = keys || u.kind == AT_UNIT_QUERIES;
      auto load = [&](int hy, int y0) {  // ring item `loads`
        const int s = loads & 1;
        const uint32_t ph = ((loads >> 1) & 1) ^ 1;
        if (!wait(&a_empty[s], ph, 11) || !wait(&b_empty[s], ph, 12)) return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(&a_full[s], L::TILE);
          for (int c = 0; c < DC; ++c)
            tma_load_3d(sbase + L::A + s * L::TILE + c * AT_BOX, keys ? &maps.q : &maps.k, &a_full[s], c * 64, hy, u.a + y0);
          mbar_arrive_expect_tx(&b_full[s], L::TILE);
          for (int c = 0; c < DC; ++c)
            tma_load_3d(sbase + L::B + s * L::TILE + c * AT_BOX, keys ? &maps.dout : &maps.v, &b_full[s], c * 64, hy,
                        u.a + y0);
        }
        issued = loads + 1;
        return true;
      };
      if (main) {
        if (!wait(xy_empty, (tiles & 1) ^ 1, 9)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(xy_full, 2 * L::TILE);
          for (int c = 0; c < DC; ++c) {
            tma_load_3d(sbase + L::X + c * AT_BOX, keys ? &maps.k : &maps.q, xy_full, c * 64, u.h, u.a + u.i0);
            tma_load_3d(sbase + L::Y + c * AT_BOX, keys ? &maps.v : &maps.dout, xy_full, c * 64, u.h, u.a + u.i0);
          }
        }
        ++tiles;
        if (!load(keys ? u.h0 : u.hk, u.yt0 * AT_TILE)) break;  // the ring's first tiles before anything else
      } else if (u.kind == AT_UNIT_JOIN) {
        const long long t0 = clock64();
        const volatile unsigned* done = w.tickets + u.join;
        while (ok && *done < 8u * unsigned(split)) {  // every elementwise warp of every share
          if (*abort_flag) {
            ok = false;
          } else if (clock64() - t0 >= p.wait_cycles) {
            *abort_flag = 1;
            atomicExch(&g_attn_error, 27);
            ok = false;
          }
        }
        __threadfence();
        ok = __all_sync(0xffffffffu, ok);
      }
      if (!wait(&unit_empty[k & 1], ((k >> 1) & 1) ^ 1, 10)) break;
      if (lane == 0) {
        units[k & 1] = u;
        mbar_arrive(&unit_full[k & 1]);
      }
      if (u.kind == AT_UNIT_END) break;
      if (!main) continue;
      // (slot: units with tiles; the tiles of the unit before have been waited for, so the last reader of this
      // slot is done)
      int k_exp = 0;
      if (at_p_shift<T>() != 0.f) {
        const int other = slot - (u.i0 >> 7) + u.yt0;  // the ring's first tile
        k_exp = keys ? at_ds_exponent(p, w, u.h0, grp / split, other, u.nt, u.hk, slot, 1)
                     : at_ds_exponent(p, w, u.h, 1, slot, 1, u.hk, other, u.nt);
        if (lane == 0) {
          exponent[(tiles - 1) & 1] = k_exp;
          mbar_arrive(&exp_full[(tiles - 1) & 1]);
        }
      }
      const float sc = at_pow2(k_exp - int(at_p_shift<T>()));
      int hy = keys ? u.h0 : u.hk, yt = 0;
      for (int it = 0; it < u.n; ++it, ++loads) {
        const int s = loads & 1, y0 = (u.yt0 + yt) * AT_TILE;
        if (it > 0 && !load(hy, y0)) break;
        if (keys) {
          const float2* src = w.row + int64_t(hy) * p.tokens + u.a;
          float2 x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)  // p = 0 behind the end
            x[e] = y0 + e * 32 + lane < u.len ? src[y0 + e * 32 + lane] : make_float2(INFINITY, 0.f);
          if (!wait(&aux_empty[aux & 1], ((aux >> 1) & 1) ^ 1, 13)) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            aux_lse[(aux & 1) * AT_TILE + e * 32 + lane] = at_p_shift<T>() - x[e].x;
            aux_dl[(aux & 1) * AT_TILE + e * 32 + lane] = -x[e].y * sc;
          }
          ++aux;
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&a_full[s]);
        if (++yt == u.nt) {
          yt = 0;
          ++hy;
        }
      }
      if (!ok) break;
    }
    // the loads must have landed before the CTA's shared memory goes (see the forward)
    if (lane == 0) {
      if (tiles > 0) at_drain(xy_full, (tiles - 1) & 1);
      if (issued > loads) mbar_arrive(&a_full[loads & 1]);
      for (unsigned i = issued > 2 ? issued - 2 : 0; i < issued; ++i) {
        at_drain(&a_full[i & 1], (i >> 1) & 1);
        at_drain(&b_full[i & 1], (i >> 1) & 1);
      }
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- MMA
    const uint32_t lead = elect_one();
    const int kd = (p.head_dim + 15) / 16;
    const uint32_t id_g = at_idesc<T>(kd * 16, true);
    const uint64_t dx = smem_desc_sw128(sbase + L::X, 16, 1024), dy = smem_desc_sw128(sbase + L::Y, 16, 1024);
    const uint64_t da = smem_desc_sw128(sbase + L::A, 16, 1024), db = smem_desc_sw128(sbase + L::B, 16, 1024);
    const uint64_t ta = smem_desc_sw128(sbase + L::A, AT_BOX, 1024), tb = smem_desc_sw128(sbase + L::B, AT_BOX, 1024);
    constexpr uint64_t STEP = uint64_t(L::TILE >> 4);
    // d (128 x the ring tile's tokens) = x a^T over head_dim
    auto scores = [&](uint32_t d, uint64_t x, uint64_t a, int steps) {
      const uint32_t id = at_idesc<T>(steps * 16, false);
#pragma unroll
      for (int k = 0; k < DC * 4; ++k) {
        const uint64_t off = uint64_t((k >> 2) * (AT_BOX >> 4) + (k & 3) * 2);
        if (k < kd) at_mma_ss(lead, d, x + off, a + off, id, k > 0);
      }
    };
    // d (128 x head_dim) += p b over the ring tile's tokens; each half of the columns of p lies
    // at the start of its own half of the scores it overwrote
    auto sum = [&](uint32_t d, uint32_t pm, uint64_t b, bool acc, int steps) {
#pragma unroll
      for (int k = 0; k < AT_TILE / 16; ++k)
        if (k < steps) at_mma_ts(lead, d, pm + (k >> 2) * 64 + (k & 3) * 8, b + uint64_t(k * (2048 >> 4)), id_g, acc || k > 0);
    };
    unsigned r = 0, m = 0;  // ring items and units with tiles so far
    // S and dP of ring item i, overwriting P and dS of the one before: MMAs of one thread run in order
    auto s_of = [&](unsigned i, int steps) {
      if (!wait(&a_full[i & 1], (i >> 1) & 1, 16)) return false;
      tc_fence_after();
      scores(tmem + AT_TM_S, dx, da + (i & 1) * STEP, steps);
      at_commit(lead, s_full);
      return true;
    };
    auto dp_of = [&](unsigned i, bool keys, int steps) {
      if (!wait(&b_full[i & 1], (i >> 1) & 1, 17)) return false;
      tc_fence_after();
      scores(tmem + AT_TM_DP, dy, db + (i & 1) * STEP, steps);
      at_commit(lead, dp_full);
      if (!keys) at_commit(lead, &b_empty[i & 1]);
      return true;
    };
    // One unit's MMAs; a copy for each kind of dS (a test around the second product cost 5 % of a short backward).
    auto unit = [&](auto fine_tag, bool keys, int n, int nt, int tokens) {
      // MMAs over 16 tokens each: nothing behind the sequence's end
      int yt = 0, steps = (min(tokens, AT_TILE) + 15) >> 4;
      if (!wait(xy_full, m & 1, 18) || !s_of(r, steps) || !dp_of(r, keys, steps)) return;
      if (n == 1) at_commit(lead, xy_empty);
      for (int it = 0; it < n; ++it, ++r) {
        const bool more = it + 1 < n;
        if (++yt == nt) yt = 0;
        const int next = (min(tokens - yt * AT_TILE, AT_TILE) + 15) >> 4;
        if (!wait(p_ready, r & 1, 19)) return;
        // the sums of the unit before have been read
        if (it == 0 && !wait(acc_empty, (m & 1) ^ 1, 20)) return;
        tc_fence_after();
        if (keys) {
          sum(tmem + AT_TM_DV, tmem + AT_TM_S, tb + (r & 1) * STEP, it > 0, steps);
          at_commit(lead, &b_empty[r & 1]);
        }
        if (more && !s_of(r + 1, next)) return;
        if (!wait(ds_ready, r & 1, 21)) return;
        tc_fence_after();
        sum(tmem + AT_TM_DX, tmem + AT_TM_DP, ta + (r & 1) * STEP, it > 0, steps);
        if (decltype(fine_tag)::value) sum(tmem + AT_TM_DX, tmem + AT_TM_DP + 32, ta + (r & 1) * STEP, true, steps);
        at_commit(lead, &a_empty[r & 1]);
        if (more && !dp_of(r + 1, keys, next)) return;
        if (it + 2 == n) at_commit(lead, xy_empty);  // no more scores of this unit
        steps = next;
      }
      at_commit(lead, acc_full);
      ++m;
    };
    for (int k = 0;; ++k) {
      if (!wait(&unit_full[k & 1], (k >> 1) & 1, 15)) break;
      auto of_unit = [&](int v) { return __shfl_sync(0xffffffffu, v, 0); };
      const int kind = of_unit(units[k & 1].kind), n = of_unit(units[k & 1].n), nt = of_unit(units[k & 1].nt);
      const int fine = of_unit(units[k & 1].fine);
      const int tokens = of_unit(units[k & 1].len - units[k & 1].yt0 * AT_TILE);  // from the ring's first tile on
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[k & 1]);
      if (kind == AT_UNIT_END) break;
      if (kind == AT_UNIT_JOIN) continue;
      if (fine) unit(std::true_type{}, kind == AT_UNIT_KEYS, n, nt, tokens);
      else unit(std::false_type{}, kind == AT_UNIT_KEYS, n, nt, tokens);
      if (!ok) break;
    }
    at_commit(lead, drained);  // nothing in flight when TMEM and shared memory go
    at_drain(drained, 0);
  } else {
    // ---------------------------------------------------------------- elementwise
    const int half = warp >> 2;  // columns [64 half, 64 half + 64)
    const int w0 = (warp & 3) * 32, row = w0 + lane;
    const uint32_t lane_off = uint32_t(w0) << 16;
    const uint32_t t_s = tmem + AT_TM_S + lane_off + half * 64, t_dp = tmem + AT_TM_DP + lane_off + half * 64;
    const float sl2 = p.scale * AT_LOG2E;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    uint8_t* buf = smem + L::OUT + warp * 2048;
    unsigned r = 0, aux = 0, m = 0;
    // One unit's ring items.
    int k_exp = 0;
    auto items = [&](auto keys_tag, auto fine_tag, const AttnUnit& u) {
      constexpr bool KEYS = decltype(keys_tag)::value, FINE = decltype(fine_tag)::value;
      const int x = u.i0 + row;  // this thread's row, relative to a
      float sc = 1.f;
      const int back = KEYS ? p.right : p.left, ahead = KEYS ? p.left : p.right;
      const int see_lo = back < 0 ? 0 : x - back, x0 = u.i0 + w0;
      const int see_hi = ahead < 0 ? u.len - 1 : min(u.len - 1, x + ahead);
      // what all, and what any of the warp's rows see
      const int lo_max = back < 0 ? 0 : x0 + 31 - back, lo_min = back < 0 ? 0 : x0 - back;
      const int hi_min = ahead < 0 ? u.len - 1 : min(u.len - 1, x0 + ahead);
      const int hi_max = ahead < 0 ? u.len - 1 : min(u.len - 1, x0 + 31 + ahead);
      uint64_t row_lse = 0;  // twice
      float row_dl = 0.f;
      if (!KEYS) {
        const float2 v = x < u.len ? w.row[int64_t(u.h) * p.tokens + u.a + x] : make_float2(INFINITY, 0.f);
        row_lse = f2_pack(at_p_shift<T>() - v.x, at_p_shift<T>() - v.x);
        row_dl = -v.y;
      }
      auto scale = [&](int it) {
        if (it > 0) return true;
        if (at_p_shift<T>() != 0.f) {
          if (!wait(&exp_full[m & 1], (m >> 1) & 1, 29)) return false;
          k_exp = exponent[m & 1];
        }
        sc = at_pow2(k_exp - int(at_p_shift<T>()));
        row_dl *= sc;
        return true;
      };
      int yt = 0;
      for (int it = 0; it < u.n; ++it, ++r) {
        const int s = r & 1, sa = aux & 1;
        const int tile0 = (u.yt0 + yt) * AT_TILE, y0 = tile0 + half * 64;
        if (++yt == u.nt) yt = 0;
        if (!wait(s_full, r & 1, 22)) return;
        tc_fence_after();
        // rows of other sequences behind a ragged ring tile must add nothing to a sum over its tokens: Q's and dO's
        // for a key tile, K's for a query tile (V only meets scores that are masked).  The scores that read the
        // tiles are done by then.
        auto cut_tile = [&] {
          const int end = u.len - tile0;
          if (end >= AT_TILE) return true;
          if (KEYS) {
            if (!wait(dp_full, r & 1, 14)) return false;
            at_zero_rows<DC, AT_TILE, 256>(smem + L::B + s * L::TILE, end, threadIdx.x);
          }
          at_zero_rows<DC, AT_TILE, 256>(smem + L::A + s * L::TILE, end, threadIdx.x);
          fence_proxy_async_smem();
          return true;
        };
        // no token in this half (no MMA reads it), or none that the warp's rows see
        if (y0 >= u.len || y0 + 63 < lo_min || y0 > hi_max) {
          uint32_t zeros[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) zeros[c] = 0;
          if (KEYS) {
            tmem_st_32x32b_x32(t_s, zeros);
            tmem_st_wait();
          }
          if (!cut_tile()) return;
          tc_fence_before();
          mbar_arrive(p_ready);
          if (!scale(it) || !wait(dp_full, r & 1, 24)) return;
          tc_fence_after();
          tmem_st_32x32b_x32(t_dp, zeros);
          if (FINE) tmem_st_32x32b_x32(t_dp + 32, zeros);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(ds_ready);
          if (KEYS) {
            if (lane == 0) mbar_arrive(&aux_empty[sa]);
            ++aux;
          }
          continue;
        }
        uint32_t sv[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(t_s + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + c * 32));
        tmem_ld_wait();
        if (!KEYS) {
          tc_fence_before();
          mbar_arrive(p_ready);  // the scores are in registers: the next tile's may overwrite them
        }
        uint64_t pv[32];
        const ulonglong2* la = reinterpret_cast<const ulonglong2*>(aux_lse + sa * AT_TILE + half * 64);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          ulonglong2 l4 = make_ulonglong2(row_lse, row_lse);
          if (KEYS) l4 = la[c];
          const float2 f = f2_unpack(f2_fma(f2_pack_u(sv[4 * c], sv[4 * c + 1]), sl2x2, l4.x));
          const float2 g = f2_unpack(f2_fma(f2_pack_u(sv[4 * c + 2], sv[4 * c + 3]), sl2x2, l4.y));
          pv[2 * c] = f2_pack(at_exp2(f.x), at_exp2(f.y));
          pv[2 * c + 1] = f2_pack(at_exp2(g.x), at_exp2(g.y));
        }
        auto hide = [&] {  // 0 where the pair is not visible, whatever is there
          at_hide(see_lo - y0, see_hi - y0, [&](int c) {
            const float2 v = f2_unpack(pv[c >> 1]);
            pv[c >> 1] = c & 1 ? f2_pack(v.x, 0.f) : f2_pack(0.f, v.y);
          });
        };
        if (y0 < lo_max || y0 + 63 > hi_min) hide();
        if (!cut_tile()) return;
        auto put = [&](uint32_t taddr) {  // rounded to the MMA's operand type
          uint32_t pk[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float2 v = f2_unpack(pv[k]);
            pk[k] = at_pack<T>(v.x, v.y);
          }
          tmem_st_32x32b_x32(taddr, pk);
          tmem_st_wait();
          tc_fence_before();
        };
        auto put_rest = [&](uint32_t taddr) {  // what that rounding leaves, rounded again
          uint32_t pk[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float2 v = f2_unpack(pv[k]), w = at_unpack<T>(at_pack<T>(v.x, v.y));
            pk[k] = at_pack<T>(v.x - w.x, v.y - w.y);
          }
          tmem_st_32x32b_x32(taddr, pk);
        };
        if (KEYS) {
          put(t_s);
          mbar_arrive(p_ready);
        }
        if (!scale(it) || !wait(dp_full, r & 1, 24)) return;
        tc_fence_after();
        const uint64_t scx2 = f2_pack(sc, sc), row_dl2 = f2_pack(row_dl, row_dl);
        uint32_t dpv[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(t_dp + c * 32, *reinterpret_cast<uint32_t(*)[32]>(dpv + c * 32));
        tmem_ld_wait();
        const ulonglong2* ld = reinterpret_cast<const ulonglong2*>(aux_dl + sa * AT_TILE + half * 64);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          ulonglong2 d4 = make_ulonglong2(row_dl2, row_dl2);
          if (KEYS) d4 = ld[c];
          pv[2 * c] = f2_mul(pv[2 * c], f2_fma(f2_pack_u(dpv[4 * c], dpv[4 * c + 1]), scx2, d4.x));
          pv[2 * c + 1] = f2_mul(pv[2 * c + 1], f2_fma(f2_pack_u(dpv[4 * c + 2], dpv[4 * c + 3]), scx2, d4.y));
        }
        if (y0 + 64 > u.len) hide();  // tokens of another sequence (inside this one p = 0 has done it)
        if (FINE) put_rest(t_dp + 32);
        put(t_dp);
        mbar_arrive(ds_ready);
        if (KEYS) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&aux_empty[sa]);
          ++aux;
        }
      }
    };
    for (int k = 0;; ++k) {
      if (!wait(&unit_full[k & 1], (k >> 1) & 1, 25)) break;
      const AttnUnit u = units[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[k & 1]);
      if (u.kind == AT_UNIT_END) break;
      if (u.kind == AT_UNIT_JOIN) {
        // piece u.rank of the features of [dK | dV], share by share; thread: a row, half of the piece
        constexpr int N = DC * 32 / AT_PIECES / 2;  // groups of four features
        const int jr = threadIdx.x & (AT_TILE - 1), g0 = (u.rank * 2 + (threadIdx.x >> 7)) * N;
        const float4* from = at_part<DC>(w.parts, u.join, split, 0) + g0 * AT_TILE + jr;
        const int f0 = g0 * 4 & (DC * 64 - 1);
        if (jr < u.len - u.i0 && f0 < p.head_dim) {
          float4 v[N];
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = __ldcg(from + e * AT_TILE);
#pragma unroll 2
          for (int q = 1; q < split; ++q) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float4 y = __ldcg(from + (int64_t(q) * (DC * 32) + e) * AT_TILE);
              v[e].x += y.x, v[e].y += y.y, v[e].z += y.z, v[e].w += y.w;
            }
          }
          T* to = (g0 < DC * 16 ? dk : dv) + (int64_t(u.a + u.i0 + jr) * p.kv_heads + u.h) * p.head_dim + f0;
#pragma unroll
          for (int e = 0; e < N; e += 2)
            if (f0 + e * 4 < p.head_dim)
              *reinterpret_cast<uint4*>(to + e * 4) =
                  make_uint4(at_pack<T>(v[e].x, v[e].y), at_pack<T>(v[e].z, v[e].w), at_pack<T>(v[e + 1].x, v[e + 1].y),
                             at_pack<T>(v[e + 1].z, v[e + 1].w));
        }
        continue;
      }
      const bool keys = u.kind == AT_UNIT_KEYS;
      if (keys) {
        if (u.fine) items(std::true_type{}, std::true_type{}, u);
        else items(std::true_type{}, std::false_type{}, u);
      } else {
        if (u.fine) items(std::false_type{}, std::true_type{}, u);
        else items(std::false_type{}, std::false_type{}, u);
      }
      if (!ok || !wait(acc_full, m & 1, 26)) break;
      ++m;
      tc_fence_after();
      const int rows = u.len - u.i0 - w0;  // of this warp's 32
      const float fx = p.scale * at_pow2(-k_exp);
      if (!keys) {
        const int c0 = half * DC * 32;
        T* to = dq + (int64_t(u.a + u.i0 + w0) * p.heads + u.h) * p.head_dim + c0;
#pragma unroll
        for (int c = 0; c < DC * 32; c += 32)
          at_store_rows<T, 32>(tmem + AT_TM_DX + lane_off + c0 + c, buf, to + c, int64_t(p.heads) * p.head_dim, rows,
                               p.head_dim - c0 - c, fx);
      } else {
        const uint32_t from = tmem + (half == 0 ? AT_TM_DX : AT_TM_DV) + lane_off;
        const float f = half == 0 ? fx : at_pow2(-int(at_p_shift<T>()));
        if (split == 1) {
          T* to = (half == 0 ? dk : dv) + (int64_t(u.a + u.i0 + w0) * p.kv_heads + u.h) * p.head_dim;
#pragma unroll
          for (int c = 0; c < DC * 64; c += 32)
            at_store_rows<T, 32>(from + c, buf, to + c, int64_t(p.kv_heads) * p.head_dim, rows, p.head_dim - c, f);
        } else if (rows > 0) {
          float4* mine = at_part<DC>(w.parts, u.join, split, u.rank) + half * DC * 16 * AT_TILE + row;
#pragma unroll
          for (int c = 0; c < DC * 64; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(from + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              mine[(c + e) / 4 * AT_TILE] = make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f,
                                                        __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(acc_empty);
      if (keys && split > 1) {  // this warp's part of the share is in memory
        __threadfence();
        __syncwarp();
        if (lane == 0) atomicAdd(w.tickets + u.join, 1u);
      }
    }
    __syncwarp();
    tmem_st_wait();  // (a warp that gave up may have stores under way)
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (warp == 8 && *abort_flag) {
    // A wait ran out: NaN in the rows of the units under way (four at most: the one whose sums are read, one
    // with its MMAs, one published, one just taken), and of all that this CTA can still take, so that
    // none is left unwritten.  A lost share of a key tile's heads lets the wait of its sum run out.
    auto poison = [&](const AttnUnit& u) {
      const int64_t row = u.a + u.i0, n = min(AT_TILE, u.len - u.i0);
      if (u.kind == AT_UNIT_QUERIES) {
        at_poison_rows(dq + (row * p.heads + u.h) * p.head_dim, int64_t(p.heads) * p.head_dim, n, p.head_dim, lane, 32);
      } else if (u.kind == AT_UNIT_JOIN || (u.kind == AT_UNIT_KEYS && split == 1)) {
        const int64_t off = (row * p.kv_heads + u.h) * p.head_dim, stride = int64_t(p.kv_heads) * p.head_dim;
        at_poison_rows(dk + off, stride, n, p.head_dim, lane, 32);
        at_poison_rows(dv + off, stride, n, p.head_dim, lane, 32);
      }
    };
    for (int i = 0; i < 4; ++i) poison(taken[i]);
    const AttnUnits order(p, split);
    for (;;) {
      unsigned at = 0;
      if (lane == 0) at = atomicAdd(w.next, 1u);
      at = __shfl_sync(0xffffffffu, at, 0);
      if (at >= order.n_all) break;
      AttnUnit u;
      int slot = 0;
      if (at_unit(p, order, split, at, u, slot)) poison(u);
    }
  }
}

static bool attn_strides_ok(int64_t stride, int64_t head_stride, const nf4b_attn& a) {
  return stride >= a.head_dim && head_stride >= a.head_dim && stride % 8 == 0 && head_stride % 8 == 0 &&
         stride < (int64_t(1) << 38) && head_stride < (int64_t(1) << 38);
}

// Checks the call and writes its normalised form (window bounds cut to the token count, so that
// index + bound stays in 32 bits).
static int attn_checks(const nf4b_attn* in, nf4b_attn* a) {
  NF4B_RETURN_IF(in == nullptr, NF4B_ERR_INVALID_ARG);
  *a = *in;
  NF4B_RETURN_IF(a->tokens < 0 || a->rows < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->head_dim <= 0,
                 NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(a->heads % a->kv_heads != 0, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!(a->scale > 0.f && a->scale < 0x1p127f), NF4B_ERR_INVALID_ARG);  // scale log2(e) is fp32, too
  NF4B_RETURN_IF(a->dtype != NF4B_F16 && a->dtype != NF4B_BF16, NF4B_ERR_UNSUPPORTED);
  NF4B_RETURN_IF(a->head_dim % 8 != 0 || a->head_dim > AT_MAX_DIM, NF4B_ERR_UNSUPPORTED);
  NF4B_RETURN_IF(a->tokens > 0x3FFFFFFF || a->rows > 0x3FFFFFFF || a->heads > 65535, NF4B_ERR_UNSUPPORTED);
  // CTAs of a launch
  NF4B_RETURN_IF(at_slots(a->tokens, a->rows) * (2 + AT_PIECES) * a->heads > 0x3FFFFFFF, NF4B_ERR_UNSUPPORTED);
  if (a->tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!a->q || !a->k || !a->v || !a->cu, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cu, 4), NF4B_ERR_ALIGNMENT);
  // a dimension of one element may carry any stride
  if (a->tokens == 1) a->q_stride = a->k_stride = a->v_stride = int64_t(a->heads) * a->head_dim;
  if (a->heads == 1) a->q_head_stride = a->head_dim;
  if (a->kv_heads == 1) a->k_head_stride = a->v_head_stride = a->head_dim;
  NF4B_RETURN_IF(!attn_strides_ok(a->q_stride, a->q_head_stride, *a) || !attn_strides_ok(a->k_stride, a->k_head_stride, *a) ||
                     !attn_strides_ok(a->v_stride, a->v_head_stride, *a),
                 NF4B_ERR_ALIGNMENT);
  a->left = a->left < 0 || a->left >= a->tokens ? -1 : a->left;
  a->right = a->right < 0 || a->right >= a->tokens ? -1 : a->right;
  return NF4B_OK;
}

}  // namespace nf4b

using namespace nf4b;

// [tokens][heads][head_dim] as 64-feature boxes of `rows` tokens of one head, 128-byte swizzle, zeros
// outside the tensor.
static int attn_tmap(CUtensorMap* m, const nf4b_attn& a, const void* base, int heads, int64_t stride, int64_t head_stride,
                     int rows) {
  const uint64_t dims[3] = {uint64_t(a.head_dim), uint64_t(heads), uint64_t(a.tokens)};
  const uint64_t strides[2] = {uint64_t(head_stride) * 2, uint64_t(stride) * 2};
  const uint32_t box[3] = {64, 1, uint32_t(rows)};
  return make_tmap_tiled(m, a.dtype == NF4B_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Clocks after which a wait of the kernels gives up.  STEW_ATTN_WAIT_CYCLES sets another limit (0: a wait that
// is not over when it begins gives up), to see what a caller gets then.
static long long attn_wait_cycles() {
  const char* v = std::getenv("STEW_ATTN_WAIT_CYCLES");
  if (v == nullptr || v[0] < '0' || v[0] > '9') return kAttnWaitCycles;
  const long long c = std::atoll(v);
  return c < kAttnWaitCycles ? c : kAttnWaitCycles;
}

static AttnParams attn_params(const nf4b_attn& a) {
  return AttnParams{a.cu,       int32_t(a.tokens), a.rows,  a.heads, a.kv_heads,
                    a.head_dim, a.left,            a.right, int32_t(at_slots(a.tokens, a.rows)), a.scale, attn_wait_cycles()};
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
static int attn_fwd_launch(const nf4b_attn& a, void* out, void* rest, float* lse, cudaStream_t s) {
  CUtensorMap q, k, v;
  int st = attn_tmap(&q, a, a.q, a.heads, a.q_stride, a.q_head_stride, AT_TILE);
  if (st == NF4B_OK) st = attn_tmap(&k, a, a.k, a.kv_heads, a.k_stride, a.k_head_stride, AT_KEYS);
  if (st == NF4B_OK) st = attn_tmap(&v, a, a.v, a.kv_heads, a.v_stride, a.v_head_stride, AT_KEYS);
  static bool done[64] = {false};
  if (st == NF4B_OK) st = attn_smem(attn_fwd_kernel<T, DC>, AttnFwdSmem<DC>::ALLOC, done);
  if (st != NF4B_OK) return st;
  const AttnParams p = attn_params(a);
  NF4B_CUDA_TRY(launch_pdl(attn_fwd_kernel<T, DC>, dim3(unsigned(p.slots) * unsigned(a.heads)), dim3(AT_FWD_THREADS),
                           size_t(AttnFwdSmem<DC>::ALLOC), s, q, k, v, p, static_cast<T*>(out), static_cast<T*>(rest), lse));
  return launch_status("attn_fwd_kernel launch");
}

extern "C" int nf4b_attn_fwd(const nf4b_attn* args, void* out, void* rest, float* lse, void* stream) {
  nf4b_attn a;
  int st = attn_checks(args, &a);
  if (st != NF4B_OK) return st;
  if (a.tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!out || !lse, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(out, 16) || !aligned(rest, 16) || !aligned(lse, 16), NF4B_ERR_ALIGNMENT);
  st = check_device();
  if (st != NF4B_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = a.head_dim > 64;
  if (a.dtype == NF4B_F16)
    return wide ? attn_fwd_launch<__half, 2>(a, out, rest, lse, s) : attn_fwd_launch<__half, 1>(a, out, rest, lse, s);
  return wide ? attn_fwd_launch<__nv_bfloat16, 2>(a, out, rest, lse, s) : attn_fwd_launch<__nv_bfloat16, 1>(a, out, rest, lse, s);
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

static int attn_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();  // (no device: the scratch may be asked for all the same)
    return 148;
  }
  if (cached[dev] == 0) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = v > 0 ? v : 148;
  }
  return cached[dev];
}

// CTAs that share a key tile's heads: the divisor of the group with the shortest estimated time on the device's
// SMs, from an average sequence: the longer of all units' work shared out and the longest key-tile unit.  In
// microseconds, as measured: about 3 of start and store for a unit, 2 more for a shared one, 1.6 a key-tile
// step, 1.2 a query-tile step.
static int attn_split(const nf4b_attn& a) {
  const int grp = a.heads / a.kv_heads;
  const double len = double(a.tokens) / (a.rows > 0 ? a.rows : 1);
  const double seen_max = (a.left < 0 ? len : a.left) + (a.right < 0 ? len : a.right) + 1;
  const double most = (seen_max < len ? seen_max : len) / AT_TILE + 1;                          // tiles a key tile meets
  const double mean = (a.left < 0) != (a.right < 0) && most * AT_TILE > len ? (most + 1) / 2 : most;
  const double tiles = double(a.tokens) / AT_TILE + 0.5 * a.rows;
  // (the shares' sums take 128 KB each: half a GB at most)
  auto fits = [&](int c) { return grp % c == 0 && (c == 1 || at_slots(a.tokens, a.rows) * a.kv_heads * c <= 4096); };
  const int sms = attn_sms();
  int best = 1;
  double best_us = 0;
  for (int c = 1; c <= grp; ++c) {
    if (!fits(c)) continue;
    const double one = 3.0 + (c > 1 ? 2.0 : 0.0);
    const double keys = tiles * a.kv_heads * c * (one + 1.6 * mean * (grp / c));
    const double queries = tiles * a.heads * (3.0 + 1.2 * mean);
    const double all = (keys + queries) / sms, longest = one + 1.6 * most * (grp / c);
    const double us = all > longest ? all : longest;
    if (c == 1 || us < best_us) {
      best = c;
      best_us = us;
    }
  }
  const char* v = std::getenv("STEW_ATTN_SPLIT");
  if (v != nullptr && v[0] >= '1' && v[0] <= '9' && fits(v[0] - '0')) best = v[0] - '0';
  return best;
}

static int64_t attn_work(const nf4b_attn& a, int split, void* base, AttnWork* w) {
  const int64_t slots = at_slots(a.tokens, a.rows), pairs = slots * a.kv_heads;
  char* b = static_cast<char*>(base);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* here = b + at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  AttnWork x;
  x.row = reinterpret_cast<float2*>(take(a.heads * a.tokens * 8));
  x.tile = reinterpret_cast<float2*>(take(a.heads * slots * 8));
  x.vmax = reinterpret_cast<float*>(take(pairs * 4));
  x.next = reinterpret_cast<unsigned*>(take(4));
  x.tickets = reinterpret_cast<unsigned*>(take(pairs * 4));
  x.parts = reinterpret_cast<float*>(take(split > 1 ? pairs * split * AT_TILE * (a.head_dim > 64 ? 256 : 128) * 4 : 0));
  if (w != nullptr) *w = x;
  return at;
}

extern "C" int64_t nf4b_attn_bwd_work_bytes(const nf4b_attn* args) {
  nf4b_attn a;
  if (attn_checks(args, &a) != NF4B_OK) return -1;
  return attn_work(a, attn_split(a), nullptr, nullptr);
}

template <typename T, int DC>
static int attn_bwd_launch(const nf4b_attn& a, const void* out, const void* rest, const float* lse, const void* dout, void* dq, void* dk,
                           void* dv, void* work, int split, cudaStream_t s) {
  AttnBwdMaps m;
  int st = attn_tmap(&m.q, a, a.q, a.heads, a.q_stride, a.q_head_stride, AT_TILE);
  if (st == NF4B_OK) st = attn_tmap(&m.k, a, a.k, a.kv_heads, a.k_stride, a.k_head_stride, AT_TILE);
  if (st == NF4B_OK) st = attn_tmap(&m.v, a, a.v, a.kv_heads, a.v_stride, a.v_head_stride, AT_TILE);
  if (st == NF4B_OK) st = attn_tmap(&m.dout, a, dout, a.heads, int64_t(a.heads) * a.head_dim, a.head_dim, AT_TILE);
  static bool done[64] = {false};
  if (st == NF4B_OK) st = attn_smem(attn_bwd_kernel<T, DC>, AttnBwdSmem<DC>::ALLOC, done);
  if (st != NF4B_OK) return st;
  const AttnParams p = attn_params(a);
  AttnWork w;
  attn_work(a, split, work, &w);
  T *tq = static_cast<T*>(dq), *tk = static_cast<T*>(dk), *tv = static_cast<T*>(dv);
  NF4B_CUDA_TRY(launch_pdl(attn_prep_kernel<T>, dim3(unsigned(p.slots) * unsigned(a.heads + a.kv_heads)),
                           dim3(AT_PREP_THREADS),
                           size_t(0), s, p, static_cast<const T*>(out), static_cast<const T*>(rest), static_cast<const T*>(dout), lse,
                           static_cast<const T*>(a.v), a.v_stride, a.v_head_stride, w, tq, tk, tv));
  const int64_t units = int64_t(p.slots) * (int64_t(a.kv_heads) * (split > 1 ? split + AT_PIECES : 1) + a.heads);
  const int64_t sms = attn_sms();
  NF4B_CUDA_TRY(launch_pdl(attn_bwd_kernel<T, DC>, dim3(unsigned(units < sms ? units : sms)), dim3(AT_BWD_THREADS),
                           size_t(AttnBwdSmem<DC>::ALLOC), s, m, p, w, split, tq, tk, tv));
  return launch_status("attn_bwd_kernel launch");
}

extern "C" int nf4b_attn_bwd(const nf4b_attn* args, const void* out, const void* rest, const float* lse,
                             const void* dout, void* dq, void* dk, void* dv, void* work, int64_t work_bytes, void* stream) {
  nf4b_attn a;
  int st = attn_checks(args, &a);
  if (st != NF4B_OK) return st;
  if (a.tokens == 0) return NF4B_OK;
  NF4B_RETURN_IF(!out || !lse || !dout || !dq || !dk || !dv || !work, NF4B_ERR_INVALID_ARG);
  NF4B_RETURN_IF(!aligned(out, 16) || !aligned(rest, 16) || !aligned(lse, 16) || !aligned(dout, 16) || !aligned(dq, 16) || !aligned(dk, 16) ||
                     !aligned(dv, 16) || !aligned(work, 16),
                 NF4B_ERR_ALIGNMENT);
  const int split = attn_split(a);
  NF4B_RETURN_IF(work_bytes < attn_work(a, split, nullptr, nullptr), NF4B_ERR_INVALID_ARG);
  st = check_device();
  if (st != NF4B_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto tag, auto dc) {
    using T = decltype(tag);
    return attn_bwd_launch<T, decltype(dc)::value>(a, out, rest, lse, dout, dq, dk, dv, work, split, s);
  };
  auto typed = [&](auto tag) {
    return a.head_dim > 64 ? launch(tag, std::integral_constant<int, 2>()) : launch(tag, std::integral_constant<int, 1>());
  };
  return a.dtype == NF4B_F16 ? typed(__half()) : typed(__nv_bfloat16());
}
