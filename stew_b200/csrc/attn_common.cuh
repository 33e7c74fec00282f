// Shared pieces of the attention kernels (attention.cu): the split of the packed rows into tiles,
// the tensor-memory and TMA wrappers beyond common.cuh's, bounded waits, conversions.
#pragma once

#include <cuda_bf16.h>
#include <math.h>

#include "common.cuh"
#include "stew_step.h"

namespace nf4b {

constexpr int AT_TILE = 128;      // tokens of a query or key tile: the MMA's M, and N of the scores
constexpr int AT_MAX_DIM = 128;
constexpr int AT_BOX = AT_TILE * 128;  // bytes of a TMA box: 128 tokens x 64 features (one 128-byte swizzle row each)
constexpr float AT_LOG2E = 1.4426950408889634f;

// What the kernels need of an nf4b_attn.
struct AttnParams {
  const int32_t* cu;
  int32_t tokens, rows, heads, kv_heads, head_dim;
  int32_t left, right;
  int32_t slots;       // tile slots of the packed rows, at_slots()
  float scale;
  long long wait_cycles;  // limit of a wait, in clocks
};

// Tiles never cross a sequence.  Sequence s owns the tile slots from floor(start_s / 128) + s on: that many
// hold its tiles for any lengths (floor(b/128) - floor(a/128) + 1 >= ceil((b-a)/128)), so the launch needs
// only the token and row counts, and a CTA finds its sequence by searching a strictly ascending function
// of s.  Slots from that of s = rows on cover the rows behind the last sequence.
inline int64_t at_slots(int64_t tokens, int64_t rows) { return tokens / AT_TILE + rows + 1; }

struct AttnTile {
  int a, len;   // the sequence's first token and length
  int i0;       // the tile's first token, relative to a
  bool tail;    // rows behind the last sequence (a, len: that range)
};

// cu[0] is taken as 0; other values are cut to [0, tokens], so no index leaves the tensors.
__device__ __forceinline__ int at_start(const AttnParams& p, int s) {
  return s == 0 ? 0 : min(max(__ldg(p.cu + s), 0), p.tokens);
}
__device__ __forceinline__ int at_first_slot(const AttnParams& p, int s) { return (at_start(p, s) >> 7) + s; }

// Whole warp; 32 probes a step (one step for up to 31 sequences).
__device__ __forceinline__ AttnTile at_find(const AttnParams& p, int slot) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.rows + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int s = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, s < hi && at_first_slot(p, s) <= slot);
    lo += (below == 0xffffffffu ? 31 : max(__ffs(~below) - 2, 0)) * step;
    hi = min(hi, lo + step);
  }
  AttnTile t;
  t.tail = lo == p.rows;
  t.a = at_start(p, lo);
  t.len = (t.tail ? p.tokens : max(at_start(p, lo + 1), t.a)) - t.a;
  t.i0 = (slot - ((t.a >> 7) + lo)) << 7;
  return t;
}

template <typename T>
__device__ __forceinline__ uint32_t at_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t at_pack<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t at_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 at_unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 at_unpack<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <>
__device__ __forceinline__ float2 at_unpack<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

__device__ __forceinline__ float at_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one 64-bit register: half the issue slots of the scalar forms.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_pack_u(uint32_t a, uint32_t b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t d) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(d));
  return v;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Instruction descriptor of kind::f16 for T (A and B of the same type), fp32 accumulation.
template <typename T>
__host__ __device__ constexpr uint32_t at_idesc(int n, bool b_mn_major);
template <>
constexpr uint32_t at_idesc<__half>(int n, bool b_mn_major) { return idesc_f16(AT_TILE, n, false, b_mn_major); }
template <>
constexpr uint32_t at_idesc<__nv_bfloat16>(int n, bool b_mn_major) {
  return idesc_f16(AT_TILE, n, false, b_mn_major) | (1u << 7) | (1u << 10);
}

// The MMA warp runs its loop as a whole, so that descriptors stay in uniform registers, and one lane's
// predicate issues: inside a one-lane branch each MMA took 80-100 clocks to issue, longer than to run.
// D[tmem] (+)= A[smem] . B[smem]^T.
__device__ __forceinline__ void at_mma_ss(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]^T: A holds two 16-bit values of a row per 32-bit column.
__device__ __forceinline__ void at_mma_ts(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void at_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// One lane of a whole warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(lead));
  return lead;
}

// 32 lanes x 32 columns of 32-bit values into TMEM (the layout of tmem_ld_32x32b_x32).
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// N threads (this one `id`): zeros in the rows from `first` to the next multiple of 16 (the tokens of one
// MMA; those behind it are not multiplied) of a [ROWS tokens][DC x 64 features] tile that has arrived, so
// that the rows of other sequences behind a ragged tile add nothing to a product over tokens (0 x their NaN
// would).  The 128-byte swizzle permutes inside a row only.  (The caller makes the writes visible to the
// MMAs: fence_proxy_async_smem.)
template <int DC, int ROWS, int N>
__device__ __forceinline__ void at_zero_rows(uint8_t* tile, int first, int id) {
#pragma unroll
  for (int c = 0; c < DC; ++c)
    for (int at = first * 128 + id * 16; at < ((first + 15) & ~15) * 128; at += N * 16)
      *reinterpret_cast<uint4*>(tile + c * ROWS * 128 + at) = make_uint4(0, 0, 0, 0);
}

// kill(c) for the columns c of [0, 64) outside [lo, hi], from bit masks (a test and a select a column).
template <typename F>
__device__ __forceinline__ void at_hide(int lo, int hi, F kill) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int l = min(max(lo - 32 * w, 0), 32), h = min(max(hi + 1 - 32 * w, 0), 32);  // bits [l, h) stay
    const uint32_t keep = (h == 32 ? 0xffffffffu : (1u << h) - 1u) & (l == 32 ? 0u : 0xffffffffu << l);
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (!(keep >> c & 1u)) kill(w * 32 + c);
  }
}

// What is left of v after its rounding to T.
template <typename T>
__device__ __forceinline__ float at_rest(float v) {
  const float2 r = at_unpack<T>(at_pack<T>(v, 0.f));
  return v - r.x;
}

// Whole warp: `cols` fp32 columns (a multiple of 8, at most MAX) from TMEM column `taddr` on of the warp's 32
// rows, row r times its thread's f, rounded to T and written to out + r * stride for r < rows.  The rows pass
// through `buf` (32 x 2 MAX bytes of shared memory, the 16-byte pieces of a row permuted by its number against
// bank conflicts), so that a warp writes whole rows instead of 16 bytes of each of 32.  REST: what the rounding
// left, instead.
template <typename T, int MAX, bool REST = false>
__device__ __forceinline__ void at_store_rows(uint32_t taddr, uint8_t* buf, T* out, int64_t stride, int rows, int cols, float f) {
  const int lane = threadIdx.x & 31;
  constexpr int VEC = MAX / 8;  // 16-byte pieces of a row: 4, 8 or 16
  __syncwarp();  // the rows before are out
  auto place = [&](int r, int c) { return buf + r * (2 * MAX) + (c ^ (VEC >= 8 ? r & 7 : (r >> 1) & 3)) * 16; };
#pragma unroll
  for (int c = 0; c < MAX; c += 32) {
    uint32_t o[32];
    tmem_ld_32x32b_x32(taddr + c, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 v;
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = __uint_as_float(o[k * 8 + 2 * e]) * f, b = __uint_as_float(o[k * 8 + 2 * e + 1]) * f;
        w[e] = REST ? at_pack<T>(at_rest<T>(a), at_rest<T>(b)) : at_pack<T>(a, b);
      }
      *reinterpret_cast<uint4*>(place(lane, c / 8 + k)) = v;
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int i = k * 32 + lane, r = i / VEC, c = i % VEC;
    if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(out + r * stride + c * 8) = *reinterpret_cast<const uint4*>(place(r, c));
  }
}

// Bounded waits: after `limit` clocks (about two seconds) the CTA's abort flag is raised, g_attn_error records
// where, and every role winds down.
__device__ int g_attn_error;

constexpr long long kAttnWaitCycles = 4000000000ll;

struct AttnWait {
  volatile int* abort;  // in shared memory, of the CTA
  long long limit;
};

__device__ __forceinline__ bool at_wait_slow(uint64_t* bar, uint32_t parity, const AttnWait& w, int where) {
  const long long t0 = clock64();
  for (;;) {
    if (w.limit > 0 && mbar_try_wait_sleep(bar, parity, 1000000u)) return true;
    if (*w.abort) return false;
    if (clock64() - t0 >= w.limit) {
      *w.abort = 1;
      atomicExch(&g_attn_error, where);
      return false;
    }
  }
}
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, const AttnWait& w, int where) {
  if (mbar_test_wait(bar, parity)) return true;
  return at_wait_slow(bar, parity, w, where);
}
// Waits for work in flight whatever the abort flag and the limit say.
__device__ __forceinline__ void at_drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait_sleep(bar, parity, 1000000u)) {
    if (clock64() - t0 > kAttnWaitCycles) {
      atomicExch(&g_attn_error, 99);
      return;
    }
  }
}

// NaN in `rows` rows of head_dim values: what a CTA whose wait ran out leaves of the rows that are its own.
// Thread `id` of `n`.
template <typename T>
__device__ __forceinline__ void at_poison_rows(T* to, int64_t stride, int rows, int head_dim, int id, int n) {
  const int vec = head_dim / 8;
  const uint32_t nan2 = 0x7fff7fffu;  // two NaN of either 16-bit type
  for (int i = id; i < rows * vec; i += n)
    *reinterpret_cast<uint4*>(to + (i / vec) * stride + (i % vec) * 8) = make_uint4(nan2, nan2, nan2, nan2);
}

}  // namespace nf4b
