// Shared pieces of the decoder's attention kernels (decoder_attention_forward.cu,
// decoder_attention_backward.cu).  For batch entry b, head h with shared head g = h / rep,
// query i and key j:
//
//   x = scale q_i.k_j,   z = cap tanh(x / cap)  (cap > 0; else z = x),
//   s = z - slope_{b,i,h} |qpos_i - kpos_j|     (|.| the Euclidean distance in 1 or 2 coordinates)
//   allowed when j < k_len[b] and segment(i) == segment(j) >= 0; everything else has weight 0.
//
// All exponentials are of base 2: the factor log2(e) is folded into the scale, the cap and the
// slopes on the way in, and taken out of the log-sum-exp on the way out.
#pragma once

#include <cuda.h>
#include <limits.h>

#include <type_traits>

#include "decoder_types.cuh"
#include "tc_ptx.cuh"

namespace s4d {

constexpr int kAttnRows = 128;      // rows of a tile = tensor-memory lanes
constexpr int kAttnMaxTiles = 8192; // tiles of the other axis one CTA walks (its table of tile kinds)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  const void* q;
  int64_t q_sb, q_sn, q_sh;  // element strides of batch, row and head
  const void* v;             // (forward)
  int64_t v_sb, v_sn, v_sh;
  const void* dout;
  int64_t do_sb, do_sn, do_sh;
  void* out;   // [B, Nq, H, D] contiguous (backward: read)
  float* lse;  // [B, H, Nq], natural logarithm (backward: read)
  const float* slopes;
  int64_t sl_b, sl_n, sl_h;
  const float *q_pos, *k_pos;        // [B, N, pos]
  const int32_t *q_seg, *k_seg;      // [B, N] or null
  const int32_t* k_len;              // [B] or null
  int64_t nq, nk;
  int batch, heads, kv_heads, rep, dim;
  float scale, cap;
  // A CTA takes tile first_tile + blockIdx.x / splits and one of the parts of the other axis.
  int64_t first_tile;
  int splits;   // parts
  int cluster;  // CTAs that join their parts in shared memory: splits, or 1 (forward: joined by a second launch)
  int64_t tiles_per_split;
  // A launch over the first tiles, and one over the rest (from first_tile) beside the end of it.
  int ahead, behind;
  float* part_o;    // [splits, B, Nq, H, D]
  float* part_lse;  // [splits, B, H, Nq]
  // backward
  void *dq, *dk, *dv;
  float* records;  // [B, H, query tiles of 64][6][64]: what dK and dV need of each query (see below)
  float* dslopes;  // [B, Nq, H], by head [B, H, Nq], or null
  int dslopes_by_head;
  int32_t* error_flag;
  unsigned long long wait_limit_ns;
};

// Query values of one head, written by the dQ kernel and copied a tile at a time by the dK, dV kernel:
// -log2e lse (-inf: the query sees no key, or does not exist), -delta, x, y, -log2e slope, segment
// (-1: sees nothing).
constexpr int kRecordTile = 64, kRecordFields = 6;
constexpr int kRecordBytes = kRecordTile * kRecordFields * 4;

// ---- arithmetic ---------------------------------------------------------------------------------

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Two fp32 values in one 64-bit register: an instruction of the score loops does two scores, which
// leaves the issue slots to the special-function unit.  Each half is rounded as the scalar
// instruction would.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// The scores' constants: without a cap s2 = acc * k1; with one, cap tanh(y) = cap - 2 cap / (1 + e^2y)
// (an absolute error of a few 2^-23 cap, and the logits' absolute error is what counts), y = x / cap.
struct ScoreConst {
  float k1;   // scale log2e, or 2 scale / cap log2e
  float c;    // cap log2e
  __host__ __device__ ScoreConst(float scale, float cap)
      : k1(cap > 0.0f ? 2.0f * scale / cap * kLog2e : scale * kLog2e), c(cap * kLog2e) {}
  __device__ explicit ScoreConst(const AttnParams& p) : ScoreConst(p.scale, p.cap) {}
};

// 2 / (1 + e^2y): tanh(y) = 1 - that
__device__ __forceinline__ F2 tanh_rest(F2 acc, float k1) {
  float a, b;
  split(mul2(acc, f2(k1)), a, b);
  split(add2(f2(ex2(a), ex2(b)), f2(1.0f)), a, b);
  return mul2(f2(rcp(a), rcp(b)), f2(2.0f));
}

// Distances of one point, given by its negated coordinates (nx, ny), to two points.
template <int POS>
__device__ __forceinline__ F2 distance(F2 nx, F2 ny, F2 x, F2 y) {
  const F2 dx = add2(x, nx);
  float a, b;
  if constexpr (POS == 1) {
    split(dx, a, b);
    return f2(fabsf(a), fabsf(b));
  } else {
    const F2 dy = add2(y, ny);
    split(fma2(dx, dx, mul2(dy, dy)), a, b);
    return f2(sqrt_approx(a), sqrt_approx(b));
  }
}

// ---- tensor memory and tensor cores ----------------------------------------------------------------

__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld8_async(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// Waits for this thread's tensor-memory loads.  The registers pass through it, so that no use of them
// is scheduled ahead of the wait.
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// N consecutive columns of this thread's lane.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "one load");
  if constexpr (N == 8) tmem_ld8_async(taddr, r);
  if constexpr (N == 16) tmem_ld16_async(taddr, r);
  if constexpr (N == 32) tmem_ld32_async(taddr, r);
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "one store");
  if constexpr (N == 8) tmem_st8(taddr, r);
  if constexpr (N == 16) tmem_st16(taddr, r);
  if constexpr (N == 32) tmem_st32(taddr, r);
}

// Shared-memory descriptors of a tile of 128-byte rows (64 16-bit elements) stored with the 128-byte
// swizzle from a 1024-byte aligned base: start >> 4 in bits 0-13, descriptor version 1 in bits
// 46-47, swizzle mode 2 (128 B) in bits 61-63.
//  - K-major (the row is the K axis): 1024 B between 8-row groups (bits 32-45); the leading offset
//    is not used.  16 K elements further on: +2.
//  - MN-major (the row is the M/N axis, the tile's rows are K): 1024 B between groups of 8 K rows (bits
//    32-45), `block` bytes between blocks of 64 M/N elements (bits 16-29).  16 K rows further on: +128.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t block) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t((block >> 4) & 0x3FFFu) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// Instruction descriptor of kind::f16: D f32 (bits 4-5 = 1), A and B f16 (0) or bf16 (1) in bits 7-9
// and 10-12, B MN-major in bit 16, N >> 3 in bits 17-22, M = 128 >> 4 in bits 24-28.
template <typename T>
__device__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  const uint32_t t = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

// One lane of the (converged) warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from tensor memory: lane = row, two 16-bit K elements per column.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D[128, n] (+)= A B^T over DP columns: both tiles K-major, in blocks of 64 columns (a_block / b_block
// bytes apart).
template <typename T, int DP>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t a_block, uint32_t b, uint32_t b_block, int n) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    mma_ss(d, desc_sw128(a + (k / 4) * a_block, 1024) + 2 * (k % 4), desc_sw128(b + (k / 4) * b_block, 1024) + 2 * (k % 4),
           idesc_f16<T>(n, false), k != 0);
}

// D[128, DP] (+)= A B with A [128, ROWS] in tensor memory (16 values of a row every STEP columns) and B
// [ROWS, DP] in shared memory.
template <typename T, int DP, int ROWS, int STEP = 8>
__device__ __forceinline__ void mma_accumulate(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k)
    mma_ts(d, a + STEP * k, desc_sw128(b, DP > 64 ? ROWS * 128 : 1024) + 128 * k, idesc_f16<T>(DP, true), accumulate || k != 0);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int h, int n,
                                            int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(h), "r"(n), "r"(b)
      : "memory");
}

// One tile of ROWS rows and DP columns: blocks of 64 columns, ROWS * 128 bytes each.
template <int DP, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int h, int n, int b) {
  mbar_expect_tx(bar, DP / 64 * ROWS * 128);
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + c * ROWS * 128, map, bar, c * 64, h, n, b);
}

// Barriers of row threads (the other warps take no part).  Every row thread passes the same number of
// them whatever happens: one that gave up waiting goes on through its loop without work.
// barrier_sync / barrier_any: `threads` threads meet at barrier `id`; any: whether one brought true.
__device__ __forceinline__ void barrier_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool barrier_any(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(uint32_t(v))
      : "memory");
  return r != 0;
}

// mbar_wait (tc_ptx.cuh) with sleeping tests.
__device__ __forceinline__ bool sleep_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                           unsigned long long limit_ns) {
  constexpr uint32_t kNap = 20000;  // ns
  if (mbar_test_sleep(bar, parity, kNap)) return true;
  const unsigned long long t0 = now_ns();
  for (;;) {
    if (mbar_test_sleep(bar, parity, kNap)) return true;
    if (*abort_flag) return false;
    if (now_ns() - t0 > limit_ns) {
      *abort_flag = 1;
      return false;
    }
  }
}

// With a limit of 0 the warp that fetches the tiles stops half way, so that the other warps' waits do run out.
__device__ __forceinline__ bool withheld(const AttnParams& p, int t, int tiles) {
  return p.wait_limit_ns == 0 && 2 * (t + 1) > tiles;
}

// Warp-uniform bounded wait (the tensor-memory loads behind it are warp-collective).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned long long limit_ns) {
  const bool ok = __all_sync(0xffffffffu, sleep_wait(bar, parity, abort_flag, limit_ns));
  tc_fence_after();
  return ok;
}

// One arrival for a whole (converged) warp, after its tensor-memory stores: a barrier takes arrivals one
// at a time, and 128 of them are a visible part of a tile's turn-round.
constexpr uint32_t kRowWarps = kAttnRows / 32;  // arrivals of a stream's row threads
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// ---- asynchronous copies of a walked tile's small values ----------------------------------------------

// 4 bytes from global to shared memory without a register; copy_arrive arrives on `bar` once this
// thread's copies so far have landed (an arrival that the barrier's count includes).
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void store4(uint32_t dst, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(v) : "memory");
}
// `bytes` (a multiple of 16) between 16-byte aligned addresses, counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// The values of 64 keys of a tile, x[64], y[64] (POS) and segment[64] at shared-memory address dst, two
// keys a lane of one warp: asynchronous, so that a warp may be several tiles ahead.  Key j of the tile
// exists when j < left; what is past that is masked by segment -1 (rows have ids >= 0).  `bar`
// counts kKeyValueArrivals arrivals for them.
constexpr uint32_t kKeyValueArrivals = 33;
template <int POS>
__device__ __forceinline__ void load_key_values(uint32_t dst, uint32_t bar, const float* k_pos, const int32_t* k_seg,
                                                int64_t left) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = 2 * int(threadIdx.x & 31) + u;
    const bool in = j < left;
    if constexpr (POS > 0) {
      if (in) {
        copy4(dst + j * 4, k_pos + j * POS);
        if constexpr (POS > 1) copy4(dst + 256 + j * 4, k_pos + j * POS + 1);
      } else {
        store4(dst + j * 4, 0u);
        store4(dst + 256 + j * 4, 0u);
      }
    }
    if (in && k_seg != nullptr)
      copy4(dst + 512 + j * 4, k_seg + j);
    else
      store4(dst + 512 + j * 4, in ? 0u : 0xffffffffu);
  }
  copy_arrive(bar);
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);  // for the plain stores
}

// ---- values that are no numbers behind a mask --------------------------------------------------------

// Whether row `row` of a swizzled tile (DP columns, blocks `block` bytes apart) holds an infinity or a
// NaN.
template <typename T, int DP>
__device__ __forceinline__ bool row_not_finite(const unsigned char* tile, int block, int row) {
  constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int c = 0; c < DP / 8; ++c) {
    const int cc = c ^ (row & 7);  // lanes of a quarter warp on different banks
    const uint4 v = *reinterpret_cast<const uint4*>(tile + (c / 8) * block + row * 128 + ((cc & 7) << 4));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      bad |= (w[i] & kExp) == kExp || (w[i] & (kExp << 16)) == (kExp << 16);
  }
  return bad;
}

// acc[lane, :] (+)= sum over the rows j in [begin, end) (multiples of 16) of a tile of ROWS rows whose segment ids[j]
// is the lane's (`seg`, when it `sees` anything) of a[lane, j] tile[j, :]: what mma_accumulate computes, except
// that the other rows' infinities and NaNs take no part instead of being multiplied by 0.  A weight of a row that
// is seen which came out as 0 makes them NaN, as there.  For tiles that are masked in part and hold such values.
template <typename T, int DP, int ROWS, int STEP = 8>
__device__ __noinline__ void accumulate_seen(uint32_t acc, uint32_t a, const unsigned char* tile, bool init, const int* ids,
                                             int seg, bool sees, int begin = 0, int end = ROWS) {
  for (int c = 0; c < DP / 16; ++c) {
    float o[16];
    uint32_t r[16];
    tmem_ld16_async(acc + c * 16, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = init ? 0.0f : __uint_as_float(r[i]);
    const unsigned char* block = tile + (c / 4) * (ROWS * 128);
    for (int j0 = begin; j0 < end; j0 += 16) {
      uint32_t w[8];
      tmem_ld8_async(a + j0 / 16 * STEP, w);
      tmem_ld_wait(w);
#pragma unroll
      for (int jj = 0; jj < 16; ++jj) {
        const int j = j0 + jj;
        if (!sees || ids[j] != seg) continue;
        const float2 pr = unpack2<T>(w[jj / 2]);
        const float weight = jj & 1 ? pr.y : pr.x;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = *reinterpret_cast<const uint4*>(block + j * 128 + ((((c % 4) * 2 + h) ^ (j & 7)) << 4));
          const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(e[i]);
            o[h * 8 + 2 * i] = fmaf(weight, f.x, o[h * 8 + 2 * i]);
            o[h * 8 + 2 * i + 1] = fmaf(weight, f.y, o[h * 8 + 2 * i + 1]);
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(o[i]);
    tmem_st16(acc + c * 16, r);
  }
  tmem_st_wait();
}

// ---- which tiles a CTA walks -------------------------------------------------------------------------

enum : unsigned char { kTileSkip = 0, kTileFull = 1, kTileMasked = 2 };

// Smallest and largest id >= 0 among `n` consecutive ids (lo > hi when there is none), and whether all
// are one id >= 0.  Warp-collective.
struct SegRange {
  int lo, hi;
  bool one;
};
__device__ __forceinline__ SegRange seg_range(const int32_t* ids, int n) {
  int lo = INT_MAX, hi = -1;
  bool all = true;
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const int s = __ldg(ids + i);
    if (s >= 0) {
      lo = min(lo, s);
      hi = max(hi, s);
    } else {
      all = false;
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  all = __all_sync(0xffffffffu, all);
  return {lo, hi, all && lo == hi};
}

// Kind of every tile of `rows` ids in [first, first + tiles) of an axis with `valid` ids, for an own tile
// with range `own` (own_whole: none of its rows is past the end).  All warps of the CTA.
__device__ __forceinline__ void classify_tiles(unsigned char* kinds, int64_t first, int tiles, int rows, int64_t valid,
                                               const int32_t* ids, const SegRange& own, bool own_whole) {
  for (int t = threadIdx.x >> 5; t < tiles; t += blockDim.x / 32) {
    const int64_t r0 = (first + t) * rows;
    const int n = int(valid - r0 < rows ? (valid > r0 ? valid - r0 : 0) : rows);
    const SegRange r = seg_range(ids + r0, n);
    if ((threadIdx.x & 31) == 0) {
      const bool meet = n > 0 && r.lo <= own.hi && own.lo <= r.hi;
      kinds[t] = !meet ? kTileSkip : (own.one && r.one && own_whole && n == rows ? kTileFull : kTileMasked);
    }
  }
}

// Ring position of a tile: stage and parity, advanced without a division.
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) stage = 0, parity ^= 1;
  }
};

// The tiles a CTA walks: by the table of kinds, or without segments all of them, the first `whole` of
// them full and the others masked (the axis ends in the last one, or the own tile is not whole).
struct TileWalk {
  const unsigned char* kinds;
  int tiles, whole;
  __device__ __forceinline__ bool masked(int t) const { return kinds != nullptr ? kinds[t] == kTileMasked : t >= whole; }
  __device__ __forceinline__ int next(int t) const {
    ++t;
    if (kinds != nullptr)
      while (t < tiles && kinds[t] == kTileSkip) ++t;
    return t;
  }
  __device__ __forceinline__ int first() const { return next(-1); }
};

// ---- clusters -----------------------------------------------------------------------------------------

// All threads of all CTAs of the cluster, none of whose waits before it is without a limit.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Shared-memory address `addr` of this CTA in CTA `rank` of the cluster, and loads from there.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 peer_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 peer_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ int peer_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// Whether the flag at `addr` of any CTA of the cluster is set.
__device__ __forceinline__ bool cluster_any(uint32_t addr, int cluster) {
  int any = 0;
  for (int s = 0; s < cluster; ++s) any |= peer_int(peer_addr(addr, s));
  return any != 0;
}

// Four of the fp32 values at `addr` of every CTA of the cluster, added in the order of the ranks.
__device__ __forceinline__ float4 cluster_sum(uint32_t addr, int cluster) {
  float4 v[8], sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int s = 0; s < 8; ++s)
    if (s < cluster) v[s] = peer_f4(peer_addr(addr, s));
#pragma unroll
  for (int s = 0; s < 8; ++s)
    if (s < cluster) sum.x += v[s].x, sum.y += v[s].y, sum.z += v[s].z, sum.w += v[s].w;
  return sum;
}
__device__ __forceinline__ float cluster_sum1(uint32_t addr, int cluster) {
  float sum = 0.0f;
  for (int s = 0; s < cluster; ++s) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(addr, s)));
    sum += v;
  }
  return sum;
}

// NaNs over a row of `dim` 16-bit values, from a CTA that gave up waiting: what it computed is not to pass for
// a result.
__device__ __forceinline__ void store_nans(void* base, int64_t row, int dim) {
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + row * dim);
  for (int c = 0; c < dim / 8; ++c) dst[c] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
}

// ---- host ---------------------------------------------------------------------------------------------

struct AttnForwardMaps {
  CUtensorMap q, k, v;  // boxes of 128 rows of the heads of a shared head; of 64 keys
};
// One translation unit for each padded head dimension.
int launch_attention_forward_d64(int dtype, int pos, const AttnParams& p, const AttnForwardMaps& m, cudaStream_t st);
int launch_attention_forward_d128(int dtype, int pos, const AttnParams& p, const AttnForwardMaps& m, cudaStream_t st);

// Maps of the backward kernels: boxes of 128 own rows (of the heads that share keys), and of 64 rows of a
// walked tile.
struct AttnBackwardMaps {
  CUtensorMap q_rows, do_rows, k_rows, v_rows, q_tile, do_tile, k_tile, v_tile;
};
int launch_attention_backward_d64(int pos, const AttnParams& p, const AttnBackwardMaps& m, cudaStream_t st);
int launch_attention_backward_d128(int pos, const AttnParams& p, const AttnBackwardMaps& m, cudaStream_t st);

// The dynamic shared-memory limit of `kernel`, set once per device; `done` is the caller's record.
template <typename K>
int set_kernel_smem(K kernel, size_t bytes, const char* what, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  if (dev >= 0 && dev < 64 && done[dev]) return S4D_OK;
  const int st = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), what);
  if (st == S4D_OK && dev >= 0 && dev < 64) done[dev] = true;
  return st;
}

}  // namespace s4d
