// Attention backward (formulas in decoder_attention.cuh), from the forward pass's log-sum-exp:
//
//   P = 2^(s - lse),  dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta),
//   dslope_i = -sum_j dS_ij dist_ij,  dX = dS (1 - tanh^2),
//   dQ = scale dX K,  dK = scale dX^T Q,  dV = P^T dO.
//
// Two kernels, so that nothing is added by atomics and equal calls give equal bits: one owns 128
// query rows and walks the keys (dQ, dslopes, and a record of each query for the second), one owns 128
// keys of a shared head and walks the query rows of every head that shares them (dK and dV).  That
// costs the two score products and the exponential a second time (8 products instead of 5, with the P K
// below), and saves a pass of fp32 additions over dQ in memory.  Both have the forward kernel's roles: one score
// row a thread, S and dP side by side in tensor memory (64 columns each), the 16-bit P and dS
// written back over them as the tensor-memory operand of the next products, the other operand read
// MN-major from the same shared-memory tile that served the scores.  The products of the scores and
// the ones that add to the sums are issued by two warps, so that neither waits for the other's turn.
//
// P and dS are rounded to bf16 because the tensor cores multiply them with bf16 operands (dQ and dK then
// are off by 0.0017 of their size from this, as much again from their own rounding); the bias's gradient
// is summed from the unrounded fp32 values.  fp16 is not offered: dS of a long row lies in fp16's
// subnormal range.  delta comes from an O that is rounded too, which would weigh as much as dP itself where
// a row's weight lies on few keys.  So the first kernel also adds R_i = sum_j dS_ij, which an exact delta
// makes 0, and the product P K: the second kernel gets delta + R, dQ loses R P K, dslope R sum P dist
// (8192 tokens: dq 735 us without the product, 740 with it).
//
// What bounds it: as in the forward pass the work per score in registers (one exponential, one more
// special-function instruction with a 2-D distance, two with a cap, and about twenty others), and the
// turn-round of a tile: its dS has to be multiplied before the next scores can go over it, about 1,800
// clocks.  So one CTA takes the SM's whole tensor memory: S and dP of three tiles of 64 (128 columns
// each), a stream of four row warps for each, so that two streams compute while the third waits (two
// tiles and streams at D = 128, whose two sums take the other half).  The sums dQ, dK and dV
// are linear in the tiles, so the streams share them; the tensor cores take the tiles in order.  Twelve
// row warps leave a thread 128 registers: it holds 16 scores and 16 dP at a time.
//
// Measured at 8192 tokens, 16 heads of 64 on 8, 1-D distance, calls in a CUDA graph: dq 740, dk and dv 711 us.  On the
// way there, before P K was added and tiles were cut (launch_tiles below): dq 756, dk and dv 862 us; with two
// streams and three tiles 807 and 908, those with 32 scores at a time 862 and 1000; with two CTAs an SM, two streams
// and tiles of 32 each 930 and 1180.  Then dk and dv took 574 us without the arithmetic of the scores and 337 without
// the products too.
#include "decoder_attention.cuh"

namespace s4d {
namespace {

using T = __nv_bfloat16;
constexpr int kCols = 64;   // rows of a walked tile
constexpr int kChunk = 16;  // of them a row thread holds in registers at a time (twice)

// Waits until the sums hold every tile before tile n, whose turn it is next: the last tile of each other
// score buffer (the own buffer's is done, it is in use again).  acc_done[s] counts the tiles of buffer
// s; none after n can be in, so a parity is enough.
template <int BUFFERS>
__device__ __forceinline__ bool earlier_done(uint32_t acc_done, int n, volatile int* abort_flag, unsigned long long limit_ns) {
  bool ok = true;
#pragma unroll
  for (int e = 1; e < BUFFERS; ++e)
    if (n >= e) ok = ok && warp_wait(acc_done + 8 * ((n - e) % BUFFERS), ((n - e) / BUFFERS) & 1, abort_flag, limit_ns);
  return ok;
}

template <int DP>
struct Dq {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kCols * 128;
  static constexpr int kOwn = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStreams = DP == 64 ? 3 : 2, kBuffers = kStreams, kWarps = 4 * kStreams;
  static constexpr int kThreads = (kWarps + 3) * 32;
  // a K tile is needed until its product with dS, a V tile only for dP
  static constexpr int kKStages = DP == 64 ? 6 : 5, kVStages = DP == 64 ? 4 : 3;
  static constexpr int kDo = kOwn, kK = kDo + kOwn, kV = kK + kKStages * kTile, kAux = kV + kVStages * kTile;
  // with each K tile: x, y and segment of its keys (at the end: each stream's sums and all's)
  static constexpr int kSums = (kStreams + 1) * 3 * kAttnRows * 4;
  static constexpr int kAuxBytes = kKStages * 3 * kCols * 4 > kSums ? kKStages * 3 * kCols * 4 : kSums;
  static constexpr int kBars = kAux + kAuxBytes;
  static constexpr int kNumBars = 2 * kKStages + 2 * kVStages + 3 * kBuffers + 3;
  static constexpr int kCtl = kBars + (kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kKinds = kCtl + 32;
  static constexpr uint32_t kTmem = 512;  // per buffer S / dS and P 64, dP 64; dQ DP, P K DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

template <int DP>
struct Dkv {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kCols * 128;
  static constexpr int kOwn = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStreams = DP == 64 ? 3 : 2, kBuffers = kStreams, kWarps = 4 * kStreams;
  static constexpr int kThreads = (kWarps + 3) * 32;
  static constexpr int kStages = DP == 64 ? 6 : 4;  // of a Q and a dO tile
  static constexpr int kV = kOwn, kQ = kV + kOwn, kAux = kQ + kStages * 2 * kTile;
  // with each stage: its queries' record
  static constexpr int kBars = kAux + kStages * 6 * kCols * 4;
  static constexpr int kNumBars = 2 * kStages + 3 * kBuffers + 3;
  static constexpr int kCtl = kBars + (kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kKinds = kCtl + 32;
  static constexpr uint32_t kTmem = 512;  // per buffer S / P 64, dP / dS 64; dV DP, dK DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

// Two scores: their weights P, gradients dS, and both times (CAP) the cap's derivative 1 - tanh^2 =
// rest (2 - rest).
struct Terms {
  F2 p, ds, px, dx;
};
template <int POS, bool CAP, bool MASKED>
__device__ __forceinline__ Terms score_terms(F2 acc, const ScoreConst& k, F2 nslope, F2 dist, F2 nlse2, F2 dp,
                                             F2 ndelta, bool seen0, bool seen1) {
  F2 s, deriv = f2(1.0f);
  if constexpr (CAP) {
    const F2 rest = tanh_rest(acc, k.k1);
    s = fma2(f2(-k.c), rest, f2(k.c));
    deriv = mul2(rest, fma2(f2(-1.0f), rest, f2(2.0f)));
  } else {
    s = mul2(acc, f2(k.k1));
  }
  if constexpr (POS > 0) s = fma2(nslope, dist, s);
  float a, b;
  split(add2(s, nlse2), a, b);
  a = ex2(a), b = ex2(b);
  if constexpr (MASKED) a = seen0 ? a : 0.0f, b = seen1 ? b : 0.0f;
  Terms r;
  r.p = f2(a, b);
  r.ds = mul2(r.p, add2(dp, ndelta));
  r.px = CAP ? mul2(r.p, deriv) : r.p;
  r.dx = CAP ? mul2(r.ds, deriv) : r.ds;
  if constexpr (MASKED) {  // dP and the derivative of a masked pair may be no numbers
    split(r.ds, a, b);
    r.ds = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
    split(r.dx, a, b);
    r.dx = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
    if constexpr (CAP) {
      split(r.px, a, b);
      r.px = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
    }
  }
  return r;
}

__device__ __forceinline__ F2 half_of(const float4& v, int u) { return u == 0 ? f2(v.x, v.y) : f2(v.z, v.w); }
__device__ __forceinline__ F2 pair_of(const uint32_t* r) { return f2(__uint_as_float(r[0]), __uint_as_float(r[1])); }
__device__ __forceinline__ uint32_t pack(F2 v) {
  float a, b;
  split(v, a, b);
  return pack2<T>(a, b);
}

// One chunk of CH keys of a query row (qx, qy negated).  aux arrays of a tile: x, y, segment.
template <int POS, bool CAP, bool MASKED, int CH>
__device__ __forceinline__ void dq_chunk(const uint32_t (&sr)[CH], const uint32_t (&pr)[CH], uint32_t (&w)[CH],
                                         const ScoreConst& k, float slope2, float qx, float qy, int seg, bool sees, float lse2,
                                         float delta, const float* aux, float (&sums)[3]) {
  F2 r0 = f2(0.0f), r1 = r0, e1 = r0;
  const F2 x2 = f2(qx), y2 = f2(qy), nslope = f2(-slope2), nlse2 = f2(-lse2), ndelta = f2(-delta);
#pragma unroll
  for (int j4 = 0; j4 < CH; j4 += 4) {
    float4 x4, y4;
    int4 s4;
    if constexpr (POS > 0) x4 = *reinterpret_cast<const float4*>(aux + j4);
    if constexpr (POS > 1) y4 = *reinterpret_cast<const float4*>(aux + kCols + j4);
    if constexpr (MASKED) s4 = *reinterpret_cast<const int4*>(aux + 2 * kCols + j4);
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      bool seen0 = true, seen1 = true;
      if constexpr (MASKED) seen0 = sees && (u == 0 ? s4.x : s4.z) == seg, seen1 = sees && (u == 0 ? s4.y : s4.w) == seg;
      F2 dist = f2(0.0f);
      if constexpr (POS > 0) dist = distance<POS>(x2, y2, half_of(x4, u), POS > 1 ? half_of(y4, u) : x2);
      const Terms t = score_terms<POS, CAP, MASKED>(pair_of(sr + j4 + u), k, nslope, dist, nlse2, pair_of(pr + j4 + u),
                                                    ndelta, seen0, seen1);
      r0 = add2(r0, t.ds);
      if constexpr (POS > 0) {
        if constexpr (MASKED) {
          float a, b;
          split(dist, a, b);
          dist = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
        }
        r1 = fma2(t.ds, dist, r1);
        e1 = fma2(t.p, dist, e1);
      }
      w[(j4 + u) / 2] = pack(t.dx);
      w[CH / 2 + (j4 + u) / 2] = pack(t.px);
    }
  }
  float a, b;
  split(r0, a, b), sums[0] += a + b;
  if constexpr (POS > 0) {
    split(r1, a, b), sums[1] += a + b;
    split(e1, a, b), sums[2] += a + b;
  }
}

// Columns [col, col + 32) of a row from fp32 accumulators (zeros when nothing was accumulated).
__device__ __forceinline__ void store_row32(T* row, int col, int dim, const uint32_t (&o)[32], bool any, float scale) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
      w[x] = any ? pack2<T>(__uint_as_float(o[8 * e + 2 * x]) * scale, __uint_as_float(o[8 * e + 2 * x + 1]) * scale) : 0u;
    if (col + e * 8 < dim) *reinterpret_cast<uint4*>(row + col + e * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A row's fp32 sums for the other CTAs of a cluster: N values in pieces of four, piece j of row r at
// j ^ (r & 7), from the start of the tiles in shared memory, which nothing reads any more.
template <int N>
__device__ __forceinline__ uint32_t shared_piece(uint32_t base, int r, int j) {
  return base + r * (N * 4) + ((j ^ (r & 7)) << 4);
}
// ... from the accumulators (zeros when nothing was accumulated).
template <int N, int STREAMS>
__device__ __forceinline__ void share_rows(unsigned char* smem, uint32_t acc, int row, int stream, bool any) {
  for (int c = stream; c < N / 32; c += STREAMS) {
    uint32_t o[32];
    tmem_ld32_async(acc + c * 32, o);
    tmem_ld_wait(o);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<uint4*>(smem + row * (N * 4) + (((c * 8 + e) ^ (row & 7)) << 4)) =
          any ? make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]) : make_uint4(0, 0, 0, 0);
  }
}

// The CTA's part of an own tile of 128 rows (dq) or keys (dkv) of a shared head: blockIdx.x, divided by the
// parts, counts (b G + g) tiles + tile from first_tile.
struct OwnTile {
  int part, g, b;
  uint32_t row0;
};
template <bool PARTS>
__device__ __forceinline__ OwnTile own_tile(const AttnParams& p, uint32_t rows) {
  uint32_t u = blockIdx.x;
  const uint32_t tiles = (rows + kAttnRows - 1) / kAttnRows;
  OwnTile o;
  o.part = 0;
  if constexpr (PARTS) {
    o.part = int(u % uint32_t(p.cluster));
    u = uint32_t(p.first_tile) + u / uint32_t(p.cluster);
  }
  o.row0 = u % tiles * kAttnRows;
  u /= tiles;
  o.g = int(u % uint32_t(p.kv_heads));
  o.b = int(u / uint32_t(p.kv_heads));
  return o;
}

template <int POS>
__device__ __forceinline__ void write_record(const AttnParams& p, int b, int h, int64_t i, float nlse2, float ndelta, float x,
                                             float y, float nslope2, int seg) {
  const int64_t tiles = (p.nq + kRecordTile - 1) / kRecordTile;
  float* r = p.records + ((int64_t(b) * p.heads + h) * tiles + i / kRecordTile) * (kRecordTile * kRecordFields) +
             i % kRecordTile;
  r[0] = nlse2;
  r[kRecordTile] = ndelta;
  if constexpr (POS > 0) {
    r[2 * kRecordTile] = x;
    r[3 * kRecordTile] = y;
    r[4 * kRecordTile] = nslope2;
  }
  reinterpret_cast<int*>(r)[5 * kRecordTile] = seg;
}

template <int DP, int POS, bool CAP, bool PARTS>
__global__ void __launch_bounds__(Dq<DP>::kThreads, 1)
    attention_dq_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap dom,
                        const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                        const AttnParams p) {
  using S = Dq<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t k_full = sbase + S::kBars, k_empty = k_full + 8 * S::kKStages, v_full = k_empty + 8 * S::kKStages,
                 v_empty = v_full + 8 * S::kVStages, s_full = v_empty + 8 * S::kVStages,
                 ds_full = s_full + 8 * S::kBuffers, acc_done = ds_full + 8 * S::kBuffers, o_full = acc_done + 8 * S::kBuffers,
                 own_full = o_full + 8, scores_out = own_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // row r is query r / rep of head g rep + r % rep
  const uint32_t rep = uint32_t(p.rep), rows = uint32_t(p.nq) * rep;
  const OwnTile own = own_tile<PARTS>(p, rows);
  const int64_t row0 = own.row0;
  const int g = own.g, b = own.b;
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  const int first = PARTS ? own.part * int(p.tiles_per_split) : 0;  // the part's first tile of keys
  const int tiles = max(0, min(int(p.tiles_per_split), int((valid + kCols - 1) / kCols) - first));
  // the tile is 128 / rep whole queries; nothing is fetched for a part without keys, whose row threads leave zeros
  // for the cluster over Q and dO without waiting for anything
  const bool gather = kAttnRows % p.rep != 0, own_by_tma = !gather && tiles > 0;

  if (warp == S::kWarps && lane == 0) {
    for (int s = 0; s < S::kKStages; ++s) {
      mbar_init(k_full + 8 * s, 1 + kKeyValueArrivals);  // the K tile, and the keys' values
      mbar_init(k_empty + 8 * s, 1);
    }
    for (int s = 0; s < S::kVStages; ++s) {
      mbar_init(v_full + 8 * s, 1);
      mbar_init(v_empty + 8 * s, 1);
    }
    for (int s = 0; s < S::kBuffers; ++s) {
      mbar_init(s_full + 8 * s, 2);  // the products, and the warp that saw the tile's values
      mbar_init(ds_full + 8 * s, kRowWarps);
      mbar_init(acc_done + 8 * s, 1);
    }
    mbar_init(o_full, 1);
    mbar_init(scores_out, 1);
    mbar_init(own_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (own_by_tma) {
      mbar_expect_tx(own_full, 2 * S::kOwn);
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_4d(sbase + c * S::kOwnBlock, &qm, own_full, c * 64, g * p.rep, int(uint32_t(row0) / rep), b);
        tma_load_4d(sbase + S::kDo + c * S::kOwnBlock, &dom, own_full, c * 64, g * p.rep, int(uint32_t(row0) / rep), b);
      }
    }
  }
  if (warp == S::kWarps + 1) tmem_alloc(smem_u32(tmem_slot), S::kTmem);
  TileWalk walk{nullptr, tiles, max(0, min(tiles, int(valid / kCols) - first))};
  if (!PARTS && p.q_seg != nullptr) {
    const int64_t i0 = row0 / rep, i1 = (min(int64_t(rows), row0 + kAttnRows) - 1) / rep;
    const SegRange ids = seg_range(p.q_seg + b * p.nq + i0, int(i1 - i0 + 1));
    classify_tiles(kinds, 0, tiles, kCols, valid, p.k_seg + b * p.nk, ids, true);
    walk.kinds = kinds;
  }

  // The row threads' own values
  const int stream = warp / 4, tid = threadIdx.x & 127;  // tid: the row, and the tensor-memory lane
  const int64_t row = row0 + tid;
  const bool live = row < rows;
  const uint32_t i = live ? (rep == 1 ? uint32_t(row) : uint32_t(row) / rep) : 0;
  const int h = int(g * rep + (live ? uint32_t(row) - i * rep : 0));
  const int64_t out_row = (b * p.nq + i) * p.heads + h, lse_row = (int64_t(b) * p.heads + h) * p.nq + i;
  float slope2 = 0.0f, qx = 0.0f, qy = 0.0f;
  float lse2 = INFINITY, delta = 0.0f;  // a row without a key (or past the last): weights of 2^-inf
  int seg = 0;       // without segments 0
  bool sees = true;  // false: a negative id, which sees nothing
  if (warp < S::kWarps) {
    if constexpr (POS > 0) {
      slope2 = __ldg(p.slopes + b * p.sl_b + i * p.sl_n + h * p.sl_h) * kLog2e;
      qx = -__ldg(p.q_pos + (b * p.nq + i) * POS);  // negated: differences are sums
      if constexpr (POS > 1) qy = -__ldg(p.q_pos + (b * p.nq + i) * POS + 1);
    }
    if (p.q_seg != nullptr) {
      seg = __ldg(p.q_seg + b * p.nq + i);
      sees = seg >= 0;
    }
    if (live) {
      const float l = __ldg(p.lse + lse_row);
      if (l != -INFINITY) {
        lse2 = l * kLog2e;
        const uint4* o4 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.out) + out_row * p.dim);
        const uint4* d4 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.dout) + b * p.do_sb + i * p.do_sn +
                                                         h * p.do_sh);
#pragma unroll 4
        for (int c = 0; c < p.dim / 8; ++c) {
          float fo[8], fd[8];
          bf16x8_to_f32(ldg_nc_v4(o4 + c), fo);
          bf16x8_to_f32(ldg_nc_v4(d4 + c), fd);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf(fo[e], fd[e], delta);
        }
      }
    }
    // queries that fill up the last tile of records
    if (row0 + kAttnRows >= rows) {
      const int64_t end = (p.nq + kRecordTile - 1) / kRecordTile * kRecordTile;
      for (int64_t e = p.nq * rep + threadIdx.x; e < end * rep; e += S::kWarps * 32)
        write_record<POS>(p, b, int(g * rep + e % rep), e / rep, -INFINITY, 0.0f, 0.0f, 0.0f, 0.0f, -1);
    }
  }
  if (gather && tiles > 0) {
    for (int c = threadIdx.x; c < 2 * kAttnRows * (DP / 8); c += S::kThreads) {
      const bool is_do = c >= kAttnRows * (DP / 8);
      const int e = is_do ? c - kAttnRows * (DP / 8) : c, r = e / (DP / 8), d = e % (DP / 8);
      const uint32_t at = uint32_t(row0) + r;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (at < rows && d * 8 < p.dim) {
        const int64_t qi = at / rep, hh = g * rep + at % rep;
        v = is_do ? ldg_nc_v4(static_cast<const T*>(p.dout) + b * p.do_sb + qi * p.do_sn + hh * p.do_sh + d * 8)
                  : ldg_nc_v4(static_cast<const T*>(p.q) + b * p.q_sb + qi * p.q_sn + hh * p.q_sh + d * 8);
      }
      *reinterpret_cast<uint4*>(smem + (is_do ? S::kDo : 0) + (d / 8) * S::kOwnBlock + r * 128 +
                                (((d & 7) ^ (r & 7)) << 4)) = v;
    }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!PARTS && p.ahead) griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + S::kBuffers * 2 * kCols;
  const int t0 = walk.first();

  if (warp == S::kWarps) {
    int nk = 0, nv = 0;  // loads under way or done
    Ring kr, vr;
    for (int t = t0; t < tiles && !withheld(p, t, tiles);) {
      // V first: its stage is free once dP is there, K's only after dQ
      if (nv >= S::kVStages && !warp_wait(v_empty + 8 * vr.stage, vr.parity ^ 1, abort_flag, p.wait_limit_ns)) break;
      if (lane == 0) load_tile<DP, kCols>(sbase + S::kV + vr.stage * S::kTile, &vm, v_full + 8 * vr.stage, g, (first + t) * kCols, b);
      ++nv;
      if (nk >= S::kKStages && !warp_wait(k_empty + 8 * kr.stage, kr.parity ^ 1, abort_flag, p.wait_limit_ns)) break;
      if (lane == 0) load_tile<DP, kCols>(sbase + S::kK + kr.stage * S::kTile, &km, k_full + 8 * kr.stage, g, (first + t) * kCols, b);
      const int64_t key = int64_t(first + t) * kCols, at = b * p.nk + key;
      load_key_values<POS>(sbase + S::kAux + kr.stage * 3 * kCols * 4, k_full + 8 * kr.stage, p.k_pos + at * POS,
                           p.k_seg != nullptr ? p.k_seg + at : nullptr, valid - key);
      ++nk;
      kr.next(S::kKStages);
      vr.next(S::kVStages);
      t = walk.next(t);
    }
    // no copy may land in the memory of a CTA that is gone: the last one of each stage
    if (own_by_tma) mbar_wait(own_full, 0, nullptr);
    for (int e = max(0, nk - S::kKStages); e < nk; ++e)
      mbar_wait(k_full + 8 * (e % S::kKStages), (e / S::kKStages) & 1, nullptr);
    for (int e = max(0, nv - S::kVStages); e < nv; ++e)
      mbar_wait(v_full + 8 * (e % S::kVStages), (e / S::kVStages) & 1, nullptr);
  } else if (warp == S::kWarps + 1) {
    const uint32_t leader = elect_one();
    Ring ks, vs, buf;
    bool ok = t0 >= tiles || !own_by_tma || warp_wait(own_full, 0, abort_flag, p.wait_limit_ns);
    int n = 0;
    for (int t = t0; ok && t < tiles; t = walk.next(t), ++n) {
      // the buffer's last dS is multiplied (its parity is the one before this tile's)
      ok = warp_wait(v_full + 8 * vs.stage, vs.parity, abort_flag, p.wait_limit_ns) &&
           warp_wait(k_full + 8 * ks.stage, ks.parity, abort_flag, p.wait_limit_ns) &&
           (n < S::kBuffers || warp_wait(acc_done + 8 * buf.stage, buf.parity ^ 1, abort_flag, p.wait_limit_ns));
      if (!ok) break;
      if (leader) {
        const uint32_t d = tmem + buf.stage * 2 * kCols;
        mma_scores<T, DP>(d + kCols, sbase + S::kDo, S::kOwnBlock, sbase + S::kV + vs.stage * S::kTile, S::kBlock, kCols);
        mma_commit(v_empty + 8 * vs.stage);
        mma_scores<T, DP>(d, sbase, S::kOwnBlock, sbase + S::kK + ks.stage * S::kTile, S::kBlock, kCols);
        mma_commit(s_full + 8 * buf.stage);
        mbar_arrive(s_full + 8 * buf.stage);
      }
      __syncwarp();
      ks.next(S::kKStages);
      vs.next(S::kVStages);
      buf.next(S::kBuffers);
    }
    if (leader) {
      mma_commit(scores_out);  // also on the abort path: nothing may run once tensor memory is freed
      mbar_wait(scores_out, 0, nullptr);
    }
    __syncwarp();
  } else if (warp == S::kWarps + 2) {
    const uint32_t leader = elect_one();
    Ring ka, buf;
    bool ok = true, any = false;
    for (int t = t0; ok && t < tiles; t = walk.next(t), any = true) {
      if (!(ok = warp_wait(ds_full + 8 * buf.stage, buf.parity, abort_flag, p.wait_limit_ns))) break;
      if (leader) {
        if (!(walk.masked(t) && skip[buf.stage])) {
          const uint32_t a = tmem + buf.stage * 2 * kCols, kt = sbase + S::kK + ka.stage * S::kTile;
          mma_accumulate<T, DP, kCols, 16>(tmem_o, a, kt, any);
          mma_accumulate<T, DP, kCols, 16>(tmem_o + DP, a + 8, kt, any);
        }
        mma_commit(acc_done + 8 * buf.stage);
        mma_commit(k_empty + 8 * ka.stage);
      }
      __syncwarp();
      ka.next(S::kKStages);
      buf.next(S::kBuffers);
    }
    if (leader) {
      mma_commit(o_full);
      mbar_wait(o_full, 0, nullptr);
    }
    __syncwarp();
  } else {
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const bool warp_live = row0 + warp % 4 * 32 < rows;
    const ScoreConst k(p);
    auto nth = [&](int t, int steps) {  // `steps` walked tiles on
      for (int e = 0; e < steps && t < tiles; ++e) t = walk.next(t);
      return t;
    };
    int t = nth(t0, stream), n = stream;
    float sums[3] = {0.0f, 0.0f, 0.0f};  // sum dS, sum dS dist, sum P dist
    bool dead = false;
    Ring r{stream, 0}, buf{stream, 0};  // K stages and score buffers of this stream's tiles
    for (; t < tiles; n += S::kStreams) {
      const uint32_t tmem_s = tmem + lanes + buf.stage * 2 * kCols;
      const int next = nth(t, S::kStreams);
      const bool masked = walk.masked(t);
      bool bad = false;  // a masked tile whose K holds values that are no numbers
      const unsigned char* kt = smem + S::kK + r.stage * S::kTile;
      const float* aux = reinterpret_cast<const float*>(smem + S::kAux) + r.stage * 3 * kCols;
      if (masked) {
        if (!dead) dead = !warp_wait(k_full + 8 * r.stage, r.parity, abort_flag, p.wait_limit_ns);
        bad = barrier_any(1 + stream, kAttnRows, !dead && tid < kCols && row_not_finite<T, DP>(kt, S::kBlock, tid));
      }
      if (!dead) dead = !warp_wait(s_full + 8 * buf.stage, buf.parity, abort_flag, p.wait_limit_ns);
      // only now: this tile's scores follow the product that read the flag's last value
      if (masked && tid == 0) skip[buf.stage] = bad;
      if (!dead && warp_live) {
        // the next chunk's loads are under way while one is computed
        uint32_t sr[2][kChunk], pr[2][kChunk];
        tmem_ld<kChunk>(tmem_s, sr[0]);
        tmem_ld<kChunk>(tmem_s + kCols, pr[0]);
#pragma unroll
        for (int c = 0; c < kCols / kChunk; ++c) {
          uint32_t w[kChunk];  // dS, then P
          tmem_ld_wait(sr[c & 1]);
          tmem_ld_wait(pr[c & 1]);
          if (c + 1 < kCols / kChunk) {
            tmem_ld<kChunk>(tmem_s + (c + 1) * kChunk, sr[(c + 1) & 1]);
            tmem_ld<kChunk>(tmem_s + kCols + (c + 1) * kChunk, pr[(c + 1) & 1]);
          }
          const float* cx = aux + c * kChunk;
          if (masked)
            dq_chunk<POS, CAP, true>(sr[c & 1], pr[c & 1], w, k, slope2, qx, qy, seg, sees, lse2, delta, cx, sums);
          else
            dq_chunk<POS, CAP, false>(sr[c & 1], pr[c & 1], w, k, slope2, qx, qy, seg, sees, lse2, delta, cx, sums);
          tmem_st<kChunk>(tmem_s + c * kChunk, w);
        }
        tmem_st_wait();
        if (bad) {
          // dQ is about to change outside the tensor cores
          dead = !earlier_done<S::kBuffers>(acc_done, n, abort_flag, p.wait_limit_ns);
          const int* ids = reinterpret_cast<const int*>(aux + 2 * kCols);
          if (!dead) accumulate_seen<T, DP, kCols, 16>(tmem_o + lanes, tmem_s, kt, n == 0, ids, seg, sees);
          if (!dead) accumulate_seen<T, DP, kCols, 16>(tmem_o + DP + lanes, tmem_s + 8, kt, n == 0, ids, seg, sees);
        }
      }
      warp_arrive(ds_full + 8 * buf.stage);
      t = next;
#pragma unroll
      for (int e = 0; e < S::kStreams; ++e) r.next(S::kKStages), buf.next(S::kBuffers);
    }
    if (!dead && t0 < tiles) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    // The streams' sums; o_full: no warp reads its keys' values any more.
    float* all = reinterpret_cast<float*>(smem + S::kAux);
#pragma unroll
    for (int e = 0; e < (POS > 0 ? 3 : 1); ++e) all[(stream * 3 + e) * kAttnRows + tid] = sums[e], sums[e] = 0.0f;
    barrier_sync(1 + S::kStreams, S::kWarps * 32);
#pragma unroll
    for (int s = 0; s < S::kStreams; ++s)
#pragma unroll
      for (int e = 0; e < (POS > 0 ? 3 : 1); ++e) sums[e] += all[(s * 3 + e) * kAttnRows + tid];
    // What a row's sums and products give.  With an exact delta sum dS would be 0; the O that delta was made
    // from is rounded to 16 bits (and made from 16-bit P), so delta is short of that sum, sum dS dist is off
    // by it times sum P dist, and dQ by it times P K.
    auto finish_row = [&](const float (&total)[3], float add) {  // add: 0, or the NaN of a CTA that gave up
      write_record<POS>(p, b, h, i, -lse2 + add, -(delta + total[0]), -qx, -qy, -slope2, sees ? seg : -1);
      if constexpr (POS > 0)
        if (p.dslopes != nullptr) p.dslopes[p.dslopes_by_head ? lse_row : out_row] = add - fmaf(-total[0], total[2], total[1]);
    };
    if constexpr (!PARTS) {
      if (live && stream == 0) finish_row(sums, 0.0f);
      if (!dead && warp_live) {
        // dQ's columns in 32s, shared out among the streams
        for (int c = stream; c * 32 < p.dim; c += S::kStreams) {
          uint32_t o[32], pk[32];
          tmem_ld32_async(tmem_o + lanes + c * 32, o);
          tmem_ld32_async(tmem_o + DP + lanes + c * 32, pk);
          tmem_ld_wait(o);
          tmem_ld_wait(pk);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(fmaf(-sums[0], __uint_as_float(pk[e]), __uint_as_float(o[e])));
          if (live) store_row32(static_cast<T*>(p.dq) + out_row * p.dim, c * 32, p.dim, o, t0 < tiles, p.scale);
        }
      }
    } else {
      // dQ, P K and the sums of this part of the keys, for the cluster
      float* total = all + S::kStreams * 3 * kAttnRows;
      if (stream == 0)
#pragma unroll
        for (int e = 0; e < (POS > 0 ? 3 : 1); ++e) total[e * kAttnRows + tid] = sums[e];
      share_rows<2 * DP, S::kStreams>(smem, tmem_o + lanes, tid, stream, t0 < tiles);
      cluster_sync();
      // a NaN when a CTA of the cluster gave up: all of their roles are done, and with them what sets the flag
      const float add = cluster_any(sbase + S::kCtl + 4, p.cluster) ? __int_as_float(0x7fc00000) : 0.0f;
      if (live && stream == 0 && tid % p.cluster == own.part) {
        float v[3] = {};
#pragma unroll
        for (int e = 0; e < (POS > 0 ? 3 : 1); ++e) v[e] = cluster_sum1(smem_u32(total + e * kAttnRows + tid), p.cluster);
        finish_row(v, add);
      }
      constexpr int kLanes = DP / 8, kRowsPerWarp = 32 / kLanes;
      const int col = lane % kLanes * 8;
      for (int r = own.part + p.cluster * (warp * kRowsPerWarp + lane / kLanes); r < kAttnRows && row0 + r < rows;
           r += p.cluster * kRowsPerWarp * S::kWarps) {
        const float short_of = cluster_sum1(smem_u32(total + r), p.cluster) + add;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 o = cluster_sum(shared_piece<2 * DP>(sbase, r, col / 4 + e), p.cluster);
          const float4 pk = cluster_sum(shared_piece<2 * DP>(sbase, r, (DP + col) / 4 + e), p.cluster);
          w[2 * e] = pack2<T>(fmaf(-short_of, pk.x, o.x) * p.scale, fmaf(-short_of, pk.y, o.y) * p.scale);
          w[2 * e + 1] = pack2<T>(fmaf(-short_of, pk.z, o.z) * p.scale, fmaf(-short_of, pk.w, o.w) * p.scale);
        }
        const uint32_t at = uint32_t(row0) + r, qi = at / rep, hh = g * rep + (at - qi * rep);
        if (col < p.dim)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.dq) + ((b * p.nq + qi) * p.heads + hh) * p.dim + col) =
              make_uint4(w[0], w[1], w[2], w[3]);
      }
      cluster_sync();  // the peers still read this CTA's shared memory
    }
  }
  if (PARTS && warp >= S::kWarps) {
    cluster_sync();
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == S::kWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
  const bool gave_up = *abort_flag;
  if (threadIdx.x == 0 && gave_up && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
  // every role is done: rows of a CTA that gave up become NaN, and through their records dK and dV
  if (!PARTS && gave_up && warp < 4 && live) {
    const float nan = __int_as_float(0x7fc00000);
    store_nans(p.dq, out_row, p.dim);
    write_record<POS>(p, b, h, i, nan, nan, -qx, -qy, -slope2, sees ? seg : -1);
    if (POS > 0 && p.dslopes != nullptr) p.dslopes[p.dslopes_by_head ? lse_row : out_row] = nan;
  }
  if (PARTS && p.behind) griddep_wait();  // what follows this launch follows the one ahead too
}

// One chunk of CH query columns of a key's row (kx, ky negated).  aux: the queries' record.
template <int POS, bool CAP, bool MASKED, int CH>
__device__ __forceinline__ void dkv_chunk(const uint32_t (&sr)[CH], const uint32_t (&pr)[CH], uint32_t (&wp)[CH / 2],
                                          uint32_t (&wd)[CH / 2], const ScoreConst& k, float kx, float ky, int seg, bool sees,
                                          const float* aux) {
  const F2 x2 = f2(kx), y2 = f2(ky);
#pragma unroll
  for (int j4 = 0; j4 < CH; j4 += 4) {
    const float4 l4 = *reinterpret_cast<const float4*>(aux + j4);
    const float4 d4 = *reinterpret_cast<const float4*>(aux + kCols + j4);
    float4 x4, y4, sl4;
    int4 s4;
    if constexpr (POS > 0) x4 = *reinterpret_cast<const float4*>(aux + 2 * kCols + j4);
    if constexpr (POS > 1) y4 = *reinterpret_cast<const float4*>(aux + 3 * kCols + j4);
    if constexpr (POS > 0) sl4 = *reinterpret_cast<const float4*>(aux + 4 * kCols + j4);
    if constexpr (MASKED) s4 = *reinterpret_cast<const int4*>(aux + 5 * kCols + j4);
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      bool seen0 = true, seen1 = true;
      if constexpr (MASKED) seen0 = sees && (u == 0 ? s4.x : s4.z) == seg, seen1 = sees && (u == 0 ? s4.y : s4.w) == seg;
      F2 dist = f2(0.0f), nslope = dist;
      if constexpr (POS > 0) {
        dist = distance<POS>(x2, y2, half_of(x4, u), POS > 1 ? half_of(y4, u) : x2);
        nslope = half_of(sl4, u);
      }
      const Terms t = score_terms<POS, CAP, MASKED>(pair_of(sr + j4 + u), k, nslope, dist, half_of(l4, u),
                                                    pair_of(pr + j4 + u), half_of(d4, u), seen0, seen1);
      wp[(j4 + u) / 2] = pack(t.p);
      wd[(j4 + u) / 2] = pack(t.dx);
    }
  }
}

template <int DP, int POS, bool CAP, bool PARTS>
__global__ void __launch_bounds__(Dkv<DP>::kThreads, 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                         const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap dom,
                         const AttnParams p) {
  using S = Dkv<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full = sbase + S::kBars, empty = full + 8 * S::kStages, s_full = empty + 8 * S::kStages,
                 ds_full = s_full + 8 * S::kBuffers, own_full = ds_full + 8 * S::kBuffers, acc_done = own_full + 8,
                 o_full = acc_done + 8 * S::kBuffers, scores_out = o_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const OwnTile own = own_tile<PARTS>(p, uint32_t(p.nk));
  const int64_t key0 = own.row0;
  const int g = own.g, b = own.b;
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  // the part's query tiles, walked once for every head that shares the keys; none when no key here is valid
  const int first = PARTS ? own.part * int(p.tiles_per_split) : 0, query_tiles = int((p.nq + kCols - 1) / kCols);
  const int tiles = key0 < valid ? max(0, min(int(p.tiles_per_split), query_tiles - first)) : 0;

  if (warp == S::kWarps && lane == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < S::kBuffers; ++s) {
      mbar_init(s_full + 8 * s, 2);  // the products, and the warp that saw the tile's values
      mbar_init(ds_full + 8 * s, kRowWarps);
      mbar_init(acc_done + 8 * s, 1);
    }
    mbar_init(own_full, 1);
    mbar_init(o_full, 1);
    mbar_init(scores_out, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (tiles > 0) {
      mbar_expect_tx(own_full, 2 * S::kOwn);
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_4d(sbase + c * S::kOwnBlock, &km, own_full, c * 64, g, int(key0), b);
        tma_load_4d(sbase + S::kV + c * S::kOwnBlock, &vm, own_full, c * 64, g, int(key0), b);
      }
    }
  }
  if (warp == S::kWarps + 1) tmem_alloc(smem_u32(tmem_slot), S::kTmem);
  const bool own_whole = key0 + kAttnRows <= valid;
  TileWalk walk{nullptr, tiles, own_whole ? max(0, min(tiles, int(p.nq / kCols) - first)) : 0};
  if (!PARTS && p.k_seg != nullptr) {
    const SegRange ids = seg_range(p.k_seg + b * p.nk + key0, int(min(valid - key0, int64_t(kAttnRows))));
    classify_tiles(kinds, 0, tiles, kCols, p.nq, p.q_seg + b * p.nq, ids, own_whole);
    walk.kinds = kinds;
  }

  // The row threads' own key
  const int stream = warp / 4, tid = threadIdx.x & 127;  // tid: the key, and the tensor-memory lane
  const int64_t key = key0 + tid;
  const bool live = key < p.nk;
  float kx = 0.0f, ky = 0.0f;
  int seg = 0;                // without segments 0
  bool sees = key < valid;  // false: past the valid length, or a negative id: seen by nothing
  if (warp < S::kWarps && live) {
    if (p.k_seg != nullptr) {
      seg = __ldg(p.k_seg + b * p.nk + key);
      sees = sees && seg >= 0;
    }
    if constexpr (POS > 0) {
      kx = -__ldg(p.k_pos + (b * p.nk + key) * POS);  // negated: differences are sums
      if constexpr (POS > 1) ky = -__ldg(p.k_pos + (b * p.nk + key) * POS + 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!PARTS && p.ahead) griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot, tmem_dv = tmem + S::kBuffers * 2 * kCols, tmem_dk = tmem_dv + DP;
  const int t0 = walk.first();
  const bool work = t0 < tiles;
  // the walk is repeated for every head: (head, tile) pairs in order
  auto advance = [&](int& hh, int& t) {
    t = walk.next(t);
    if (t >= tiles) t = t0, ++hh;
  };

  if (warp == S::kWarps) {
    if (lane == 0) {
      int n = 0, hh = work ? 0 : p.rep, t = t0;
      Ring r;
      for (; hh < p.rep && !withheld(p, t, tiles); advance(hh, t), ++n) {
        if (n >= S::kStages && !sleep_wait(empty + 8 * r.stage, r.parity ^ 1, abort_flag, p.wait_limit_ns)) break;
        const uint32_t st = sbase + S::kQ + r.stage * 2 * S::kTile, bar = full + 8 * r.stage;
        const int h = g * p.rep + hh;
        mbar_expect_tx(bar, 2 * S::kTile + kRecordBytes);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          tma_load_4d(st + c * S::kBlock, &qm, bar, c * 64, h, (first + t) * kCols, b);
          tma_load_4d(st + S::kTile + c * S::kBlock, &dom, bar, c * 64, h, (first + t) * kCols, b);
        }
        bulk_load(sbase + S::kAux + r.stage * kRecordBytes,
                  p.records + ((int64_t(b) * p.heads + h) * query_tiles + first + t) * (kRecordTile * kRecordFields), kRecordBytes,
                  bar);
        r.next(S::kStages);
      }
      if (tiles > 0) mbar_wait(own_full, 0, nullptr);
      for (int e = max(0, n - S::kStages); e < n; ++e)
        mbar_wait(full + 8 * (e % S::kStages), (e / S::kStages) & 1, nullptr);
    }
  } else if (warp == S::kWarps + 1) {
    const uint32_t leader = elect_one();
    Ring r, buf;
    bool ok = !work || warp_wait(own_full, 0, abort_flag, p.wait_limit_ns);
    int n = 0, hh = work ? 0 : p.rep, t = t0;
    for (; ok && hh < p.rep; advance(hh, t), ++n) {
      // the buffer's last P and dS are multiplied (its parity is the one before this tile's)
      ok = warp_wait(full + 8 * r.stage, r.parity, abort_flag, p.wait_limit_ns) &&
           (n < S::kBuffers || warp_wait(acc_done + 8 * buf.stage, buf.parity ^ 1, abort_flag, p.wait_limit_ns));
      if (!ok) break;
      if (leader) {
        const uint32_t d = tmem + buf.stage * 2 * kCols, qt = sbase + S::kQ + r.stage * 2 * S::kTile;
        mma_scores<T, DP>(d, sbase, S::kOwnBlock, qt, S::kBlock, kCols);
        mma_scores<T, DP>(d + kCols, sbase + S::kV, S::kOwnBlock, qt + S::kTile, S::kBlock, kCols);
        mma_commit(s_full + 8 * buf.stage);
        mbar_arrive(s_full + 8 * buf.stage);
      }
      __syncwarp();
      r.next(S::kStages);
      buf.next(S::kBuffers);
    }
    if (leader) {
      mma_commit(scores_out);  // also on the abort path: nothing may run once tensor memory is freed
      mbar_wait(scores_out, 0, nullptr);
    }
    __syncwarp();
  } else if (warp == S::kWarps + 2) {
    const uint32_t leader = elect_one();
    Ring r, buf;
    bool ok = true, any = false;
    int hh = work ? 0 : p.rep, t = t0;
    for (; ok && hh < p.rep; advance(hh, t), any = true) {
      if (!(ok = warp_wait(ds_full + 8 * buf.stage, buf.parity, abort_flag, p.wait_limit_ns))) break;
      if (leader) {
        if (!(walk.masked(t) && skip[buf.stage])) {
          const uint32_t d = tmem + buf.stage * 2 * kCols, qt = sbase + S::kQ + r.stage * 2 * S::kTile;
          mma_accumulate<T, DP, kCols>(tmem_dv, d, qt + S::kTile, any);
          mma_accumulate<T, DP, kCols>(tmem_dk, d + kCols, qt, any);
        }
        mma_commit(acc_done + 8 * buf.stage);
        mma_commit(empty + 8 * r.stage);
      }
      __syncwarp();
      r.next(S::kStages);
      buf.next(S::kBuffers);
    }
    if (leader) {
      mma_commit(o_full);
      mbar_wait(o_full, 0, nullptr);
    }
    __syncwarp();
  } else {
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const ScoreConst k(p);
    auto skip_tiles = [&](int& hh, int& t, int steps) {
      for (int e = 0; e < steps && hh < p.rep; ++e) advance(hh, t);
    };
    int hh = work ? 0 : p.rep, t = t0, n = stream;
    skip_tiles(hh, t, stream);
    bool dead = false;
    Ring r{stream, 0}, buf{stream, 0};  // stages and score buffers of this stream's tiles
    for (; hh < p.rep; n += S::kStreams) {
      const uint32_t tmem_s = tmem + lanes + buf.stage * 2 * kCols;
      const bool masked = walk.masked(t);
      bool bad = false;  // a masked tile whose Q or dO holds values that are no numbers
      const unsigned char *qt = smem + S::kQ + r.stage * 2 * S::kTile, *dot = qt + S::kTile;
      const float* aux = reinterpret_cast<const float*>(smem + S::kAux) + r.stage * 6 * kCols;
      if (masked) {
        if (!dead) dead = !warp_wait(full + 8 * r.stage, r.parity, abort_flag, p.wait_limit_ns);
        bad = barrier_any(1 + stream, kAttnRows,
                          !dead && tid < 2 * kCols && row_not_finite<T, DP>(tid < kCols ? qt : dot, S::kBlock, tid % kCols));
      }
      if (!dead) dead = !warp_wait(s_full + 8 * buf.stage, buf.parity, abort_flag, p.wait_limit_ns);
      // only now: this tile's scores follow the products that read the flag's last value
      if (masked && tid == 0) skip[buf.stage] = bad;
      if (!dead) {
        uint32_t sr[2][kChunk], pr[2][kChunk];
        tmem_ld<kChunk>(tmem_s, sr[0]);
        tmem_ld<kChunk>(tmem_s + kCols, pr[0]);
#pragma unroll
        for (int c = 0; c < kCols / kChunk; ++c) {
          uint32_t wp[kChunk / 2], wd[kChunk / 2];
          tmem_ld_wait(sr[c & 1]);
          tmem_ld_wait(pr[c & 1]);
          if (c + 1 < kCols / kChunk) {
            tmem_ld<kChunk>(tmem_s + (c + 1) * kChunk, sr[(c + 1) & 1]);
            tmem_ld<kChunk>(tmem_s + kCols + (c + 1) * kChunk, pr[(c + 1) & 1]);
          }
          if (masked)
            dkv_chunk<POS, CAP, true>(sr[c & 1], pr[c & 1], wp, wd, k, kx, ky, seg, sees, aux + c * kChunk);
          else
            dkv_chunk<POS, CAP, false>(sr[c & 1], pr[c & 1], wp, wd, k, kx, ky, seg, sees, aux + c * kChunk);
          tmem_st<kChunk / 2>(tmem_s + c * (kChunk / 2), wp);
          tmem_st<kChunk / 2>(tmem_s + kCols + c * (kChunk / 2), wd);
        }
        tmem_st_wait();
        if (bad) {
          // dV and dK are about to change outside the tensor cores
          dead = !earlier_done<S::kBuffers>(acc_done, n, abort_flag, p.wait_limit_ns);
          if (!dead) {
            const int* ids = reinterpret_cast<const int*>(aux + 5 * kCols);
            accumulate_seen<T, DP, kCols>(tmem_dv + lanes, tmem_s, dot, n == 0, ids, seg, sees);
            accumulate_seen<T, DP, kCols>(tmem_dk + lanes, tmem_s + kCols, qt, n == 0, ids, seg, sees);
          }
        }
      }
      warp_arrive(ds_full + 8 * buf.stage);
      skip_tiles(hh, t, S::kStreams);
#pragma unroll
      for (int e = 0; e < S::kStreams; ++e) r.next(S::kStages), buf.next(S::kBuffers);
    }
    if (!dead && work) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    if constexpr (PARTS) {
      // dV and dK of this part of the queries, for the cluster
      share_rows<2 * DP, S::kStreams>(smem, tmem_dv + lanes, tid, stream, work);
      cluster_sync();
      const bool gave_up = cluster_any(sbase + S::kCtl + 4, p.cluster);  // as in the dQ kernel
      constexpr int kLanes = 2 * DP / 8, kRowsPerWarp = 32 / kLanes;
      const int at = lane % kLanes * 8, col = at % DP;
      for (int r = own.part + p.cluster * (warp * kRowsPerWarp + lane / kLanes); r < kAttnRows && key0 + r < p.nk;
           r += p.cluster * kRowsPerWarp * S::kWarps) {
        const float4 x = cluster_sum(shared_piece<2 * DP>(sbase, r, at / 4), p.cluster);
        const float4 y = cluster_sum(shared_piece<2 * DP>(sbase, r, at / 4 + 1), p.cluster);
        const float f = gave_up ? __int_as_float(0x7fc00000) : at >= DP ? p.scale : 1.0f;
        if (col < p.dim)
          *reinterpret_cast<uint4*>(static_cast<T*>(at >= DP ? p.dk : p.dv) +
                                    ((b * p.nk + key0 + r) * p.kv_heads + g) * p.dim + col) =
              make_uint4(pack2<T>(x.x * f, x.y * f), pack2<T>(x.z * f, x.w * f), pack2<T>(y.x * f, y.y * f),
                         pack2<T>(y.z * f, y.w * f));
      }
      cluster_sync();  // the peers still read this CTA's shared memory
    } else if (!dead) {
      // dV's and dK's columns in 32s, shared out among the streams
      const int64_t off = ((b * p.nk + (live ? key : 0)) * p.kv_heads + g) * p.dim;
      for (int c = stream; c < 2 * DP / 32; c += S::kStreams) {
        const int col = c * 32 % DP;
        const bool is_k = c * 32 >= DP;
        if (col >= p.dim) continue;
        uint32_t o[32];
        tmem_ld32_async(tmem_dv + lanes + c * 32, o);
        tmem_ld_wait(o);
        if (live) store_row32(static_cast<T*>(is_k ? p.dk : p.dv) + off, col, p.dim, o, work, is_k ? p.scale : 1.0f);
      }
    }
  }
  if (PARTS && warp >= S::kWarps) {
    cluster_sync();
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == S::kWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
  const bool gave_up = *abort_flag;
  if (threadIdx.x == 0 && gave_up && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
  if (!PARTS && gave_up && warp < 4 && live) {  // as in the dQ kernel
    store_nans(p.dk, (b * p.nk + key) * p.kv_heads + g, p.dim);
    store_nans(p.dv, (b * p.nk + key) * p.kv_heads + g, p.dim);
  }
  if (PARTS && p.behind) griddep_wait();  // what follows this launch follows the one ahead too
}

// `tiles` own tiles (a CTA an SM) with `walked` tiles of the other axis each, `weight` times.  The tiles that
// fill the SMs are one launch of `whole_kernel`.  The rest, which would leave SMs idle for as long as a whole
// tile takes, are one of `kernel` beside the end of the first, cut into as many parts of the other axis as
// there is room for clusters of that many CTAs, up to eight: each keeps its sums in shared memory and
// joins a share of the rows.  A part keeps six tiles or more, since its start and the join take as long as
// two; the last ones get what is left, which may be none.  (Graph times of the backward pass without and with it:
// 4 x 1800 tokens, 8 heads, 480 own tiles 309 and 280 us; 8192 tokens, 512 tiles of keys 1544 and 1452 us; 900 tokens,
// 64 tiles, all cut 38.9 and 33.5 us.)  Tiles with segments differ in length and fill the SMs as they come, and are
// short: those are not cut (when that was tried, both passes over 8 x 1437 tokens in groups, 768 tiles, took 251 us,
// cut 256; 900 in three groups, 64 tiles, 55.0 and 55.2 us).
template <typename S, typename K, typename... Maps>
int launch_tiles(K whole_kernel, K kernel, const char* what, bool (&smem_set)[2][64], int (&fits)[64][9], AttnParams p,
                 int64_t tiles, int64_t walked, int64_t weight, cudaStream_t st, const Maps&... maps) {
  int rc = set_kernel_smem(whole_kernel, S::smem(kAttnMaxTiles), what, smem_set[0]);
  if (rc == S4D_OK) rc = set_kernel_smem(kernel, S::smem(kAttnMaxTiles), what, smem_set[1]);
  if (rc != S4D_OK) return rc;
  const int64_t sms = device_sms(), rest = tiles % sms;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.blockDim = dim3(S::kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {1, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  int dev = 0, parts = 1;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  for (int c = 8; c > 1 && rest > 0 && p.q_seg == nullptr && parts == 1; --c) {
    if (rest * c > sms || walked * weight < 6 * c || walked < c) continue;
    int fit = dev >= 0 && dev < 64 ? fits[dev][c] : 0;
    if (fit == 0) {
      attr[0].val.clusterDim.x = unsigned(c);
      cfg.gridDim = dim3(unsigned(c));
      cfg.dynamicSmemBytes = S::smem(0);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        fit = 0;
      }
      if (dev >= 0 && dev < 64) fits[dev][c] = fit > 0 ? fit : -1;
    }
    if (rest <= fit) parts = c;
  }
  const int64_t whole = parts > 1 ? tiles - rest : tiles;
  p.splits = p.cluster = 1;
  p.first_tile = 0;
  p.ahead = parts > 1;
  p.behind = 0;
  p.tiles_per_split = walked;
  if (whole > 0) {
    cfg.gridDim = dim3(unsigned(whole));
    cfg.dynamicSmemBytes = S::smem(p.q_seg != nullptr ? walked : 0);
    cfg.numAttrs = 0;
    rc = cuda_check(cudaLaunchKernelEx(&cfg, whole_kernel, maps..., p), what);
  }
  if (rc != S4D_OK || parts == 1) return rc;
  p.tiles_per_split = (walked + parts - 1) / parts;
  p.splits = p.cluster = parts;
  p.first_tile = whole;
  p.behind = whole > 0;
  attr[0].val.clusterDim.x = unsigned(parts);
  cfg.gridDim = dim3(unsigned(rest * parts));
  cfg.dynamicSmemBytes = S::smem(0);
  cfg.numAttrs = whole > 0 ? 2 : 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, maps..., p), what);
}

template <int DP, int POS, bool CAP>
int launch(const AttnParams& p, const AttnBackwardMaps& m, cudaStream_t st) {
  static bool dq_set[2][64] = {}, dkv_set[2][64] = {};
  static int dq_fits[64][9] = {}, dkv_fits[64][9] = {};
  const int64_t groups = int64_t(p.kv_heads) * p.batch;
  const int64_t query_tiles = (p.nq + kCols - 1) / kCols, key_tiles = (p.nk + kCols - 1) / kCols;
  int rc = S4D_OK;
  if (p.nq > 0)
    rc = launch_tiles<Dq<DP>>(attention_dq_kernel<DP, POS, CAP, false>, attention_dq_kernel<DP, POS, CAP, true>,
                              "attention_dq_kernel launch", dq_set, dq_fits, p,
                              (p.nq * p.rep + kAttnRows - 1) / kAttnRows * groups, key_tiles, 1, st, m.q_rows, m.do_rows,
                              m.k_tile, m.v_tile);
  if (rc == S4D_OK && p.nk > 0 && p.dk != nullptr)
    rc = launch_tiles<Dkv<DP>>(attention_dkv_kernel<DP, POS, CAP, false>, attention_dkv_kernel<DP, POS, CAP, true>,
                               "attention_dkv_kernel launch", dkv_set, dkv_fits, p,
                               (p.nk + kAttnRows - 1) / kAttnRows * groups, query_tiles, p.rep, st, m.k_rows, m.v_rows,
                               m.q_tile, m.do_tile);
  return rc;
}

}  // namespace

// This source is compiled once for each padded head dimension.
#define S4D_CAT2(a, b) a##b
#define S4D_CAT(a, b) S4D_CAT2(a, b)
int S4D_CAT(launch_attention_backward_d, S4D_HEAD_DIM)(int pos, const AttnParams& p, const AttnBackwardMaps& m,
                                                      cudaStream_t st) {
  constexpr int DP = S4D_HEAD_DIM;
  const bool cap = p.cap > 0.0f;
  switch (pos) {
    case 0: return cap ? launch<DP, 0, true>(p, m, st) : launch<DP, 0, false>(p, m, st);
    case 1: return cap ? launch<DP, 1, true>(p, m, st) : launch<DP, 1, false>(p, m, st);
    default: return cap ? launch<DP, 2, true>(p, m, st) : launch<DP, 2, false>(p, m, st);
  }
}

}  // namespace s4d
