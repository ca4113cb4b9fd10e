// Attention backward (formulas in decoder_attention.cuh), from the forward pass's log-sum-exp:
//
//   P = 2^(s - lse),  dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta),
//   dslope_i = -sum_j dS_ij dist_ij,  dX = dS (1 - tanh^2),
//   dQ = scale dX K,  dK = scale dX^T Q,  dV = P^T dO.
//
// Two kernels, so that nothing is added by atomics and equal calls give equal bits: one owns 128
// query rows and walks the keys (dQ, dslopes and delta, which the second needs), one owns 128 keys of
// a shared head and walks the query rows of every head that shares them (dK and dV).  That costs the
// two score products and the exponential a second time (7 products instead of 5), and saves a pass
// of fp32 additions over dQ in memory.  Both have the forward kernel's roles: one score row a thread, S and
// dP side by side in tensor memory (64 columns each), the 16-bit P and dS written back over them as
// the tensor-memory operand of the next products, the other operand read MN-major from the same
// shared-memory tile that served the scores.
//
// P and dS are rounded to bf16 because the tensor cores multiply them with bf16 operands; the bias's
// gradient is summed from the unrounded fp32 values.  fp16 is not offered: dS of a long row lies in
// fp16's subnormal range.
//
// What bounds it: as in the forward pass the work per score in registers (one exponential, one more
// special-function instruction with a 2-D distance, two with a cap, and about twenty others), which
// is why the tiles of the walked axis are 64 wide: two CTAs then share an SM at D <= 64.
#include "decoder_attention.cuh"

namespace s4d {
namespace {

using T = __nv_bfloat16;
constexpr int kCols = 64;  // rows of a walked tile
constexpr int kAttnThreads = 192;  // warps 0-3: one score row a thread; 4: TMA; 5: tensor cores

template <int DP>
struct Dq {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kCols * 128;
  static constexpr int kOwn = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStages = DP == 64 ? 2 : 1;
  static constexpr int kDo = kOwn, kK = kDo + kOwn, kV = kK + kStages * kTile, kAux = kV + kStages * kTile;
  static constexpr int kBars = kAux + 2 * 3 * kCols * 4;
  static constexpr int kNumBars = 4 * kStages + 3;
  static constexpr int kCtl = kBars + kNumBars * 8;
  static constexpr int kKinds = kCtl + 16;
  static constexpr uint32_t kTmem = 256;  // S / dS 64, dP 64, dQ DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

template <int DP>
struct Dkv {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kCols * 128;
  static constexpr int kOwn = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStages = 2;  // of a Q and a dO tile
  static constexpr int kV = kOwn, kQ = kV + kOwn, kAux = kQ + kStages * 2 * kTile;
  static constexpr int kBars = kAux + 2 * 6 * kCols * 4;
  static constexpr int kNumBars = 2 * kStages + 4;
  static constexpr int kCtl = kBars + kNumBars * 8;
  static constexpr int kKinds = kCtl + 16;
  static constexpr uint32_t kTmem = DP == 64 ? 256 : 512;  // S / P 64, dP / dS 64, dV DP, dK DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

// Two scores: their weights, gradients dS and (CAP) the cap's derivative 1 - tanh^2 = rest (2 - rest).
struct Terms {
  F2 p, ds, dx;
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
  r.dx = CAP ? mul2(r.ds, deriv) : r.ds;
  if constexpr (MASKED) {  // dP and the derivative of a masked pair may be no numbers
    split(r.ds, a, b);
    r.ds = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
    split(r.dx, a, b);
    r.dx = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
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

// One chunk of 32 keys of a query row.  aux arrays of a tile: -x, -y, segment.
template <int POS, bool CAP, bool MASKED>
__device__ __forceinline__ void dq_chunk(const uint32_t (&sr)[32], const uint32_t (&pr)[32], uint32_t (&w)[16],
                                         const ScoreConst& k, float slope2, float qx, float qy, int seg, float lse2,
                                         float delta, const float* aux, float (&sums)[3]) {
  F2 r0 = f2(0.0f), r1 = r0, e1 = r0;
  const F2 x2 = f2(qx), y2 = f2(qy), nslope = f2(-slope2), nlse2 = f2(-lse2), ndelta = f2(-delta);
#pragma unroll
  for (int j4 = 0; j4 < 32; j4 += 4) {
    float4 x4, y4;
    int4 s4;
    if constexpr (POS > 0) x4 = *reinterpret_cast<const float4*>(aux + j4);
    if constexpr (POS > 1) y4 = *reinterpret_cast<const float4*>(aux + kCols + j4);
    if constexpr (MASKED) s4 = *reinterpret_cast<const int4*>(aux + 2 * kCols + j4);
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      bool seen0 = true, seen1 = true;
      if constexpr (MASKED) seen0 = (u == 0 ? s4.x : s4.z) == seg, seen1 = (u == 0 ? s4.y : s4.w) == seg;
      F2 dist = f2(0.0f);
      if constexpr (POS > 0) dist = distance<POS>(x2, y2, half_of(x4, u), POS > 1 ? half_of(y4, u) : x2);
      const Terms t = score_terms<POS, CAP, MASKED>(pair_of(sr + j4 + u), k, nslope, dist, nlse2, pair_of(pr + j4 + u),
                                                    ndelta, seen0, seen1);
      if constexpr (POS > 0) {
        if constexpr (MASKED) {
          float a, b;
          split(dist, a, b);
          dist = f2(seen0 ? a : 0.0f, seen1 ? b : 0.0f);
        }
        r0 = add2(r0, t.ds);
        r1 = fma2(t.ds, dist, r1);
        e1 = fma2(t.p, dist, e1);
      }
      w[(j4 + u) / 2] = pack(t.dx);
    }
  }
  if constexpr (POS > 0) {
    float a, b;
    split(r0, a, b), sums[0] += a + b;
    split(r1, a, b), sums[1] += a + b;
    split(e1, a, b), sums[2] += a + b;
  }
}

template <int DP, int POS, bool CAP>
__global__ void __launch_bounds__(kAttnThreads, 2)
    attention_dq_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                        const AttnParams p) {
  using S = Dq<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t k_full = sbase + S::kBars, k_empty = k_full + 8 * S::kStages, v_full = k_empty + 8 * S::kStages,
                 v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages, ds_full = s_full + 8,
                 o_full = ds_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // blockIdx.x = (b G + g) row tiles + row tile; row r is query r / rep of head g rep + r % rep
  const uint32_t rep = uint32_t(p.rep);
  const int64_t rows = p.nq * p.rep, row_tiles = (rows + kAttnRows - 1) / kAttnRows;
  int64_t u = blockIdx.x;
  const int64_t row0 = u % row_tiles * kAttnRows;
  u /= row_tiles;
  const int g = int(u % p.kv_heads), b = int(u / p.kv_heads);
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  const int tiles = int((valid + kCols - 1) / kCols);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(k_full + 8 * s, 1);
      mbar_init(k_empty + 8 * s, 1);
      mbar_init(v_full + 8 * s, 1);
      mbar_init(v_empty + 8 * s, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(ds_full, kAttnRows);
    mbar_init(o_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), S::kTmem);
  TileWalk walk{nullptr, tiles, int(valid / kCols)};
  if (p.q_seg != nullptr) {
    const int64_t i0 = row0 / p.rep, i1 = (min(rows, row0 + kAttnRows) - 1) / p.rep;
    const SegRange own = seg_range(p.q_seg + b * p.nq + i0, int(i1 - i0 + 1));
    classify_tiles(kinds, 0, tiles, kCols, valid, p.k_seg + b * p.nk, own, true);
    walk.kinds = kinds;
  }
  for (int c = threadIdx.x; c < 2 * kAttnRows * (DP / 8); c += kAttnThreads) {
    const bool is_do = c >= kAttnRows * (DP / 8);
    const int e = is_do ? c - kAttnRows * (DP / 8) : c, r = e / (DP / 8), d = e % (DP / 8);
    const int64_t row = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows && d * 8 < p.dim) {
      const int64_t i = uint32_t(row) / rep, h = g * p.rep + uint32_t(row) % rep;
      v = is_do ? ldg_nc_v4(static_cast<const T*>(p.dout) + b * p.do_sb + i * p.do_sn + h * p.do_sh + d * 8)
                : ldg_nc_v4(static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_sn + h * p.q_sh + d * 8);
    }
    *reinterpret_cast<uint4*>(smem + (is_do ? S::kDo : 0) + (d / 8) * S::kOwnBlock + r * 128 +
                              (((d & 7) ^ (r & 7)) << 4)) = v;
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_dp = tmem + kCols, tmem_o = tmem + 2 * kCols;
  const int t0 = walk.first();

  if (warp == 4) {
    if (lane == 0) {
      int n = 0;
      for (int t = t0; t < tiles; t = walk.next(t), ++n) {
        const int s = n % S::kStages;
        const uint32_t parity = (n / S::kStages + 1) & 1;
        // V first: its stage is free once dP is there, K's only after dQ
        if (n >= S::kStages && !sleep_wait(v_empty + 8 * s, parity, abort_flag, p.wait_limit_ns)) break;
        load_tile<DP, kCols>(sbase + S::kV + s * S::kTile, &vm, v_full + 8 * s, g, t * kCols, b);
        if (n >= S::kStages && !sleep_wait(k_empty + 8 * s, parity, abort_flag, p.wait_limit_ns)) {
          mbar_wait(v_full + 8 * s, (n / S::kStages) & 1, nullptr);
          break;
        }
        load_tile<DP, kCols>(sbase + S::kK + s * S::kTile, &km, k_full + 8 * s, g, t * kCols, b);
      }
      for (int i = max(0, n - S::kStages); i < n; ++i) {
        mbar_wait(k_full + 8 * (i % S::kStages), (i / S::kStages) & 1, nullptr);
        mbar_wait(v_full + 8 * (i % S::kStages), (i / S::kStages) & 1, nullptr);
      }
    }
  } else if (warp == 5) {
    if (lane == 0) {
      int n = 0;
      for (int t = t0; t < tiles; t = walk.next(t), ++n) {
        const int s = n % S::kStages;
        const uint32_t parity = (n / S::kStages) & 1;
        const uint32_t kt = sbase + S::kK + s * S::kTile, vt = sbase + S::kV + s * S::kTile;
        if (!sleep_wait(v_full + 8 * s, parity, abort_flag, p.wait_limit_ns)) break;
        tc_fence_after();
        mma_scores<T, DP>(tmem_dp, sbase + S::kDo, S::kOwnBlock, vt, S::kBlock, kCols);
        mma_commit(v_empty + 8 * s);
        if (!sleep_wait(k_full + 8 * s, parity, abort_flag, p.wait_limit_ns)) break;
        tc_fence_after();
        mma_scores<T, DP>(tmem, sbase, S::kOwnBlock, kt, S::kBlock, kCols);
        mma_commit(s_full);
        if (!sleep_wait(ds_full, n & 1, abort_flag, p.wait_limit_ns)) break;
        tc_fence_after();
        if (!(walk.masked(t) && skip[n & 1])) mma_accumulate<T, DP, kCols>(tmem_o, tmem, kt, n > 0);
        mma_commit(k_empty + 8 * s);
      }
      mma_commit(o_full);
      mbar_wait(o_full, 0, nullptr);
    }
  } else {
    const int tid = threadIdx.x;
    const uint32_t lanes = uint32_t(warp * 32) << 16;
    const int64_t row = row0 + tid;
    const bool live = row < rows, warp_live = row0 + warp * 32 < rows;
    const int64_t i = live ? uint32_t(row) / rep : 0;
    const int h = g * p.rep + (live ? int(uint32_t(row) % rep) : 0);
    const int64_t out_row = (b * p.nq + i) * p.heads + h, lse_row = (int64_t(b) * p.heads + h) * p.nq + i;
    const ScoreConst k(p);
    float slope2 = 0.0f, qx = 0.0f, qy = 0.0f;
    if constexpr (POS > 0) {
      slope2 = __ldg(p.slopes + b * p.sl_b + i * p.sl_n + h * p.sl_h) * kLog2e;
      qx = __ldg(p.q_pos + (b * p.nq + i) * POS);
      if constexpr (POS > 1) qy = __ldg(p.q_pos + (b * p.nq + i) * POS + 1);
    }
    int seg = 0;
    if (p.q_seg != nullptr) {
      seg = __ldg(p.q_seg + b * p.nq + i);
      if (seg < 0) seg = -2;
    }
    // a row without a key (and a row past the last) gets weights of 2^-inf
    float lse2 = INFINITY, delta = 0.0f;
    if (live) {
      const float l = __ldg(p.lse + lse_row);
      if (l != -INFINITY) {
        lse2 = l * kLog2e;
        const uint4* o4 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.out) + out_row * p.dim);
        const uint4* d4 = reinterpret_cast<const uint4*>(static_cast<const T*>(p.dout) + b * p.do_sb + i * p.do_sn +
                                                         h * p.do_sh);
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
          if (c * 8 >= p.dim) break;
          float fo[8], fd[8];
          bf16x8_to_f32(ldg_nc_v4(o4 + c), fo);
          bf16x8_to_f32(ldg_nc_v4(d4 + c), fd);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf(fo[e], fd[e], delta);
        }
      }
      p.delta[lse_row] = delta;
    }
    float* aux = reinterpret_cast<float*>(smem + S::kAux);  // [2][3][64]: -x, -y, segment of the keys
    float nx = 0.0f, ny = 0.0f;
    int ns = -1;
    auto fetch = [&](int t) {
      if (t >= tiles || tid >= kCols) return;
      const int64_t j = int64_t(t) * kCols + tid;
      const bool in = j < valid;
      ns = in ? (p.k_seg != nullptr ? max(-1, __ldg(p.k_seg + b * p.nk + j)) : 0) : -1;
      if constexpr (POS > 0) {
        nx = in ? -__ldg(p.k_pos + (b * p.nk + j) * POS) : 0.0f;
        if constexpr (POS > 1) ny = in ? -__ldg(p.k_pos + (b * p.nk + j) * POS + 1) : 0.0f;
      }
    };
    fetch(t0);
    float sums[3] = {0.0f, 0.0f, 0.0f};  // sum dS, sum dS dist, sum P dist
    bool dead = false;
    int n = 0;
    for (int t = t0; t < tiles; ++n) {
      const int next = walk.next(t);
      const bool masked = walk.masked(t);
      float* bx = aux + (n & 1) * 3 * kCols;
      if (tid < kCols) {
        bx[tid] = nx;
        bx[kCols + tid] = ny;
        reinterpret_cast<int*>(bx)[2 * kCols + tid] = ns;
      }
      barrier_sync(1, kAttnRows);
      fetch(next);
      bool bad = false;
      const unsigned char* kt = smem + S::kK + n % S::kStages * S::kTile;
      if (masked) {
        if (!dead) dead = !warp_wait(k_full + 8 * (n % S::kStages), (n / S::kStages) & 1, abort_flag, p.wait_limit_ns);
        bad = barrier_any(2, kAttnRows, !dead && tid < kCols && row_not_finite<T, DP>(kt, S::kBlock, tid));
      }
      if (!dead) dead = !warp_wait(s_full, n & 1, abort_flag, p.wait_limit_ns);
      // only now: this tile's scores follow the products that read the flag's last value
      if (masked && tid == 0) skip[n & 1] = bad;
      if (!dead && warp_live) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sr[32], pr[32], w[16];
          tmem_ld32_async(tmem + lanes + c * 32, sr);
          tmem_ld32_async(tmem_dp + lanes + c * 32, pr);
          tmem_ld_wait(sr);
          tmem_ld_wait(pr);
          const float* cx = bx + c * 32;
          if (masked)
            dq_chunk<POS, CAP, true>(sr, pr, w, k, slope2, qx, qy, seg, lse2, delta, cx, sums);
          else
            dq_chunk<POS, CAP, false>(sr, pr, w, k, slope2, qx, qy, seg, lse2, delta, cx, sums);
          tmem_st16(tmem + lanes + c * 16, w);
        }
        tmem_st_wait();
        if (bad) accumulate_nonzero<T, DP, kCols>(tmem_o + lanes, tmem + lanes, kt, n == 0);
      }
      tc_fence_before();
      mbar_arrive(ds_full);
      t = next;
    }
    if (!dead && n > 0) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    if (!dead && warp_live) {
      if (POS > 0 && live && p.dslopes != nullptr) {
        // With an exact delta sum dS would be 0; the O that delta was made from is rounded to 16 bits, so
        // dS is off by P times that sum, and sum dS dist by that times sum P dist.
        p.dslopes[p.dslopes_by_head ? lse_row : out_row] = -fmaf(-sums[0], sums[2], sums[1]);
      }
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        if (c * 32 >= p.dim) break;
        uint32_t o[32];
        tmem_ld32_async(tmem_o + lanes + c * 32, o);
        tmem_ld_wait(o);
        if (!live) continue;
        T* dst = static_cast<T*>(p.dq) + out_row * p.dim + c * 32;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[x] = n > 0 ? pack2<T>(__uint_as_float(o[8 * e + 2 * x]) * p.scale, __uint_as_float(o[8 * e + 2 * x + 1]) * p.scale)
                         : 0u;
          if (c * 32 + e * 8 < p.dim) *reinterpret_cast<uint4*>(dst + e * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
  if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
}

// One chunk of 32 query columns of a key's row.  aux arrays of a tile: -lse2, -delta, -x, -y, -slope2, segment.
template <int POS, bool CAP, bool MASKED>
__device__ __forceinline__ void dkv_chunk(const uint32_t (&sr)[32], const uint32_t (&pr)[32], uint32_t (&wp)[16],
                                          uint32_t (&wd)[16], const ScoreConst& k, float kx, float ky, int seg,
                                          const float* aux) {
  const F2 x2 = f2(kx), y2 = f2(ky);
#pragma unroll
  for (int j4 = 0; j4 < 32; j4 += 4) {
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
      if constexpr (MASKED) seen0 = (u == 0 ? s4.x : s4.z) == seg, seen1 = (u == 0 ? s4.y : s4.w) == seg;
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

template <int DP, int POS, bool CAP>
__global__ void __launch_bounds__(kAttnThreads, DP == 64 ? 2 : 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                         const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap dom,
                         const AttnParams p) {
  using S = Dkv<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full = sbase + S::kBars, empty = full + 8 * S::kStages, own_full = empty + 8 * S::kStages,
                 s_full = own_full + 8, ds_full = s_full + 8, o_full = ds_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // blockIdx.x = (b G + g) key tiles + key tile
  const int64_t key_tiles = (p.nk + kAttnRows - 1) / kAttnRows;
  int64_t u = blockIdx.x;
  const int64_t key0 = u % key_tiles * kAttnRows;
  u /= key_tiles;
  const int g = int(u % p.kv_heads), b = int(u / p.kv_heads);
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  // query tiles, walked once for every head that shares the keys; none when no key here is valid
  const int tiles = key0 < valid ? int((p.nq + kCols - 1) / kCols) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(own_full, 1);
    mbar_init(s_full, 1);
    mbar_init(ds_full, kAttnRows);
    mbar_init(o_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), S::kTmem);
  const bool own_whole = key0 + kAttnRows <= valid;
  TileWalk walk{nullptr, tiles, own_whole ? int(p.nq / kCols) : 0};
  if (p.k_seg != nullptr) {
    const SegRange own = seg_range(p.k_seg + b * p.nk + key0, int(min(valid - key0, int64_t(kAttnRows))));
    classify_tiles(kinds, 0, tiles, kCols, p.nq, p.q_seg + b * p.nq, own, own_whole);
    walk.kinds = kinds;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_dp = tmem + kCols, tmem_dv = tmem + 2 * kCols, tmem_dk = tmem_dv + DP;
  const int t0 = walk.first();
  const bool work = t0 < tiles;

  if (warp == 4) {
    if (lane == 0 && work) {
      mbar_expect_tx(own_full, 2 * S::kOwn);
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_4d(sbase + c * S::kOwnBlock, &km, own_full, c * 64, g, int(key0), b);
        tma_load_4d(sbase + S::kV + c * S::kOwnBlock, &vm, own_full, c * 64, g, int(key0), b);
      }
      int n = 0;
      bool ok = true;
      for (int hh = 0; hh < p.rep && ok; ++hh)
        for (int t = t0; t < tiles; t = walk.next(t), ++n) {
          const int s = n % S::kStages;
          if (n >= S::kStages && !sleep_wait(empty + 8 * s, (n / S::kStages + 1) & 1, abort_flag, p.wait_limit_ns)) {
            ok = false;
            break;
          }
          const uint32_t st = sbase + S::kQ + s * 2 * S::kTile;
          mbar_expect_tx(full + 8 * s, 2 * S::kTile);
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_4d(st + c * S::kBlock, &qm, full + 8 * s, c * 64, g * p.rep + hh, t * kCols, b);
            tma_load_4d(st + S::kTile + c * S::kBlock, &dom, full + 8 * s, c * 64, g * p.rep + hh, t * kCols, b);
          }
        }
      mbar_wait(own_full, 0, nullptr);
      for (int i = max(0, n - S::kStages); i < n; ++i)
        mbar_wait(full + 8 * (i % S::kStages), (i / S::kStages) & 1, nullptr);
    }
  } else if (warp == 5) {
    if (lane == 0) {
      int n = 0;
      bool ok = !work || sleep_wait(own_full, 0, abort_flag, p.wait_limit_ns);
      for (int hh = 0; hh < p.rep && ok; ++hh)
        for (int t = t0; t < tiles; t = walk.next(t), ++n) {
          const int s = n % S::kStages;
          const uint32_t qt = sbase + S::kQ + s * 2 * S::kTile, dot = qt + S::kTile;
          if (!(ok = sleep_wait(full + 8 * s, (n / S::kStages) & 1, abort_flag, p.wait_limit_ns))) break;
          tc_fence_after();
          mma_scores<T, DP>(tmem, sbase, S::kOwnBlock, qt, S::kBlock, kCols);
          mma_scores<T, DP>(tmem_dp, sbase + S::kV, S::kOwnBlock, dot, S::kBlock, kCols);
          mma_commit(s_full);
          if (!(ok = sleep_wait(ds_full, n & 1, abort_flag, p.wait_limit_ns))) break;
          tc_fence_after();
          if (!(walk.masked(t) && skip[n & 1])) {
            mma_accumulate<T, DP, kCols>(tmem_dv, tmem, dot, n > 0);
            mma_accumulate<T, DP, kCols>(tmem_dk, tmem_dp, qt, n > 0);
          }
          mma_commit(empty + 8 * s);
        }
      mma_commit(o_full);
      mbar_wait(o_full, 0, nullptr);
    }
  } else {
    const int tid = threadIdx.x;
    const uint32_t lanes = uint32_t(warp * 32) << 16;
    const int64_t key = key0 + tid;
    const bool live = key < p.nk;
    const ScoreConst k(p);
    float kx = 0.0f, ky = 0.0f;
    // keys past the valid length match nothing (-2), nor do negative ids; without segments valid keys are 0
    int seg = key < valid ? (p.k_seg != nullptr ? __ldg(p.k_seg + b * p.nk + key) : 0) : -2;
    if (seg < 0) seg = -2;
    if constexpr (POS > 0) {
      if (live) {
        kx = __ldg(p.k_pos + (b * p.nk + key) * POS);
        if constexpr (POS > 1) ky = __ldg(p.k_pos + (b * p.nk + key) * POS + 1);
      }
    }
    // [2][6][64]: -lse2, -delta, -x, -y, -slope2, segment of the queries; threads 0-63 carry the first two
    // of their query one tile ahead, threads 64-127 the others
    float* aux = reinterpret_cast<float*>(smem + S::kAux);
    float c0 = 0.0f, c1 = 0.0f, c2 = 0.0f;
    int c3 = -1;
    const int e = tid & (kCols - 1);
    auto fetch = [&](int hh, int t) {
      if (hh >= p.rep) return;
      const int64_t i = int64_t(t) * kCols + e;
      const bool in = i < p.nq;
      const int h = g * p.rep + hh;
      if (tid < kCols) {
        const int64_t r = (int64_t(b) * p.heads + h) * p.nq + i;
        const float l = in ? __ldg(p.lse + r) : -INFINITY;
        c0 = l == -INFINITY ? -INFINITY : -l * kLog2e;  // no key seen: weights of 2^-inf
        c1 = in ? -p.delta[r] : 0.0f;
      } else {
        if constexpr (POS > 0) {
          c0 = in ? -__ldg(p.q_pos + (b * p.nq + i) * POS) : 0.0f;
          if constexpr (POS > 1) c1 = in ? -__ldg(p.q_pos + (b * p.nq + i) * POS + 1) : 0.0f;
          c2 = in ? -__ldg(p.slopes + b * p.sl_b + i * p.sl_n + h * p.sl_h) * kLog2e : 0.0f;
        }
        c3 = in ? (p.q_seg != nullptr ? max(-1, __ldg(p.q_seg + b * p.nq + i)) : 0) : -1;
      }
    };
    int hh = 0, t = t0, n = 0;
    bool dead = false;
    if (work) fetch(0, t0);
    while (work && hh < p.rep) {
      int next = walk.next(t), next_hh = hh;
      if (next >= tiles) next = t0, ++next_hh;
      const bool masked = walk.masked(t);
      float* bx = aux + (n & 1) * 6 * kCols;
      if (tid < kCols) {
        bx[e] = c0;
        bx[kCols + e] = c1;
      } else {
        bx[2 * kCols + e] = c0;
        bx[3 * kCols + e] = c1;
        bx[4 * kCols + e] = c2;
        reinterpret_cast<int*>(bx)[5 * kCols + e] = c3;
      }
      barrier_sync(1, kAttnRows);
      fetch(next_hh, next);
      bool bad = false;
      const int s = n % S::kStages;
      const unsigned char *qt = smem + S::kQ + s * 2 * S::kTile, *dot = qt + S::kTile;
      if (masked) {
        if (!dead) dead = !warp_wait(full + 8 * s, (n / S::kStages) & 1, abort_flag, p.wait_limit_ns);
        bad = barrier_any(2, kAttnRows, !dead && row_not_finite<T, DP>(tid < kCols ? qt : dot, S::kBlock, e));
      }
      if (!dead) dead = !warp_wait(s_full, n & 1, abort_flag, p.wait_limit_ns);
      // only now: this tile's scores follow the products that read the flag's last value
      if (masked && tid == 0) skip[n & 1] = bad;
      if (!dead) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t sr[32], pr[32], wp[16], wd[16];
          tmem_ld32_async(tmem + lanes + c * 32, sr);
          tmem_ld32_async(tmem_dp + lanes + c * 32, pr);
          tmem_ld_wait(sr);
          tmem_ld_wait(pr);
          if (masked)
            dkv_chunk<POS, CAP, true>(sr, pr, wp, wd, k, kx, ky, seg, bx + c * 32);
          else
            dkv_chunk<POS, CAP, false>(sr, pr, wp, wd, k, kx, ky, seg, bx + c * 32);
          tmem_st16(tmem + lanes + c * 16, wp);
          tmem_st16(tmem_dp + lanes + c * 16, wd);
        }
        tmem_st_wait();
        if (bad) {
          accumulate_nonzero<T, DP, kCols>(tmem_dv + lanes, tmem + lanes, dot, n == 0);
          accumulate_nonzero<T, DP, kCols>(tmem_dk + lanes, tmem_dp + lanes, qt, n == 0);
        }
      }
      tc_fence_before();
      mbar_arrive(ds_full);
      t = next;
      hh = next_hh;
      ++n;
    }
    if (!dead && n > 0) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    if (!dead) {
      const int64_t off = ((b * p.nk + (live ? key : 0)) * p.kv_heads + g) * p.dim;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float scale = which == 0 ? 1.0f : p.scale;
        T* base = static_cast<T*>(which == 0 ? p.dv : p.dk) + off;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          if (c * 32 >= p.dim) break;
          uint32_t o[32];
          tmem_ld32_async((which == 0 ? tmem_dv : tmem_dk) + lanes + c * 32, o);
          tmem_ld_wait(o);
          if (!live) continue;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = n > 0 ? pack2<T>(__uint_as_float(o[8 * x + 2 * y]) * scale, __uint_as_float(o[8 * x + 2 * y + 1]) * scale)
                           : 0u;
            if (c * 32 + x * 8 < p.dim)
              *reinterpret_cast<uint4*>(base + c * 32 + x * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
  if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
}

template <int DP, int POS, bool CAP>
int launch(const AttnParams& p, const AttnBackwardMaps& m, cudaStream_t st) {
  static bool dq_set[64] = {}, dkv_set[64] = {};
  int rc = set_kernel_smem(attention_dq_kernel<DP, POS, CAP>, Dq<DP>::smem(kAttnMaxTiles),
                           "cudaFuncSetAttribute(attention_dq_kernel)", dq_set);
  if (rc == S4D_OK)
    rc = set_kernel_smem(attention_dkv_kernel<DP, POS, CAP>, Dkv<DP>::smem(kAttnMaxTiles),
                         "cudaFuncSetAttribute(attention_dkv_kernel)", dkv_set);
  if (rc != S4D_OK) return rc;
  const int64_t groups = int64_t(p.kv_heads) * p.batch;
  if (p.nq > 0) {
    const int64_t row_tiles = (p.nq * p.rep + kAttnRows - 1) / kAttnRows;
    attention_dq_kernel<DP, POS, CAP><<<dim3(unsigned(row_tiles * groups)), kAttnThreads,
                                        Dq<DP>::smem(p.q_seg != nullptr ? (p.nk + kCols - 1) / kCols : 0), st>>>(m.k64, m.v64, p);
    rc = cuda_check(cudaGetLastError(), "attention_dq_kernel launch");
  }
  if (rc == S4D_OK && p.nk > 0 && p.dk != nullptr) {
    const int64_t key_tiles = (p.nk + kAttnRows - 1) / kAttnRows;
    attention_dkv_kernel<DP, POS, CAP><<<dim3(unsigned(key_tiles * groups)), kAttnThreads,
                                         Dkv<DP>::smem(p.q_seg != nullptr ? (p.nq + kCols - 1) / kCols : 0), st>>>(m.k128, m.v128, m.q64, m.do64, p);
    rc = cuda_check(cudaGetLastError(), "attention_dkv_kernel launch");
  }
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
