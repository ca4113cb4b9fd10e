// Attention forward (formulas in decoder_attention.cuh):  o_i = sum_j p_ij v_j,  p = softmax over
// the allowed keys, in one pass over the keys with a running maximum m and sum l per row.
//
// One CTA owns 128 rows of one shared head: row r is query r / rep of head g rep + r % rep, so that
// the rep heads that share keys read them once.  It walks the keys in tiles of 64:
//   one warp    loads K and V tiles by TMA into rings of shared memory, and writes the keys' positions and
//               segments beside them;
//   one warp    issues S = Q K^T for the next tile into one of two score buffers in tensor memory (64
//               columns each), and once P of this tile is there O += P V, with P read from tensor
//               memory and V as an MN-major operand;
//   the others  one row a thread: scores from tensor memory, cap, bias and mask in registers (two
//               scores an instruction), the row maximum without a shuffle, P = 2^(s - m) back over S
//               as 16-bit pairs.
// O is only rescaled when a row's maximum grew by more than 2^8 since the last time (a published method): P then stays
// under 2^8, which costs no precision in a float.  P is rounded to the inputs' type because the
// tensor cores multiply it with V in that type; l adds the unrounded values in fp32.
//
// What bounds it: a score costs one exponential (16 a clock on an SM), a second special-function
// instruction with a 2-D distance and two more with a cap, against 4 D flops: for D = 64 the
// exponentials take four times as long as the products.  So there have to be row threads that are not
// waiting: two CTAs share an SM (256 tensor-memory columns and at most 113 KB of shared memory
// each), the next tile's scores are always under way, and at D <= 64 there are two streams of four
// warps, one for the even and one for the odd tiles, each with its own O, m and l, joined at the
// end (at D = 128 tensor memory holds one O).
//
// FEW: a row tile of a few rows only.  A thread that computes 64 scores is then what a tile waits for, while
// most lanes of the products hold nothing.  So the rows are there four times, once in each quarter of the
// lanes, and a quarter's warp weighs 16 keys of the tile (its other weights are 0); the copies have their
// own O, m and l and are joined like the parts of a cluster.  Those zeros stand for keys that the row sees:
// times an infinity they make a column of O a NaN, which is put right at the end (seen_not_finite), since to look
// through every tile's V first took one query over 4 x 65,536 keys from 208 to 237 us.
//
// Few rows and many keys: the keys are cut into parts, a CTA each.  Up to eight parts are one cluster:
// every CTA leaves its O, m and l in shared memory and each joins a share of the rows from its peers'.
// More parts write normalised O and log-sum-exp to memory and a second launch joins them.
//
// Measured (calls in a CUDA graph, bf16 unless said): 32 x 900 tokens, 8 heads of 64, 2-D distance 202 us (212 M
// exponentials and as many square roots: 119 us at 16 a clock); 8 x 1437, 8 heads of 64, segments 69 us;
// 2 x 4096, 16 heads of 128 on 4, capped, f16 392 us (270 us for its three special-function instructions
// a score); 8192 tokens, 16 heads of 64 on 8, 1-D distance 544 us.  What is left over is not one unit:
// when the first took 229, it took 167 with the square root taken out, 212 without exponentials, 197 without
// products, and 105 with an empty tile loop and all its hand-overs.  At D <= 64 a thread's 96 registers do not hold
// all it needs: the kernels but FEW spill 36 to 52 bytes.
#include "decoder_attention.cuh"

namespace s4d {
namespace {

constexpr int kKeys = 64;     // keys of a tile
constexpr int kFewRows = 32;  // FEW: the rows' four copies are this far apart

template <int DP>
struct Fwd {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kKeys * 128;  // 64 columns of Q, of K or V
  static constexpr int kQ = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStages = DP == 64 ? 4 : 2;     // of K and of V
  static constexpr int kStreams = DP == 64 ? 2 : 1;    // stream s walks every kStreams-th tile from s
  static constexpr int kWarps = 4 * kStreams;          // row threads; then the TMA and the tensor-core warp
  static constexpr int kThreads = (kWarps + 2) * 32;
  static constexpr int kK = kQ, kV = kK + kStages * kTile, kAux = kV + kStages * kTile;
  // x, y and segment of a tile's keys (after the last tile: m and l of the rows).  A slot is read
  // until the tile's P is there, so it is free for tile n once V of tile n - 1 has found a free stage: one
  // slot more than stages.  Then barriers; tensor-memory slot, abort, skip[2]
  static constexpr int kSlots = kStages + 1;
  static constexpr int kBars = kAux + kSlots * 3 * kKeys * 4;
  static constexpr int kNumBars = 4 * kStages + 8;
  static constexpr int kCtl = kBars + kNumBars * 8;
  static constexpr int kKinds = kCtl + 16;
  static constexpr uint32_t kCols = 256;  // S / P: 2 x 64, O: DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

// CH scores of a row, in base 2, and their maximum.
template <int POS, bool CAP, bool MASKED, int CH>
__device__ __forceinline__ void scores(uint32_t (&r)[CH], const ScoreConst& k, float slope2, float qx, float qy,
                                       int seg, bool sees, const float* aux, float& mx) {
  const F2 x2 = f2(qx), y2 = f2(qy), nslope = f2(-slope2), k1 = f2(k.k1), c = f2(k.c), nc = f2(-k.c);
#pragma unroll
  for (int j4 = 0; j4 < CH; j4 += 4) {
    float4 x4, y4;
    int4 s4;
    if constexpr (POS > 0) x4 = *reinterpret_cast<const float4*>(aux + j4);
    if constexpr (POS > 1) y4 = *reinterpret_cast<const float4*>(aux + kKeys + j4);
    if constexpr (MASKED) s4 = *reinterpret_cast<const int4*>(aux + 2 * kKeys + j4);
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      const F2 acc = f2(__uint_as_float(r[j4 + u]), __uint_as_float(r[j4 + u + 1]));
      F2 s = CAP ? fma2(nc, tanh_rest(acc, k.k1), c) : mul2(acc, k1);
      if constexpr (POS > 0) {
        const F2 kx = u == 0 ? f2(x4.x, x4.y) : f2(x4.z, x4.w);
        F2 ky = kx;
        if constexpr (POS > 1) ky = u == 0 ? f2(y4.x, y4.y) : f2(y4.z, y4.w);
        s = fma2(nslope, distance<POS>(x2, y2, kx, ky), s);
      }
      float a, b;
      split(s, a, b);
      if constexpr (MASKED) {
        a = sees && (u == 0 ? s4.x : s4.z) == seg ? a : -INFINITY;
        b = sees && (u == 0 ? s4.y : s4.w) == seg ? b : -INFINITY;
      }
      mx = max3(mx, a, b);
      r[j4 + u] = __float_as_uint(a);
      r[j4 + u + 1] = __float_as_uint(b);
    }
  }
}

// Their weights 2^(s - m) as 16-bit pairs, and the sum of the unrounded weights.
template <typename T, int CH>
__device__ __forceinline__ void weights(const uint32_t (&r)[CH], F2 nbase, F2 (&sum)[2], uint32_t* w) {
#pragma unroll
  for (int e = 0; e < CH / 2; ++e) {
    float a, d;
    split(add2(f2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), nbase), a, d);
    a = ex2(a), d = ex2(d);
    sum[e & 1] = add2(sum[e & 1], f2(a, d));
    w[e] = pack2<T>(a, d);
  }
}

// FEW: columns [col, col + 32) of a copy's O that came out as no numbers.  Such a column is the sum of the
// infinities and NaNs among the values of the keys that this copy weighs (16 of every 64 from key `begin`)
// and the row sees, or has none: then another copy has them, and here any number will do.
template <typename T>
__device__ __forceinline__ void seen_not_finite(float (&f)[32], const AttnParams& p, int b, int g, int64_t begin, int64_t end,
                                                int seg, bool sees, int col) {
#pragma unroll
  for (int e = 0; e < 32; ++e) f[e] = isfinite(f[e]) ? f[e] : 0.0f;
  if (!sees) return;
  const int32_t* k_seg = p.k_seg != nullptr ? p.k_seg + b * p.nk : nullptr;
  const T* v = static_cast<const T*>(p.v) + b * p.v_sb + g * p.v_sh + col;
#pragma unroll 1
  for (int64_t key = begin; key < end; key = (key + 1) % 16 == 0 ? key + 1 + kKeys - 16 : key + 1) {
    if (k_seg != nullptr && __ldg(k_seg + key) != seg) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (col + e * 8 >= p.dim) break;
      const uint4 x = ldg_nc_v4(v + key * p.v_sn + e * 8);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = unpack2<T>(w[i]);
        if (!isfinite(y.x)) f[8 * e + 2 * i] += y.x;
        if (!isfinite(y.y)) f[8 * e + 2 * i + 1] += y.y;
      }
    }
  }
}

template <typename T, int DP, int POS, bool CAP, bool FEW>
__global__ void __launch_bounds__(Fwd<DP>::kThreads, 2)
    attention_forward_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                             const __grid_constant__ CUtensorMap vm, const AttnParams p) {
  using S = Fwd<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t k_full = sbase + S::kBars, k_empty = k_full + 8 * S::kStages, v_full = k_empty + 8 * S::kStages,
                 v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages, p_full = s_full + 16,
                 pv_done = p_full + 16, o_full = pv_done + 16, q_full = o_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip_pv = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // blockIdx.x = ((b G + g) row tiles + row tile) splits + part; rank in the cluster: part % cluster
  const uint32_t rep = uint32_t(p.rep);  // rows of a shared head stay below 2^31
  const uint32_t rows = uint32_t(p.nq) * rep, row_tiles = (rows + kAttnRows - 1) / kAttnRows;
  uint32_t u = blockIdx.x;
  const int part = int(u % uint32_t(p.splits));
  u /= uint32_t(p.splits);
  const int64_t row0 = int64_t(u % row_tiles) * kAttnRows;
  u /= row_tiles;
  const int g = int(u % uint32_t(p.kv_heads)), b = int(u / uint32_t(p.kv_heads));
  const int64_t first = part * p.tiles_per_split;  // this part's first tile

  if (warp == S::kWarps && lane == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(k_full + 8 * s, 1 + kKeyValueArrivals);  // the K tile, and the keys' values
      mbar_init(k_empty + 8 * s, 1);
      mbar_init(v_full + 8 * s, 1);
      mbar_init(v_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + 8 * s, 2);  // the products, and the warp that saw the keys' values
      mbar_init(p_full + 8 * s, kRowWarps);
      mbar_init(pv_done + 8 * s, 1);
    }
    mbar_init(o_full, 2);  // the products, and the warp that issued them or gave up
    mbar_init(q_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == S::kWarps + 1) tmem_alloc(smem_u32(tmem_slot), S::kCols);
  griddep_wait();
  const bool q_by_tma = !FEW && kAttnRows % p.rep == 0;  // the tile is 128 / rep whole queries
  if (q_by_tma && warp == S::kWarps && lane == 0) {
    mbar_expect_tx(q_full, S::kQ);
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
      tma_load_4d(sbase + c * S::kOwnBlock, &qm, q_full, c * 64, g * p.rep, int(uint32_t(row0) / rep), b);
  }
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  const int tiles = int(max(int64_t(0), min(p.tiles_per_split, (valid + kKeys - 1) / kKeys - first)));
  TileWalk walk{nullptr, tiles, int(max(int64_t(0), min(int64_t(tiles), valid / kKeys - first)))};
  if (p.q_seg != nullptr) {
    const int64_t i0 = row0 / rep, i1 = (min(int64_t(rows), row0 + kAttnRows) - 1) / rep;
    const SegRange own = seg_range(p.q_seg + b * p.nq + i0, int(i1 - i0 + 1));
    classify_tiles(kinds, first, tiles, kKeys, valid, p.k_seg + b * p.nk, own, true);
    walk.kinds = kinds;
  }
  // Q where TMA cannot gather it: 16-byte pieces, zero past the last row and column, in the swizzled
  // layout TMA gives K and V
  if (!q_by_tma) {
    for (int c = threadIdx.x; c < kAttnRows * (DP / 8); c += S::kThreads) {
      const int r = c / (DP / 8), d = c % (DP / 8);
      const uint32_t at = uint32_t(row0) + (FEW ? r % kFewRows : r);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (at < rows && d * 8 < p.dim)
        v = ldg_nc_v4(static_cast<const T*>(p.q) + b * p.q_sb + int64_t(at / rep) * p.q_sn +
                      int64_t(g * rep + at % rep) * p.q_sh + d * 8);
      *reinterpret_cast<uint4*>(smem + (d / 8) * S::kOwnBlock + r * 128 + (((d & 7) ^ (r & 7)) << 4)) = v;
    }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();  // tensor memory is allocated: a kernel behind this one cannot take it away
  const int stream = warp / 4, tid = threadIdx.x & 127;  // tid: the row, and the tensor-memory lane
  const int64_t row = row0 + (FEW ? tid % kFewRows : tid);
  const bool live = row < rows;
  const uint32_t i = live ? (rep == 1 ? uint32_t(row) : uint32_t(row) / rep) : 0;
  const int h = int(g * rep + (live ? uint32_t(row) - i * rep : 0));
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 2 * kKeys;
  const int t0 = walk.first();

  if (warp == S::kWarps) {
    const int64_t left = valid - first * kKeys;  // keys of this part and after it
    auto load_k = [&](int s, int slot, int t) {
      if (lane == 0) load_tile<DP, kKeys>(sbase + S::kK + s * S::kTile, &km, k_full + 8 * s, g, int((first + t) * kKeys), b);
      const int64_t key = int64_t(t) * kKeys, at = b * p.nk + first * kKeys + key;
      load_key_values<POS>(sbase + S::kAux + slot * 3 * kKeys * 4, k_full + 8 * s, p.k_pos + at * POS,
                           p.k_seg != nullptr ? p.k_seg + at : nullptr, left - key);
    };
    auto load_v = [&](int s, int t) {
      if (lane == 0) load_tile<DP, kKeys>(sbase + S::kV + s * S::kTile, &vm, v_full + 8 * s, g, int((first + t) * kKeys), b);
    };
    int nk = 0, nv = 0, t = t0;  // loads under way or done
    Ring r, slot;
    while (t < tiles && !withheld(p, t, tiles)) {
      const bool again = nk >= S::kStages;
      if (again && !warp_wait(k_empty + 8 * r.stage, r.parity ^ 1, abort_flag, p.wait_limit_ns)) break;
      load_k(r.stage, slot.stage, t);
      ++nk;
      if (again && !warp_wait(v_empty + 8 * r.stage, r.parity ^ 1, abort_flag, p.wait_limit_ns)) break;
      load_v(r.stage, t);
      ++nv;
      r.next(S::kStages);
      slot.next(S::kSlots);
      t = walk.next(t);
    }
    // no copy may land in the memory of a CTA that is gone: the last one of each stage
    if (q_by_tma) mbar_wait(q_full, 0, nullptr);
    for (int e = max(0, nk - S::kStages); e < nk; ++e)
      mbar_wait(k_full + 8 * (e % S::kStages), (e / S::kStages) & 1, nullptr);
    for (int e = max(0, nv - S::kStages); e < nv; ++e)
      mbar_wait(v_full + 8 * (e % S::kStages), (e / S::kStages) & 1, nullptr);
  } else if (warp == S::kWarps + 1) {
    // The whole warp walks the tiles, so that addresses and descriptors stay in uniform registers; one
    // lane issues.
    const uint32_t leader = elect_one();
    // S of tile n, n counting the walked tiles
    Ring kr, vr;
    auto issue_scores = [&](int n) {
      if (!warp_wait(k_full + 8 * kr.stage, kr.parity, abort_flag, p.wait_limit_ns)) return false;
      if (leader) {
        mma_scores<T, DP>(tmem + (n & 1) * kKeys, sbase, S::kOwnBlock, sbase + S::kK + kr.stage * S::kTile, S::kBlock,
                          kKeys);
        mma_commit(k_empty + 8 * kr.stage);
        mma_commit(s_full + 8 * (n & 1));
        mbar_arrive(s_full + 8 * (n & 1));
      }
      __syncwarp();
      kr.next(S::kStages);
      return true;
    };
    // the scores of two tiles are out before the first P is waited for, and tile n + 2's follow the
    // product of P of tile n, whose buffer they go over: the tensor cores work in order
    const int t1 = walk.next(t0);
    bool ok = t0 >= tiles || ((!q_by_tma || warp_wait(q_full, 0, abort_flag, p.wait_limit_ns)) && issue_scores(0) &&
                              (t1 >= tiles || issue_scores(1)));
    int n = 0, ahead = t1 < tiles ? walk.next(t1) : tiles;
    for (int t = t0; ok && t < tiles; t = walk.next(t), ++n) {
      const int s = vr.stage;
      ok = warp_wait(v_full + 8 * s, vr.parity, abort_flag, p.wait_limit_ns) &&
           warp_wait(p_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
      if (!ok) break;
      if (leader) {
        if (!(walk.masked(t) && skip_pv[n & 1]))
          mma_accumulate<T, DP, kKeys>(tmem_o + n % S::kStreams * DP, tmem + (n & 1) * kKeys,
                                       sbase + S::kV + s * S::kTile, n >= S::kStreams);
        mma_commit(v_empty + 8 * s);
        mma_commit(pv_done + 8 * (n % S::kStreams));
      }
      __syncwarp();
      vr.next(S::kStages);
      if (ahead < tiles) {
        ok = issue_scores(n + 2);
        ahead = walk.next(ahead);
      }
    }
    if (leader) {
      mma_commit(o_full);  // also on the abort path: nothing may run once tensor memory is freed
      mbar_arrive(o_full);
      mbar_wait(o_full, 0, nullptr);
    }
    __syncwarp();
  } else {
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const bool warp_live = FEW || row0 + warp % 4 * 32 < rows;
    const ScoreConst k(p);
    float slope2 = 0.0f, qx = 0.0f, qy = 0.0f;
    int seg = 0;       // without segments 0
    bool sees = true;  // false: a negative id, which sees nothing
    if constexpr (POS > 0) {
      slope2 = __ldg(p.slopes + b * p.sl_b + i * p.sl_n + h * p.sl_h) * kLog2e;
      qx = -__ldg(p.q_pos + (b * p.nq + i) * POS);  // negated: differences are sums
      if constexpr (POS > 1) qy = -__ldg(p.q_pos + (b * p.nq + i) * POS + 1);
    }
    if (p.q_seg != nullptr) {
      seg = __ldg(p.q_seg + b * p.nq + i);
      sees = seg >= 0;
    }
    auto nth = [&](int t, int steps) {  // `steps` walked tiles on
      for (int e = 0; e < steps && t < tiles; ++e) t = walk.next(t);
      return t;
    };
    int t = nth(t0, stream);
    float m = -INFINITY, l = 0.0f;
    bool dead = false;
    int n = stream;
    Ring r{stream, 0}, slot{stream, 0};  // of this stream's tiles
    for (; t < tiles; n += S::kStreams) {
      const int next = nth(t, S::kStreams);
      const bool masked = walk.masked(t), first_tile = n == stream;
      bool bad = false;  // a masked tile whose V holds values that are no numbers
      const unsigned char* vt = smem + S::kV + r.stage * S::kTile;
      const float* aux = reinterpret_cast<const float*>(smem + S::kAux) + slot.stage * 3 * kKeys;
      const uint32_t tmem_s = tmem + lanes + (n & 1) * kKeys, tmem_acc = tmem_o + lanes + stream * DP;
      if (masked) {
        if (!dead) dead = !warp_wait(v_full + 8 * r.stage, r.parity, abort_flag, p.wait_limit_ns);
        bad = barrier_any(1 + stream, kAttnRows, !dead && tid < kKeys && row_not_finite<T, DP>(vt, S::kBlock, tid));
      }
      if (!dead) dead = !warp_wait(s_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
      // only now: this tile's scores follow the product that read the flag's last value
      if (masked && tid == 0) skip_pv[n & 1] = bad;
      if (!dead && warp_live) {
        // With two streams a thread has 96 registers: the first half of the scores waits in tensor memory.
        uint32_t r0[32], r1[32];
        float mx = -INFINITY;
        uint32_t rf[16];  // FEW: the warp's quarter of the keys
        const int quarter = warp % 4;
        if constexpr (FEW) {
          tmem_ld16_async(tmem_s + quarter * 16, rf);
          tmem_ld_wait(rf);
          if (masked)
            scores<POS, CAP, true>(rf, k, slope2, qx, qy, seg, sees, aux + quarter * 16, mx);
          else
            scores<POS, CAP, false>(rf, k, slope2, qx, qy, seg, sees, aux + quarter * 16, mx);
        } else if constexpr (S::kStreams == 2) {
          tmem_ld32_async(tmem_s, r0);
          tmem_ld_wait(r0);
          if (masked)
            scores<POS, CAP, true>(r0, k, slope2, qx, qy, seg, sees, aux, mx);
          else
            scores<POS, CAP, false>(r0, k, slope2, qx, qy, seg, sees, aux, mx);
          tmem_st32(tmem_s, r0);
          tmem_ld32_async(tmem_s + 32, r1);
          tmem_ld_wait(r1);
        } else {
          tmem_ld32_async(tmem_s, r0);
          tmem_ld32_async(tmem_s + 32, r1);
          tmem_ld_wait(r0);
          tmem_ld_wait(r1);
          if (masked)
            scores<POS, CAP, true>(r0, k, slope2, qx, qy, seg, sees, aux, mx);
          else
            scores<POS, CAP, false>(r0, k, slope2, qx, qy, seg, sees, aux, mx);
        }
        if constexpr (!FEW) {
          if (masked)
            scores<POS, CAP, true>(r1, k, slope2, qx, qy, seg, sees, aux + 32, mx);
          else
            scores<POS, CAP, false>(r1, k, slope2, qx, qy, seg, sees, aux + 32, mx);
        }
        const bool grow = mx > m + 8.0f || (m == -INFINITY && mx > m);
        const bool any_grow = __any_sync(0xffffffffu, grow);
        if (!first_tile && (any_grow || bad))  // O is about to change outside the tensor cores
          dead = !warp_wait(pv_done + 8 * stream, (n / S::kStreams - 1) & 1, abort_flag, p.wait_limit_ns);
        if (any_grow && !dead) {
          const float f = grow ? ex2(m - mx) : 1.0f;  // 0 for a row's first keys
          if (grow) m = mx;
          l *= f;
          if (!first_tile) {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
              uint32_t o[16];
              tmem_ld16_async(tmem_acc + c * 16, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(tmem_acc + c * 16, o);
            }
          }
        }
        const F2 nbase = f2(m == -INFINITY ? 0.0f : -m);  // no key yet: every score is -inf, every weight 0
        F2 sum[2] = {f2(0.0f), f2(0.0f)};
        if constexpr (FEW) {
          // the other quarters' weights of this copy of the row are 0
          uint32_t w[8], none[8] = {};
          weights<T>(rf, nbase, sum, w);
          tmem_st(tmem_s + quarter * 8, w);
#pragma unroll
          for (int e = 1; e < 4; ++e) tmem_st(tmem_s + (quarter + e) % 4 * 8, none);
        } else {
          uint32_t w[32];
          weights<T>(r1, nbase, sum, w + 16);
          if constexpr (S::kStreams == 2) {
            tmem_st_wait();
            tmem_ld32_async(tmem_s, r0);
            tmem_ld_wait(r0);
          }
          weights<T>(r0, nbase, sum, w);
          tmem_st32(tmem_s, w);
        }
        float a, d;
        split(add2(sum[0], sum[1]), a, d);
        l += a + d;
        tmem_st_wait();
        if (bad && !dead)  // FEW: this copy's quarter of the keys
          accumulate_seen<T, DP, kKeys>(tmem_acc, tmem_s, vt, first_tile, reinterpret_cast<const int*>(aux + 2 * kKeys), seg,
                                        sees, FEW ? quarter * 16 : 0, FEW ? quarter * 16 + 16 : kKeys);
      }
      warp_arrive(p_full + 8 * (n & 1));
      t = next;
#pragma unroll
      for (int e = 0; e < S::kStreams; ++e) r.next(S::kStages), slot.next(S::kSlots);
    }
    // With two streams each takes half of the columns and adds what both have there.
    if (!dead && t0 < tiles) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    float2* ml = reinterpret_cast<float2*>(smem + S::kAux);  // [128] m, l; the keys' values go with them
    float m1 = -INFINITY, l1 = 0.0f;                         // the other stream's
    if constexpr (S::kStreams == 2) {
      // o_full: every row thread has handed in its last P, so none reads its keys' values any more
      ml[stream * 128 + tid] = make_float2(m, l);
      barrier_sync(3, S::kWarps * 32);
      m1 = ml[(stream ^ 1) * 128 + tid].x, l1 = ml[(stream ^ 1) * 128 + tid].y;
    }
    const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
    float f0 = S::kStreams == 2 ? ex2(m - base) : 1.0f, f1 = S::kStreams == 2 ? ex2(m1 - base) : 0.0f;
    const float total = S::kStreams == 2 ? fmaf(l, f0, l1 * f1) : l;
    const bool any0 = l != 0.0f, any1 = l1 != 0.0f;  // else tensor memory holds nothing of this row
    const int64_t out_row = (b * p.nq + i) * p.heads + h;
    if (FEW || p.cluster > 1) {
      // O (not yet divided by l) and m, l stay in shared memory for the cluster: O over the K and V tiles,
      // which nothing reads any more, 16-byte piece j of row r at j ^ (r & 7)
      if constexpr (S::kStreams == 2) barrier_sync(3, S::kWarps * 32);
      // a CTA that gave up makes its rows NaN
      if (stream == 0) ml[tid] = make_float2(top, *abort_flag ? __int_as_float(0x7fc00000) : total);
    } else {
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // no key: zeros
      f0 *= inv, f1 *= inv;
      if (live && stream == 0) {
        const int64_t lse_row = (int64_t(b) * p.heads + h) * p.nq + i;
        const float lse = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
        if (p.splits > 1)
          p.part_lse[part * (int64_t(p.batch) * p.nq * p.heads) + lse_row] = lse;
        else if (p.lse != nullptr)
          p.lse[lse_row] = lse;
      }
    }
    if (!dead && warp_live) {
#pragma unroll
      for (int c0 = 0; c0 < DP / 32 / S::kStreams; ++c0) {
        const int c = c0 + stream * (DP / 32 / S::kStreams);
        if (c * 32 >= p.dim) break;
        uint32_t o[32];
        tmem_ld32_async(tmem_o + lanes + stream * DP + c * 32, o);
        tmem_ld_wait(o);
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = any0 ? __uint_as_float(o[e]) * f0 : 0.0f;
        if constexpr (S::kStreams == 2) {
          tmem_ld32_async(tmem_o + lanes + (stream ^ 1) * DP + c * 32, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = any1 ? fmaf(__uint_as_float(o[e]), f1, f[e]) : f[e];
        }
        if constexpr (FEW) {
          bool finite = true;
#pragma unroll
          for (int e = 0; e < 32; ++e) finite = finite && isfinite(f[e]);
          if (!finite && live)
            seen_not_finite<T>(f, p, b, g, first * kKeys + warp % 4 * 16, min(valid, (first + tiles) * kKeys), seg, sees, c * 32);
        }
        if (FEW || p.cluster > 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(smem + S::kK + tid * (DP * 4) + (((c * 8 + e) ^ (tid & 7)) << 4)) =
                make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
        } else if (live && p.splits > 1) {
          float* dst = p.part_o + (part * (int64_t(p.batch) * p.nq * p.heads) + out_row) * p.dim + c * 32;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c * 32 + e * 4 < p.dim)
              *reinterpret_cast<float4*>(dst + e * 4) = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
        } else if (live) {
          T* dst = static_cast<T*>(p.out) + out_row * p.dim + c * 32;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c * 32 + e * 8 < p.dim)
              *reinterpret_cast<uint4*>(dst + e * 8) =
                  make_uint4(pack2<T>(f[8 * e], f[8 * e + 1]), pack2<T>(f[8 * e + 2], f[8 * e + 3]),
                             pack2<T>(f[8 * e + 4], f[8 * e + 5]), pack2<T>(f[8 * e + 6], f[8 * e + 7]));
        }
      }
    }
  }
  tc_fence_before();
  if (p.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp == S::kWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kCols);
  }
  // Every role is done, and with it what sets the flag.  Rows that are stored already become NaN.
  const bool gave_up = *abort_flag;
  if (threadIdx.x == 0 && gave_up && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
  if (!FEW && p.cluster == 1) {
    if (gave_up && threadIdx.x < kAttnRows && row0 + threadIdx.x < rows) {
      const uint32_t at = uint32_t(row0) + threadIdx.x, qi = at / rep, hh = g * rep + at % rep;
      const int64_t lse_row = (int64_t(b) * p.heads + hh) * p.nq + qi;
      const float nan = __int_as_float(0x7fc00000);
      if (p.splits > 1) {
        p.part_lse[part * (int64_t(p.batch) * p.nq * p.heads) + lse_row] = nan;  // and so the joined row
      } else {
        store_nans(p.out, (b * p.nq + qi) * p.heads + hh, p.dim);
        if (p.lse != nullptr) p.lse[lse_row] = nan;
      }
    }
    return;
  }

  // The cluster's rows: DP / 8 lanes a row, 8 columns a lane; this CTA takes rows rank, rank + cluster, ...
  constexpr int kLanes = DP / 8, kRowsPerWarp = 32 / kLanes;
  const int col = lane % kLanes * 8;
  const int rank = p.cluster > 1 ? part : 0;
  for (int r = rank + p.cluster * (warp * kRowsPerWarp + lane / kLanes); r < (FEW ? kFewRows : kAttnRows) && row0 + r < rows;
       r += p.cluster * kRowsPerWarp * (S::kThreads / 32)) {
    const uint32_t at = uint32_t(row0) + r, qi = rep == 1 ? at : at / rep, hh = g * rep + (at - qi * rep);
    const int64_t out_row = (b * p.nq + qi) * p.heads + hh, lse_row = (int64_t(b) * p.heads + hh) * p.nq + qi;
    const uint32_t at_ml = sbase + S::kAux + r * 8, at_o = sbase + S::kK + r * (DP * 4);
    const uint32_t piece0 = at_o + (((col / 4) ^ (r & 7)) << 4), piece1 = at_o + (((col / 4 + 1) ^ (r & 7)) << 4);
    // four peers at a time (FEW: the four copies of one), all their loads before the first use
    float top = -INFINITY, total = 0.0f;
    float4 o0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o1 = o0;
    for (int s0 = 0; s0 < p.cluster; s0 += FEW ? 1 : 4) {
      float2 v[4];
      float4 x[4], y[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t peer = FEW ? s0 : min(s0 + s, p.cluster - 1), copy = FEW ? s * kFewRows : 0;
        v[s] = peer_f2(peer_addr(at_ml + copy * 8, peer));
        x[s] = peer_f4(peer_addr(piece0 + copy * (DP * 4), peer));
        y[s] = peer_f4(peer_addr(piece1 + copy * (DP * 4), peer));
      }
      float high = top;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (FEW || s0 + s < p.cluster) high = fmaxf(high, v[s].x);
      const float base = high == -INFINITY ? 0.0f : high, old = ex2(top - base);
      top = high;
      total *= old;
      o0.x *= old, o0.y *= old, o0.z *= old, o0.w *= old, o1.x *= old, o1.y *= old, o1.z *= old, o1.w *= old;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (!FEW && s0 + s >= p.cluster) continue;
        const float w = ex2(v[s].x - base);  // 0 for a part without keys
        total = fmaf(v[s].y, w, total);
        o0.x = fmaf(w, x[s].x, o0.x), o0.y = fmaf(w, x[s].y, o0.y), o0.z = fmaf(w, x[s].z, o0.z),
        o0.w = fmaf(w, x[s].w, o0.w);
        o1.x = fmaf(w, y[s].x, o1.x), o1.y = fmaf(w, y[s].y, o1.y), o1.z = fmaf(w, y[s].z, o1.z),
        o1.w = fmaf(w, y[s].w, o1.w);
      }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // no key: zeros
    const float lse = total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
    if (FEW && p.splits != p.cluster) {  // one of many parts
      const int64_t all = int64_t(p.batch) * p.nq * p.heads;
      if (col == 0) p.part_lse[part * all + lse_row] = lse;
      if (col < p.dim) {
        float4* dst = reinterpret_cast<float4*>(p.part_o + (part * all + out_row) * p.dim + col);
        dst[0] = make_float4(o0.x * inv, o0.y * inv, o0.z * inv, o0.w * inv);
        dst[1] = make_float4(o1.x * inv, o1.y * inv, o1.z * inv, o1.w * inv);
      }
      continue;
    }
    if (col == 0 && p.lse != nullptr) p.lse[lse_row] = lse;
    if (col < p.dim)
      *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row * p.dim + col) =
          make_uint4(pack2<T>(o0.x * inv, o0.y * inv), pack2<T>(o0.z * inv, o0.w * inv),
                     pack2<T>(o1.x * inv, o1.y * inv), pack2<T>(o1.z * inv, o1.w * inv));
  }
  if (p.cluster > 1) cluster_sync();  // the peers still read this CTA's shared memory
}

// Joins the parts of one row: o = sum_s 2^(lse_s - lse) o_s.  One warp a row, lanes along D.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = int64_t(p.batch) * p.nq * p.heads;
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (b, i, h)
  griddep_wait();
  if (row >= rows) return;
  const int h = int(row % p.heads);
  const int64_t bi = row / p.heads, lse_row = (bi / p.nq * p.heads + h) * p.nq + bi % p.nq;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_lse[s * rows + lse_row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f;
  const bool mine = lane * 4 < p.dim;
  const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float lse = p.part_lse[s * rows + lse_row], w = ex2((lse - base) * kLog2e);
    total += w;
    if (mine && lse != -INFINITY) {  // a part without keys has weight 0
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.dim + lane * 4);
      o[0] = fmaf(w, v.x, o[0]), o[1] = fmaf(w, v.y, o[1]), o[2] = fmaf(w, v.z, o[2]), o[3] = fmaf(w, v.w, o[3]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (mine) {
    const uint2 v = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + row * p.dim + lane * 4) = v;
  }
  if (lane == 0 && p.lse != nullptr) p.lse[lse_row] = total == 0.0f ? -INFINITY : base + log2f(total) * kLn2;
}

template <typename T, int DP, int POS, bool CAP, bool FEW>
int launch_kernel(const AttnParams& p, const AttnForwardMaps& m, cudaStream_t st) {
  static bool smem_set[64] = {};
  const int rc = set_kernel_smem(attention_forward_kernel<T, DP, POS, CAP, FEW>, Fwd<DP>::smem(kAttnMaxTiles),
                                 "cudaFuncSetAttribute(attention_forward_kernel)", smem_set);
  if (rc != S4D_OK) return rc;
  const int64_t row_tiles = (p.nq * p.rep + kAttnRows - 1) / kAttnRows;
  const int64_t ctas = row_tiles * p.kv_heads * p.batch * p.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(Fwd<DP>::kThreads);
  cfg.dynamicSmemBytes = Fwd<DP>::smem(p.q_seg != nullptr ? p.tiles_per_split : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  // one wave of CTAs: their start overlaps the end of the kernel ahead
  if (ctas <= 2 * device_sms()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = unsigned(p.cluster);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  return cuda_check(cudaLaunchKernelEx(&cfg, attention_forward_kernel<T, DP, POS, CAP, FEW>, m.q, m.k, m.v, p),
                    "attention_forward_kernel launch");
}

// A row tile of eight rows or fewer is held four times where a score has a bias or a cap.  Graph times of 4 x 1 query
// over 65,536 keys, 32 heads on 8 shared ones, without and with it: of 128, 2-D distance 195 and 176 us, capped
// 193 and 171, both 261 and 175; of 64, 1-D distance 124 and 110, 2-D 145 and 104, capped 154 and 102 (heads of
// 128 with 1-D distance 177 either way).  Plain scores lose: 164 and 168 us for heads of 128, 100 and 103 of 64.
// So do more rows, which are fetched one by one (6 x 30 over 900: 10.6 and 12.8 us).
template <typename T, int DP, int POS, bool CAP>
int launch(const AttnParams& p, const AttnForwardMaps& m, cudaStream_t st) {
  if constexpr (POS > 0 || CAP)
    if (p.nq * p.rep <= 8) return launch_kernel<T, DP, POS, CAP, true>(p, m, st);
  return launch_kernel<T, DP, POS, CAP, false>(p, m, st);
}

template <typename T, int DP>
int by_scores(const AttnParams& p, const AttnForwardMaps& m, cudaStream_t st, int pos) {
  const bool cap = p.cap > 0.0f;
  switch (pos) {
    case 0: return cap ? launch<T, DP, 0, true>(p, m, st) : launch<T, DP, 0, false>(p, m, st);
    case 1: return cap ? launch<T, DP, 1, true>(p, m, st) : launch<T, DP, 1, false>(p, m, st);
    default: return cap ? launch<T, DP, 2, true>(p, m, st) : launch<T, DP, 2, false>(p, m, st);
  }
}

}  // namespace

// This source is compiled once for each padded head dimension.
#define S4D_CAT2(a, b) a##b
#define S4D_CAT(a, b) S4D_CAT2(a, b)
int S4D_CAT(launch_attention_forward_d, S4D_HEAD_DIM)(int dtype, int pos, const AttnParams& p,
                                                     const AttnForwardMaps& m, cudaStream_t st) {
  int rc = dtype == S4D_DTYPE_BF16 ? by_scores<__nv_bfloat16, S4D_HEAD_DIM>(p, m, st, pos)
                                   : by_scores<__half, S4D_HEAD_DIM>(p, m, st, pos);
  if (rc != S4D_OK || p.splits == p.cluster) return rc;
  const int64_t rows = int64_t(p.batch) * p.nq * p.heads;
  const dim3 grid(unsigned((rows + 7) / 8));
  const cudaError_t e = dtype == S4D_DTYPE_BF16
                            ? launch_pdl(true, attention_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p)
                            : launch_pdl(true, attention_join_kernel<__half>, grid, dim3(256), 0, st, p);
  return cuda_check(e, "attention_join_kernel launch");
}

}  // namespace s4d
