// Attention forward (formulas in decoder_attention.cuh):  o_i = sum_j p_ij v_j,  p = softmax over
// the allowed keys, in one pass over the keys with a running maximum m and sum l per row.
//
// One CTA owns 128 rows of one shared head: row r is query r / rep of head g rep + r % rep, so that
// the rep heads that share keys read them once.  It walks the keys in tiles of 64:
//   one warp    loads K and V tiles by TMA into rings of shared memory;
//   one warp    issues S = Q K^T for the next tile into one of two score buffers in tensor memory (64
//               columns each), and once P of this tile is there O += P V, with P read from tensor
//               memory and V as an MN-major operand;
//   the others  one row a thread: scores from tensor memory, cap, bias and mask in registers (two
//               scores an instruction), the row maximum without a shuffle, P = 2^(s - m) back over S
//               as 16-bit pairs.
// O is only rescaled when a row's maximum grew by more than 2^8 since the last time: P then stays
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
// Few rows and many keys: the keys are cut into parts, each CTA writes its part's normalised O and
// log-sum-exp, and a second launch joins them.
#include "decoder_attention.cuh"

namespace s4d {
namespace {

constexpr int kKeys = 64;  // keys of a tile

template <int DP>
struct Fwd {
  static constexpr int kOwnBlock = kAttnRows * 128, kBlock = kKeys * 128;  // 64 columns of Q, of K or V
  static constexpr int kQ = DP / 64 * kOwnBlock, kTile = DP / 64 * kBlock;
  static constexpr int kStages = DP == 64 ? 4 : 2;     // of K and of V
  static constexpr int kStreams = DP == 64 ? 2 : 1;    // stream s walks every kStreams-th tile from s
  static constexpr int kWarps = 4 * kStreams;          // row threads; then the TMA and the tensor-core warp
  static constexpr int kThreads = (kWarps + 2) * 32;
  static constexpr int kK = kQ, kV = kK + kStages * kTile, kAux = kV + kStages * kTile;
  // per row warp: negated x, y of the keys and their segments (after the last tile: m and l of its
  // rows); barriers; tensor-memory slot, abort, skip[2]
  static constexpr int kBars = kAux + kWarps * 3 * kKeys * 4;
  static constexpr int kNumBars = 4 * kStages + 7;
  static constexpr int kCtl = kBars + kNumBars * 8;
  static constexpr int kKinds = kCtl + 16;
  static constexpr uint32_t kCols = 256;  // S / P: 2 x 64, O: DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

// 32 scores of a row, in base 2, and their maximum.
template <int POS, bool CAP, bool MASKED>
__device__ __forceinline__ void scores(uint32_t (&r)[32], const ScoreConst& k, float slope2, float qx, float qy,
                                       int seg, const float* aux, float& mx) {
  const F2 x2 = f2(qx), y2 = f2(qy), nslope = f2(-slope2), k1 = f2(k.k1), c = f2(k.c), nc = f2(-k.c);
#pragma unroll
  for (int j4 = 0; j4 < 32; j4 += 4) {
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
        const F2 nx = u == 0 ? f2(x4.x, x4.y) : f2(x4.z, x4.w);
        F2 ny = nx;
        if constexpr (POS > 1) ny = u == 0 ? f2(y4.x, y4.y) : f2(y4.z, y4.w);
        s = fma2(nslope, distance<POS>(x2, y2, nx, ny), s);
      }
      float a, b;
      split(s, a, b);
      if constexpr (MASKED) {
        a = (u == 0 ? s4.x : s4.z) == seg ? a : -INFINITY;
        b = (u == 0 ? s4.y : s4.w) == seg ? b : -INFINITY;
      }
      mx = max3(mx, a, b);
      r[j4 + u] = __float_as_uint(a);
      r[j4 + u + 1] = __float_as_uint(b);
    }
  }
}

// Their weights 2^(s - m) as 16-bit pairs, and the sum of the unrounded weights.
template <typename T>
__device__ __forceinline__ void weights(const uint32_t (&r)[32], F2 nbase, F2 (&sum)[2], uint32_t* w) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float a, d;
    split(add2(f2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), nbase), a, d);
    a = ex2(a), d = ex2(d);
    sum[e & 1] = add2(sum[e & 1], f2(a, d));
    w[e] = pack2<T>(a, d);
  }
}

template <typename T, int DP, int POS, bool CAP>
__global__ void __launch_bounds__(Fwd<DP>::kThreads, 2)
    attention_forward_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                             const AttnParams p) {
  using S = Fwd<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t k_full = sbase + S::kBars, k_empty = k_full + 8 * S::kStages, v_full = k_empty + 8 * S::kStages,
                 v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages, p_full = s_full + 16,
                 pv_done = p_full + 16, o_full = pv_done + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* skip_pv = abort_flag + 1;
  unsigned char* kinds = smem + S::kKinds;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // blockIdx.x = ((b G + g) row tiles + row tile) splits + part
  const int64_t rows = p.nq * p.rep, row_tiles = (rows + kAttnRows - 1) / kAttnRows;
  int64_t u = blockIdx.x;
  const int part = int(u % p.splits);
  u /= p.splits;
  const int64_t row0 = u % row_tiles * kAttnRows;
  u /= row_tiles;
  const int g = int(u % p.kv_heads), b = int(u / p.kv_heads);

  // keys of this part
  const int64_t first = part * p.tiles_per_split;
  int64_t valid = p.nk;
  if (p.k_len != nullptr) valid = min(valid, max(int64_t(0), int64_t(__ldg(p.k_len + b))));
  const int64_t all_tiles = (valid + kKeys - 1) / kKeys;
  const int tiles = int(max(int64_t(0), min(p.tiles_per_split, all_tiles - first)));

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(k_full + 8 * s, 1);
      mbar_init(k_empty + 8 * s, 1);
      mbar_init(v_full + 8 * s, 1);
      mbar_init(v_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + 8 * s, 1);
      mbar_init(p_full + 8 * s, kAttnRows);
      mbar_init(pv_done + 8 * s, 1);
    }
    mbar_init(o_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == S::kWarps + 1) tmem_alloc(smem_u32(tmem_slot), S::kCols);
  {
    const bool segs = p.q_seg != nullptr;
    SegRange own{0, 0, true};
    if (segs) {
      const int64_t i0 = row0 / p.rep, i1 = (min(rows, row0 + kAttnRows) - 1) / p.rep;
      own = seg_range(p.q_seg + b * p.nq + i0, int(i1 - i0 + 1));
    }
    classify_tiles(kinds, first, tiles, kKeys, valid, segs ? p.k_seg + b * p.nk : nullptr, own, true);
  }
  const uint32_t rep = uint32_t(p.rep);  // rows of a shared head stay below 2^31
  // Q: 16-byte pieces, zero past the last row and column, in the swizzled layout TMA gives K and V
  for (int c = threadIdx.x; c < kAttnRows * (DP / 8); c += S::kThreads) {
    const int r = c / (DP / 8), d = c % (DP / 8);
    const int64_t row = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows && d * 8 < p.dim)
      v = ldg_nc_v4(static_cast<const T*>(p.q) + b * p.q_sb + int64_t(uint32_t(row) / rep) * p.q_sn + (g * p.rep + uint32_t(row) % rep) * p.q_sh +
                    d * 8);
    *reinterpret_cast<uint4*>(smem + (d / 8) * S::kOwnBlock + r * 128 + (((d & 7) ^ (r & 7)) << 4)) = v;
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 2 * kKeys;
  const int t0 = next_tile(kinds, -1, tiles);

  if (warp == S::kWarps) {
    if (lane == 0) {
      int n = 0;
      for (int t = t0; t < tiles; t = next_tile(kinds, t, tiles), ++n) {
        const int s = n % S::kStages;
        const uint32_t parity = (n / S::kStages + 1) & 1;
        const int key = int((first + t) * kKeys);
        if (n >= S::kStages && !mbar_wait(k_empty + 8 * s, parity, abort_flag, p.wait_limit_ns)) break;
        load_tile<DP, kKeys>(sbase + S::kK + s * S::kTile, &km, k_full + 8 * s, g, key, b);
        if (n >= S::kStages && !mbar_wait(v_empty + 8 * s, parity, abort_flag, p.wait_limit_ns)) {
          // the K load is out: it may not land in the memory of a CTA that is gone
          mbar_wait(k_full + 8 * s, (n / S::kStages) & 1, nullptr);
          break;
        }
        load_tile<DP, kKeys>(sbase + S::kV + s * S::kTile, &vm, v_full + 8 * s, g, key, b);
      }
      for (int i = max(0, n - S::kStages); i < n; ++i) {
        mbar_wait(k_full + 8 * (i % S::kStages), (i / S::kStages) & 1, nullptr);
        mbar_wait(v_full + 8 * (i % S::kStages), (i / S::kStages) & 1, nullptr);
      }
    }
  } else if (warp == S::kWarps + 1) {
    if (lane == 0) {
      // S of tile n, n counting the walked tiles
      auto issue_scores = [&](int n) {
        const int s = n % S::kStages;
        if (!mbar_wait(k_full + 8 * s, (n / S::kStages) & 1, abort_flag, p.wait_limit_ns)) return false;
        tc_fence_after();
        mma_scores<T, DP>(tmem + (n & 1) * kKeys, sbase, S::kOwnBlock, sbase + S::kK + s * S::kTile, S::kBlock, kKeys);
        mma_commit(k_empty + 8 * s);
        mma_commit(s_full + 8 * (n & 1));
        return true;
      };
      // the scores of two tiles are out before the first P is waited for, and tile n + 2's follow the
      // product of P of tile n, whose buffer they go over: the tensor cores work in order
      const int t1 = next_tile(kinds, t0, tiles);
      bool ok = t0 >= tiles || (issue_scores(0) && (t1 >= tiles || issue_scores(1)));
      int n = 0, ahead = t1 < tiles ? next_tile(kinds, t1, tiles) : tiles;
      for (int t = t0; ok && t < tiles; t = next_tile(kinds, t, tiles), ++n) {
        const int s = n % S::kStages;
        ok = mbar_wait(v_full + 8 * s, (n / S::kStages) & 1, abort_flag, p.wait_limit_ns) &&
             mbar_wait(p_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
        if (!ok) break;
        tc_fence_after();
        if (!(kinds[t] == kTileMasked && skip_pv[n & 1]))
          mma_accumulate<T, DP, kKeys>(tmem_o + n % S::kStreams * DP, tmem + (n & 1) * kKeys,
                                       sbase + S::kV + s * S::kTile, n >= S::kStreams);
        mma_commit(v_empty + 8 * s);
        mma_commit(pv_done + 8 * (n % S::kStreams));
        if (ahead < tiles) {
          ok = issue_scores(n + 2);
          ahead = next_tile(kinds, ahead, tiles);
        }
      }
      mma_commit(o_full);  // also on the abort path: nothing may run once tensor memory is freed
      mbar_wait(o_full, 0, nullptr);
    }
  } else {
    const int stream = warp / 4, tid = threadIdx.x & 127;  // tid: the row, and the tensor-memory lane
    const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
    const int64_t row = row0 + tid;
    const bool live = row < rows;
    const int64_t i = live ? uint32_t(row) / rep : 0;
    const int h = g * p.rep + (live ? int(uint32_t(row) % rep) : 0);
    const bool warp_live = row0 + warp % 4 * 32 < rows;
    const ScoreConst k(p);
    float slope2 = 0.0f, qx = 0.0f, qy = 0.0f;
    if constexpr (POS > 0) {
      slope2 = __ldg(p.slopes + b * p.sl_b + i * p.sl_n + h * p.sl_h) * kLog2e;
      qx = __ldg(p.q_pos + (b * p.nq + i) * POS);
      if constexpr (POS > 1) qy = __ldg(p.q_pos + (b * p.nq + i) * POS + 1);
    }
    // segments: own -2 (matches nothing) or >= 0; keys -1 when masked; without segments 0 and 0 / -1
    int seg = 0;
    if (p.q_seg != nullptr) {
      seg = __ldg(p.q_seg + b * p.nq + i);
      if (seg < 0) seg = -2;
    }
    float* aux = reinterpret_cast<float*>(smem + S::kAux) + warp * 3 * kKeys;  // [3][64]: -x, -y, segment
    // two keys of the next tile a lane, loaded one tile ahead
    float2 nx = make_float2(0.0f, 0.0f), ny = nx;
    int2 ns = make_int2(-1, -1);
    auto fetch = [&](int t) {
      if (t >= tiles) return;
      const int64_t j = (first + t) * kKeys + 2 * lane;
      const int64_t at = b * p.nk + j;
      const bool in0 = j < valid, in1 = j + 1 < valid;
      ns.x = in0 ? (p.k_seg != nullptr ? max(-1, __ldg(p.k_seg + at)) : 0) : -1;
      ns.y = in1 ? (p.k_seg != nullptr ? max(-1, __ldg(p.k_seg + at + 1)) : 0) : -1;
      if constexpr (POS > 0) {
        nx.x = in0 ? -__ldg(p.k_pos + at * POS) : 0.0f;
        nx.y = in1 ? -__ldg(p.k_pos + (at + 1) * POS) : 0.0f;
        if constexpr (POS > 1) {
          ny.x = in0 ? -__ldg(p.k_pos + at * POS + 1) : 0.0f;
          ny.y = in1 ? -__ldg(p.k_pos + (at + 1) * POS + 1) : 0.0f;
        }
      }
    };
    auto nth = [&](int t, int steps) {  // `steps` walked tiles on
      for (int e = 0; e < steps && t < tiles; ++e) t = next_tile(kinds, t, tiles);
      return t;
    };
    int t = nth(t0, stream);
    fetch(t);
    float m = -INFINITY, l = 0.0f;
    bool dead = false;
    int n = stream;
    for (; t < tiles; n += S::kStreams) {
      const int next = nth(t, S::kStreams);
      const bool masked = kinds[t] == kTileMasked, first_tile = n == stream;
      if (POS > 0 || masked) {
        __syncwarp();
        if constexpr (POS > 0) *reinterpret_cast<float2*>(aux + 2 * lane) = nx;
        if constexpr (POS > 1) *reinterpret_cast<float2*>(aux + kKeys + 2 * lane) = ny;
        *reinterpret_cast<int2*>(aux + 2 * kKeys + 2 * lane) = ns;
        __syncwarp();
      }
      fetch(next);
      bool bad = false;  // a masked tile whose V holds values that are no numbers
      const unsigned char* vt = smem + S::kV + n % S::kStages * S::kTile;
      const uint32_t tmem_s = tmem + lanes + (n & 1) * kKeys, tmem_acc = tmem_o + lanes + stream * DP;
      if (masked) {
        if (!dead) dead = !warp_wait(v_full + 8 * (n % S::kStages), (n / S::kStages) & 1, abort_flag, p.wait_limit_ns);
        bad = barrier_any(1 + stream, kAttnRows, !dead && tid < kKeys && row_not_finite<T, DP>(vt, S::kBlock, tid));
        if (tid == 0) skip_pv[n & 1] = bad;
      }
      if (!dead) dead = !warp_wait(s_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
      if (!dead && warp_live) {
        // With two streams a thread has 96 registers: the first half of the scores waits in tensor memory.
        uint32_t r0[32], r1[32];
        float mx = -INFINITY;
        if constexpr (S::kStreams == 2) {
          tmem_ld32_async(tmem_s, r0);
          tmem_ld_wait(r0);
          if (masked)
            scores<POS, CAP, true>(r0, k, slope2, qx, qy, seg, aux, mx);
          else
            scores<POS, CAP, false>(r0, k, slope2, qx, qy, seg, aux, mx);
          tmem_st32(tmem_s, r0);
          tmem_ld32_async(tmem_s + 32, r1);
          tmem_ld_wait(r1);
        } else {
          tmem_ld32_async(tmem_s, r0);
          tmem_ld32_async(tmem_s + 32, r1);
          tmem_ld_wait(r0);
          tmem_ld_wait(r1);
          if (masked)
            scores<POS, CAP, true>(r0, k, slope2, qx, qy, seg, aux, mx);
          else
            scores<POS, CAP, false>(r0, k, slope2, qx, qy, seg, aux, mx);
        }
        if (masked)
          scores<POS, CAP, true>(r1, k, slope2, qx, qy, seg, aux + 32, mx);
        else
          scores<POS, CAP, false>(r1, k, slope2, qx, qy, seg, aux + 32, mx);
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
        uint32_t w[32];
        weights<T>(r1, nbase, sum, w + 16);
        if constexpr (S::kStreams == 2) {
          tmem_st_wait();
          tmem_ld32_async(tmem_s, r0);
          tmem_ld_wait(r0);
        }
        weights<T>(r0, nbase, sum, w);
        tmem_st32(tmem_s, w);
        float a, d;
        split(add2(sum[0], sum[1]), a, d);
        l += a + d;
        tmem_st_wait();
        if (bad && !dead) accumulate_nonzero<T, DP, kKeys>(tmem_acc, tmem_s, vt, first_tile);
      }
      tc_fence_before();
      mbar_arrive(p_full + 8 * (n & 1));
      t = next;
    }
    // O / l, the log-sum-exp, and zeros for rows without a key.  Two streams: each takes half of the
    // columns and adds what both have there.
    if (!dead && t0 < tiles) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    float m1 = -INFINITY, l1 = 0.0f;  // the other stream's
    if constexpr (S::kStreams == 2) {
      float* ml = reinterpret_cast<float*>(smem + S::kAux);  // the keys' values are not needed any more ...
      barrier_sync(3, S::kWarps * 32);                       // ... by any warp
      ml[stream * 256 + tid] = m;
      ml[stream * 256 + 128 + tid] = l;
      barrier_sync(3, S::kWarps * 32);
      m1 = ml[(stream ^ 1) * 256 + tid];
      l1 = ml[(stream ^ 1) * 256 + 128 + tid];
    }
    if (!dead && warp_live) {
      const bool any0 = l != 0.0f, any1 = l1 != 0.0f;  // else tensor memory holds nothing of this row
      const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
      float f0 = S::kStreams == 2 ? ex2(m - base) : 1.0f, f1 = ex2(m1 - base);
      const float total = S::kStreams == 2 ? fmaf(l, f0, l1 * f1) : l;
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      f0 *= inv, f1 *= inv;
      const int64_t out_row = (b * p.nq + i) * p.heads + h, lse_row = (int64_t(b) * p.heads + h) * p.nq + i;
      const int64_t all_rows = int64_t(p.batch) * p.nq * p.heads;
      const float lse = total != 0.0f ? (top + log2f(total)) * kLn2 : -INFINITY;
      if (live && stream == 0) {
        if (p.splits > 1)
          p.part_lse[part * all_rows + lse_row] = lse;
        else if (p.lse != nullptr)
          p.lse[lse_row] = lse;
      }
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
        if (!live) continue;
        if (p.splits > 1) {
          float* dst = p.part_o + (part * all_rows + out_row) * p.dim + c * 32;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c * 32 + e * 4 < p.dim)
              *reinterpret_cast<float4*>(dst + e * 4) = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
        } else {
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
  __syncthreads();
  if (warp == S::kWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kCols);
  }
  if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr) atomicOr(p.error_flag, S4D_FLAG_WAIT_TIMEOUT);
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
    const float w = ex2((p.part_lse[s * rows + lse_row] - base) * kLog2e);
    total += w;
    if (mine && w != 0.0f) {  // a part without keys has weight 0
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

template <typename T, int DP, int POS, bool CAP>
int launch(const AttnParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  static bool smem_set[64] = {};
  const int rc = set_kernel_smem(attention_forward_kernel<T, DP, POS, CAP>, Fwd<DP>::smem(kAttnMaxTiles),
                                 "cudaFuncSetAttribute(attention_forward_kernel)", smem_set);
  if (rc != S4D_OK) return rc;
  const int64_t row_tiles = (p.nq * p.rep + kAttnRows - 1) / kAttnRows;
  const dim3 grid(unsigned(row_tiles * p.kv_heads * p.batch * p.splits));
  attention_forward_kernel<T, DP, POS, CAP><<<grid, Fwd<DP>::kThreads, Fwd<DP>::smem(p.tiles_per_split), st>>>(km, vm, p);
  return cuda_check(cudaGetLastError(), "attention_forward_kernel launch");
}

template <typename T, int DP>
int by_scores(const AttnParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st, int pos) {
  const bool cap = p.cap > 0.0f;
  switch (pos) {
    case 0: return cap ? launch<T, DP, 0, true>(p, km, vm, st) : launch<T, DP, 0, false>(p, km, vm, st);
    case 1: return cap ? launch<T, DP, 1, true>(p, km, vm, st) : launch<T, DP, 1, false>(p, km, vm, st);
    default: return cap ? launch<T, DP, 2, true>(p, km, vm, st) : launch<T, DP, 2, false>(p, km, vm, st);
  }
}

}  // namespace

// This source is compiled once for each padded head dimension.
#define S4D_CAT2(a, b) a##b
#define S4D_CAT(a, b) S4D_CAT2(a, b)
int S4D_CAT(launch_attention_forward_d, S4D_HEAD_DIM)(int dtype, int pos, const AttnParams& p, const CUtensorMap& km,
                                                     const CUtensorMap& vm, cudaStream_t st) {
  int rc = dtype == S4D_DTYPE_BF16 ? by_scores<__nv_bfloat16, S4D_HEAD_DIM>(p, km, vm, st, pos)
                                   : by_scores<__half, S4D_HEAD_DIM>(p, km, vm, st, pos);
  if (rc != S4D_OK || p.splits == 1) return rc;
  const int64_t rows = int64_t(p.batch) * p.nq * p.heads;
  const dim3 grid(unsigned((rows + 7) / 8));
  const cudaError_t e = dtype == S4D_DTYPE_BF16
                            ? launch_pdl(true, attention_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p)
                            : launch_pdl(true, attention_join_kernel<__half>, grid, dim3(256), 0, st, p);
  return cuda_check(e, "attention_join_kernel launch");
}

}  // namespace s4d
