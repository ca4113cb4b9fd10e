// Attention forward (formulas in decoder_attention.cuh):  o_i = sum_j p_ij v_j,  p = softmax over
// the allowed keys, in one pass over the keys with a running maximum m and sum l per row.
//
// One CTA owns 128 rows of one shared head: row r is query r / rep of head g rep + r % rep, so that
// the rep heads that share keys read them once.  It walks the keys in tiles of 64:
//   warp 4      loads K and V tiles by TMA into rings of shared memory;
//   warp 5      issues S = Q K^T for the next tile into one of two score buffers in tensor memory (64
//               columns each), and once P of this tile is there O += P V, with P read from tensor
//               memory and V as an MN-major operand;
//   warps 0-3   one row a thread: scores from tensor memory, cap, bias and mask in registers (two
//               scores an instruction), the row maximum without a shuffle, P = 2^(s - m) back over S
//               as 16-bit pairs.
// O is only rescaled when a row's maximum grew by more than 2^8 since the last time: P then stays
// under 2^8, which costs no precision in a float.  P is rounded to the inputs' type because the
// tensor cores multiply it with V in that type; l adds the unrounded values in fp32.
//
// What bounds it: a score costs one exponential (16 a clock on an SM), a second special-function
// instruction with a 2-D distance and two more with a cap, against 4 D flops: for D = 64 the
// exponentials take four times as long as the products.  So the row threads must not wait: the next
// tile's scores are always under way, and two CTAs share an SM (256 tensor-memory columns and at
// most 113 KB of shared memory each).
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
  static constexpr int kK = kQ, kV = kK + kStages * kTile, kAux = kV + kStages * kTile;
  // negated x, y of the keys and their segments, two buffers; barriers; tensor-memory slot, abort, skip[2]
  static constexpr int kBars = kAux + 2 * 3 * kKeys * 4;
  static constexpr int kNumBars = 4 * kStages + 6;
  static constexpr int kCtl = kBars + kNumBars * 8;
  static constexpr int kKinds = kCtl + 16;
  static constexpr uint32_t kCols = 256;  // S / P: 2 x 64, O: DP
  static size_t smem(int64_t tiles) { return size_t(kKinds) + size_t((tiles + 15) / 16 * 16) + 1024; }
};

// The 64 scores of a row, in base 2, and their maximum.
template <int POS, bool CAP, bool MASKED>
__device__ __forceinline__ void scores(uint32_t (&r)[64], const ScoreConst& k, float slope2, float qx, float qy,
                                       int seg, const float* aux, float& mx) {
  const F2 x2 = f2(qx), y2 = f2(qy), nslope = f2(-slope2), k1 = f2(k.k1), c = f2(k.c), nc = f2(-k.c);
#pragma unroll
  for (int j4 = 0; j4 < kKeys; j4 += 4) {
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

template <typename T, int DP, int POS, bool CAP>
__global__ void __launch_bounds__(kAttnThreads, 2)
    attention_forward_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                             const AttnParams p) {
  using S = Fwd<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t k_full = sbase + S::kBars, k_empty = k_full + 8 * S::kStages, v_full = k_empty + 8 * S::kStages,
                 v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages, p_full = s_full + 16,
                 pv_done = p_full + 16, o_full = pv_done + 8;
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
    }
    mbar_init(pv_done, 1);
    mbar_init(o_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), S::kCols);
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
  for (int c = threadIdx.x; c < kAttnRows * (DP / 8); c += kAttnThreads) {
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

  if (warp == 4) {
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
  } else if (warp == 5) {
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
      int n = 0;
      bool ok = t0 >= tiles || issue_scores(0);
      for (int t = t0; ok && t < tiles; ++n) {
        const int s = n % S::kStages, next = next_tile(kinds, t, tiles);
        // The next scores go over P of the tile before this one, whose product with V is issued: the
        // tensor cores work in order.
        if (next < tiles && !(ok = issue_scores(n + 1))) break;
        ok = mbar_wait(v_full + 8 * s, (n / S::kStages) & 1, abort_flag, p.wait_limit_ns) &&
             mbar_wait(p_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
        if (!ok) break;
        tc_fence_after();
        if (!(kinds[t] == kTileMasked && skip_pv[n & 1]))
          mma_accumulate<T, DP, kKeys>(tmem_o, tmem + (n & 1) * kKeys, sbase + S::kV + s * S::kTile, n > 0);
        mma_commit(v_empty + 8 * s);
        mma_commit(pv_done);
        t = next;
      }
      mma_commit(o_full);  // also on the abort path: nothing may run once tensor memory is freed
      mbar_wait(o_full, 0, nullptr);
    }
  } else {
    const int tid = threadIdx.x;
    const uint32_t lanes = uint32_t(warp * 32) << 16;
    const int64_t row = row0 + tid;
    const bool live = row < rows;
    const int64_t i = live ? uint32_t(row) / rep : 0;
    const int h = g * p.rep + (live ? int(uint32_t(row) % rep) : 0);
    const bool warp_live = row0 + warp * 32 < rows;
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
    float* aux = reinterpret_cast<float*>(smem + S::kAux);  // [2][3][64]: -x, -y, segment
    // threads 0-63: a key of the next tile, loaded one tile ahead
    float nx = 0.0f, ny = 0.0f;
    int ns = -1;
    auto fetch = [&](int t) {
      if (t >= tiles || tid >= kKeys) return;
      const int64_t j = (first + t) * kKeys + tid;
      const bool in = j < valid;
      ns = in ? (p.k_seg != nullptr ? max(-1, __ldg(p.k_seg + b * p.nk + j)) : 0) : -1;
      if constexpr (POS > 0) {
        nx = in ? -__ldg(p.k_pos + (b * p.nk + j) * POS) : 0.0f;
        if constexpr (POS > 1) ny = in ? -__ldg(p.k_pos + (b * p.nk + j) * POS + 1) : 0.0f;
      }
    };
    fetch(t0);
    float m = -INFINITY, l = 0.0f;
    bool dead = false;
    int n = 0;
    for (int t = t0; t < tiles; ++n) {
      const int next = next_tile(kinds, t, tiles);
      const bool masked = kinds[t] == kTileMasked;
      float* bx = aux + (n & 1) * 3 * kKeys;
      if (tid < kKeys) {
        bx[tid] = nx;
        bx[kKeys + tid] = ny;
        reinterpret_cast<int*>(bx)[2 * kKeys + tid] = ns;
      }
      rows_sync();
      fetch(next);
      bool bad = false;  // a masked tile whose V holds values that are no numbers
      const unsigned char* vt = smem + S::kV + n % S::kStages * S::kTile;
      const uint32_t tmem_s = tmem + lanes + (n & 1) * kKeys;
      if (masked) {
        if (!dead) dead = !warp_wait(v_full + 8 * (n % S::kStages), (n / S::kStages) & 1, abort_flag, p.wait_limit_ns);
        bad = rows_any(!dead && tid < kKeys && row_not_finite<T, DP>(vt, S::kBlock, tid));
        if (tid == 0) skip_pv[n & 1] = bad;
      }
      if (!dead) dead = !warp_wait(s_full + 8 * (n & 1), (n >> 1) & 1, abort_flag, p.wait_limit_ns);
      if (!dead && warp_live) {
        uint32_t r[kKeys];
        tmem_ld32_async(tmem_s, r);
        tmem_ld32_async(tmem_s + 32, r + 32);
        tmem_ld_wait(r);
        float mx = -INFINITY;
        if (masked)
          scores<POS, CAP, true>(r, k, slope2, qx, qy, seg, bx, mx);
        else
          scores<POS, CAP, false>(r, k, slope2, qx, qy, seg, bx, mx);
        const bool grow = mx > m + 8.0f || (m == -INFINITY && mx > m);
        const bool any_grow = __any_sync(0xffffffffu, grow);
        if (n > 0 && (any_grow || bad))  // O is about to change outside the tensor cores
          dead = !warp_wait(pv_done, (n - 1) & 1, abort_flag, p.wait_limit_ns);
        if (any_grow && !dead) {
          const float f = grow ? ex2(m - mx) : 1.0f;  // 0 for a row's first keys
          if (grow) m = mx;
          l *= f;
          if (n > 0) {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
              uint32_t o[16];
              tmem_ld16_async(tmem_o + lanes + c * 16, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(tmem_o + lanes + c * 16, o);
            }
          }
        }
        const F2 nbase = f2(m == -INFINITY ? 0.0f : -m);  // no key yet: every score is -inf, every weight 0
        F2 sum[2] = {f2(0.0f), f2(0.0f)};
        uint32_t w[kKeys / 2];
#pragma unroll
        for (int e = 0; e < kKeys / 2; ++e) {
          float a, d;
          split(add2(f2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), nbase), a, d);
          a = ex2(a), d = ex2(d);
          sum[e & 1] = add2(sum[e & 1], f2(a, d));
          w[e] = pack2<T>(a, d);
        }
        tmem_st32(tmem_s, w);
        float a, d;
        split(add2(sum[0], sum[1]), a, d);
        l += a + d;
        tmem_st_wait();
        if (bad && !dead) accumulate_nonzero<T, DP, kKeys>(tmem_o + lanes, tmem_s, vt, n == 0);
      }
      tc_fence_before();
      mbar_arrive(p_full + 8 * (n & 1));
      t = next;
    }
    // O / l, the log-sum-exp, and zeros for rows without a key
    if (!dead && n > 0) dead = !warp_wait(o_full, 0, abort_flag, p.wait_limit_ns);
    if (!dead && warp_live) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const bool any = n > 0 && l != 0.0f;  // else tensor memory holds nothing of this row
      const int64_t out_row = (b * p.nq + i) * p.heads + h, lse_row = (int64_t(b) * p.heads + h) * p.nq + i;
      const int64_t all_rows = int64_t(p.batch) * p.nq * p.heads;
      const float lse = any ? (m + log2f(l)) * kLn2 : -INFINITY;
      if (live) {
        if (p.splits > 1)
          p.part_lse[part * all_rows + lse_row] = lse;
        else if (p.lse != nullptr)
          p.lse[lse_row] = lse;
      }
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        if (c * 32 >= p.dim) break;
        uint32_t o[32];
        tmem_ld32_async(tmem_o + lanes + c * 32, o);
        tmem_ld_wait(o);
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = any ? __uint_as_float(o[e]) * inv : 0.0f;
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
  if (warp == 5) {
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
  attention_forward_kernel<T, DP, POS, CAP><<<grid, kAttnThreads, Fwd<DP>::smem(p.tiles_per_split), st>>>(km, vm, p);
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
