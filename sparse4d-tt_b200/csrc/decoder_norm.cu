// LayerNorm rows of any width up to 16384, forward and backward (f32, bf16, f16).
//
// Forward, one row r of N values:   n = (x - mean) rstd,  y = n w + b.
// Backward, with g = dy w:          dx = rstd (g - mean(g) - n mean(g n)),
//                                   dw = sum_r dy n,  db = sum_r dy.
// Both are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.
// So each row is read once, into the registers of a group of W warps (16 values a thread at most:
// W = 1 up to 512 columns, 2 up to 1024, ... 32 up to 16384), in 16-byte vectors where the row
// pointers and strides allow it and single elements otherwise; the mean and then the variance of
// the deviations from it (no cancellation for rows far from zero) are reduced by shuffles and,
// for W > 1, through shared memory.
//
// A block keeps the weight and bias of its columns in registers and walks the rows with the stride of a grid
// that just fills the SMs, the next row's loads under way during one row's sums (not in the backward
// pass of f32 rows, where registers are short).  Reading the parameters again for every row costs more
// than the rows: 16,384 x 4,096 bf16 forward 69 us against 49 us.
// Up to eight warps a row the registers are held to what lets three (backward: two) blocks of eight warps
// share an SM: what a block waits for, the others load over.  16,384 x 4,096 bf16 both passes 172 us with
// the compiler's choice (two and one), 158 so; 7,213 x 1,001 f16 26.9 and 25.8.  The f32 forward kernels spill 20 to
// 28 bytes for it and still gain where rows are long enough for the blocks to matter: 16,384 x 2,048 47.1 us with two,
// 45.1 with three; 7,000 x 768 10.5 and 9.9; 28,800 x 512 21.4 either way; of the sizes tried only 16,384 x 4,096
// loses (89 and 94).
// Graph times by now, forward and backward: 16,384 x 4,096 bf16 51 and 90 us, f16 52 and 89; 28,800 x 512 f32 21 and
// 33; 7,213 x 1,001 f16 11.5 and 17.2; 4,096 x 16,384 bf16 107 and 173.
//
// The sums over rows for dw and db stay in registers: a block adds its row groups through shared memory
// and writes one fp32 partial row per block; a second launch adds the partial rows in block order.
// Small inputs (up to 2048 rows and 2^20 values, which stay in the L2 cache) need no second launch: more
// blocks of the same one each read 8 columns of x and dy again and add them over all rows.
// No atomics: the order of every addition depends on the sizes alone.
#include <algorithm>

#include "decoder_types.cuh"

namespace s4d {
namespace {

struct NormParams {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;   // forward: y; backward: dx (may be null)
  float* mean;
  float* rstd;
  float* partial;  // [row_blocks, 2, width]: dw then db of each block, or null
  int row_blocks;  // blocks that walk rows; the ones behind them sum columns
  void *dweight, *dbias;  // for those
  int64_t x_ld, dy_ld, y_ld;
  int64_t rows;
  int width;
  int param_f32;  // weight and bias are f32 (else T)
  float eps;
};

constexpr int kNormMaxWidth = 16384;
constexpr int kEpt = 16;  // values a thread holds of one row

template <int W>
struct Group {
  static constexpr int kWarps = W < 8 ? 8 : W;      // warps of a block
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = kWarps / W;          // rows a block holds at a time
};

// Sum over the W warps of a group; every thread gets it.  `red` holds one value per warp and is
// used once between two block barriers.
template <int W>
__device__ __forceinline__ float group_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (W > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const float* r = red + warp / W * W;
    if constexpr (W < 8) {
      v = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += r[i];
    } else {  // the unrolled loads are all issued at once and would take W registers
      v = r[threadIdx.x % W];
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
  }
  return v;
}

// VEC parameters from column col, as 16-byte vectors where the rows are (the pointer is checked with them).
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool f32, int col, float (&f)[VEC]) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + col;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(q + i));
        f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = __ldg(q + i);
    }
  } else {
    load_vec<T, VEC>(static_cast<const T*>(p) + col, f);
  }
}

// Chunk k of a thread covers columns [col, col + VEC), col = (k * 32 W + thread of the group) VEC.
template <typename T, int W, int VEC, int K>
__global__ void __launch_bounds__(Group<W>::kThreads, W <= 8 ? 3 : 1) norm_forward_kernel(const NormParams p) {
  constexpr int R = Group<W>::kRows;
  __shared__ float red[2][Group<W>::kWarps];
  const int group = threadIdx.x / (32 * W), gt = threadIdx.x % (32 * W);
  constexpr bool kHold = W < 32;  // 1024 threads have 64 registers: they read the parameters again
  float w[K][VEC], b[K][VEC];
  auto load_params = [&](int k) {
    const int col = (k * 32 * W + gt) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[k][i] = 1.0f, b[k][i] = 0.0f;
    if (col < p.width && p.weight != nullptr) load_param<T, VEC>(p.weight, p.param_f32, col, w[k]);
    if (col < p.width && p.bias != nullptr) load_param<T, VEC>(p.bias, p.param_f32, col, b[k]);
  };
  if (kHold) {
#pragma unroll
    for (int k = 0; k < K; ++k) load_params(k);
  }
  RawVec<T, VEC> raw[K];
  auto load_row = [&](int64_t row) {
    const T* xr = static_cast<const T*>(p.x) + row * p.x_ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * 32 * W + gt) * VEC;
      if (row < p.rows && col < p.width)
        raw[k].load(xr + col);
      else
        raw[k].clear();
    }
  };
  const float inv = 1.0f / float(p.width);
  const int64_t step = int64_t(gridDim.x) * R;
  if (kHold) load_row(int64_t(blockIdx.x) * R + group);
  for (int64_t base = int64_t(blockIdx.x) * R; base < p.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < p.rows;
    if (!kHold) load_row(row);
    float v[K][VEC];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      raw[k].widen(v[k]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += v[k][i];
    }
    if (kHold && base + step < p.rows) load_row(row + step);
    const float mean = group_sum<W>(s, red[0]) * inv;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((k * 32 * W + gt) * VEC < p.width) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = v[k][i] - mean;
          q = fmaf(d, d, q);
        }
      }
    }
    // red[0] is free again behind this sum's barrier, red[1] behind the next row's first
    const float rstd = 1.0f / sqrtf(group_sum<W>(q, red[1]) * inv + p.eps);
    if (!live) continue;
    if (gt == 0 && p.mean != nullptr) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    T* yr = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * 32 * W + gt) * VEC;
      if (col >= p.width) break;
      if (!kHold) load_params(k);
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = fmaf((v[k][i] - mean) * rstd, w[k][i], b[k][i]);
      store_vec<T, VEC>(yr + col, o);
    }
  }
}

// dw and db of 8 columns: a thread adds one column over every (threads / 8)-th row, then the row lanes are
// added by shuffles and through shared memory in a fixed order.
template <typename T, int THREADS>
__device__ __forceinline__ void sum_columns(const NormParams& p, int block) {
  __shared__ float sums[2][THREADS / 32][8];
  const int col = block * 8 + threadIdx.x % 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float a = 0.0f, b = 0.0f;
  if (col < p.width) {
    const T *x = static_cast<const T*>(p.x) + col, *dy = static_cast<const T*>(p.dy) + col;
#pragma unroll 4
    for (int64_t r = threadIdx.x / 8; r < p.rows; r += THREADS / 8) {
      const float d = to_f32<T>(dy[r * p.dy_ld]);
      a = fmaf(d, (to_f32<T>(x[r * p.x_ld]) - __ldg(p.mean + r)) * __ldg(p.rstd + r), a);
      b += d;
    }
  }
#pragma unroll
  for (int o = 16; o >= 8; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane < 8) sums[0][warp][lane] = a, sums[1][warp][lane] = b;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  const int which = threadIdx.x / 8, c = block * 8 + threadIdx.x % 8;
  void* out = which == 0 ? p.dweight : p.dbias;
  if (out == nullptr || c >= p.width) return;
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += sums[which][w][threadIdx.x % 8];
  if (p.param_f32)
    static_cast<float*>(out)[c] = v;
  else
    static_cast<T*>(out)[c] = from_f32<T>(v);
}

template <typename T, int W, int VEC, int K>
__global__ void __launch_bounds__(Group<W>::kThreads, W <= 8 ? 2 : 1) norm_backward_kernel(const NormParams p) {
  if (int(blockIdx.x) >= p.row_blocks) {
    sum_columns<T, Group<W>::kThreads>(p, int(blockIdx.x) - p.row_blocks);
    return;
  }
  constexpr int R = Group<W>::kRows;
  __shared__ float red[2][2][Group<W>::kWarps];  // two sums, two buffers: one barrier a row
  // at the end: partial sums of the block's row groups, a chunk at a time
  __shared__ float join[R > 1 ? 2 * R * 32 * W * VEC : 1];
  const int group = threadIdx.x / (32 * W), gt = threadIdx.x % (32 * W);
  griddep_launch_dependents();  // the reduction waits for this whole launch before it reads
  float w[K][VEC], aw[K][VEC], ab[K][VEC];
  auto load_weight = [&](int k) {
    const int col = (k * 32 * W + gt) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[k][i] = 1.0f;
    if (p.weight != nullptr && col < p.width) load_param<T, VEC>(p.weight, p.param_f32, col, w[k]);
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (W < 32) load_weight(k);
#pragma unroll
    for (int i = 0; i < VEC; ++i) aw[k][i] = 0.0f, ab[k][i] = 0.0f;
  }
  const float inv = 1.0f / float(p.width);
  int buf = 0;
  // the next row's loads under way during this row's sums, where the registers allow it
  constexpr bool kAhead = sizeof(T) == 2 && W < 32 && (VEC == 8 || K == 8);
  RawVec<T, VEC> rx[K], rd[K];
  auto load_row = [&](int64_t row) {
    const T* xr = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* dyr = static_cast<const T*>(p.dy) + row * p.dy_ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * 32 * W + gt) * VEC;
      if (row < p.rows && col < p.width) {
        rx[k].load(xr + col);
        rd[k].load(dyr + col);
      } else {
        rx[k].clear();
        rd[k].clear();
      }
    }
  };
  const int64_t step = int64_t(p.row_blocks) * R;
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto load_stats = [&](int64_t row) {
    if (row >= p.rows) return;
    next_mean = __ldg(p.mean + row);
    next_rstd = __ldg(p.rstd + row);
  };
  load_stats(int64_t(blockIdx.x) * R + group);
  if (kAhead) load_row(int64_t(blockIdx.x) * R + group);
  for (int64_t base = int64_t(blockIdx.x) * R; base < p.rows; base += step, buf ^= 1) {
    const int64_t row = base + group;
    const bool live = row < p.rows;
    const int64_t r = live ? row : 0;
    float n[K][VEC], g[K][VEC];
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        rx[k].widen(n[k]);
        rd[k].widen(g[k]);
      }
      if (base + step < p.rows) load_row(row + step);
    } else {
      const T* xr = static_cast<const T*>(p.x) + r * p.x_ld;
      const T* dyr = static_cast<const T*>(p.dy) + r * p.dy_ld;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int col = (k * 32 * W + gt) * VEC;
        if (live && col < p.width) {
          load_vec<T, VEC>(xr + col, n[k]);
          load_vec<T, VEC>(dyr + col, g[k]);
        }
      }
    }
    const float mean = next_mean, rstd = next_rstd;
    load_stats(row + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = live && (k * 32 * W + gt) * VEC < p.width;
      if (W == 32) load_weight(k);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float nn = in ? (n[k][i] - mean) * rstd : 0.0f, d = in ? g[k][i] : 0.0f;
        aw[k][i] = fmaf(d, nn, aw[k][i]);
        ab[k][i] += d;
        n[k][i] = nn;
        g[k][i] = d * w[k][i];
        s1 += g[k][i];
        s2 = fmaf(g[k][i], nn, s2);
      }
    }
    if (p.y == nullptr) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    if constexpr (W > 1) {
      const int warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0) red[buf][0][warp] = s1, red[buf][1][warp] = s2;
      __syncthreads();
      const int w0 = warp / W * W;
      if constexpr (W < 8) {
        s1 = s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) s1 += red[buf][0][w0 + i], s2 += red[buf][1][w0 + i];
      } else {  // as in group_sum (graph times of both passes, 16,384 x 4,096 bf16 158 us with the loads, 136
                // so; 4,096 x 16,384 472 and 273)
        s1 = red[buf][0][w0 + threadIdx.x % W], s2 = red[buf][1][w0 + threadIdx.x % W];
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) {
          s1 += __shfl_xor_sync(0xffffffffu, s1, o);
          s2 += __shfl_xor_sync(0xffffffffu, s2, o);
        }
      }
    }
    if (!live) continue;
    s1 *= inv, s2 *= inv;
    T* dxr = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * 32 * W + gt) * VEC;
      if (col >= p.width) break;
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = rstd * (g[k][i] - s1 - n[k][i] * s2);
      store_vec<T, VEC>(dxr + col, o);
    }
  }
  if (p.partial == nullptr) return;
  float* pw = p.partial + int64_t(blockIdx.x) * 2 * p.width;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (k * 32 * W + gt) * VEC;
    if constexpr (R > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        join[(group * VEC + i) * 32 * W + gt] = aw[k][i];
        join[((R + group) * VEC + i) * 32 * W + gt] = ab[k][i];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float a = 0.0f, b = 0.0f;
          for (int j = 0; j < R; ++j) {
            a += join[(j * VEC + i) * 32 * W + gt];
            b += join[((R + j) * VEC + i) * 32 * W + gt];
          }
          aw[k][i] = a, ab[k][i] = b;
        }
      }
    }
    if (group == 0 && col < p.width) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) pw[col + i] = aw[k][i], pw[p.width + col + i] = ab[k][i];
    }
  }
}

// dw and db from the blocks' partial rows: 32 columns a block, its 32 warps each adding every
// 32nd partial row, then the 32 sums in warp order.
template <typename P>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* partial, int blocks, int width, P* dweight,
                                                           P* dbias) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  P* out = blockIdx.y == 0 ? dweight : dbias;
  griddep_wait();
  if (out == nullptr) return;
  const float* src = partial + int64_t(blockIdx.y) * width + col;
  float s = 0.0f;
  if (col < width) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 32) s += src[int64_t(b) * 2 * width];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < width) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sums[i][lane];
    out[col] = from_f32<P>(s);
  }
}

// Warps a row is spread over: the fewest that hold it at kEpt values a thread.
int warps_for(int64_t width) {
  int w = 1;
  while (int64_t(w) * 32 * kEpt < width) w *= 2;
  return w;
}

int rows_per_block(int w) { return w < 8 ? 8 / w : 1; }

// Partial rows of dw and db at most: the blocks of a backward launch that fills the SMs (at most four of 256
// threads an SM, one of 512 or 1024).
int64_t most_row_blocks(int64_t rows, int64_t width) {
  const int w = warps_for(width), r = rows_per_block(w);
  const int64_t need = (rows + r - 1) / r, fill = int64_t(device_sms()) * (w <= 8 ? 4 : 1);
  return need < fill ? need : fill;
}

// Blocks of `kernel` that fill the device at once; the SMs' share is asked once per device and kernel.
template <typename Kern>
int64_t filling_blocks(Kern kernel, int threads, int (&cache)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  int each = dev >= 0 && dev < 64 ? cache[dev] : 0;
  if (each == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, threads, 0) != cudaSuccess || each < 1) {
      cudaGetLastError();
      each = 1;
    }
    if (dev >= 0 && dev < 64) cache[dev] = each;
  }
  return int64_t(device_sms()) * each;
}

// Whether dw and db are summed by the backward launch itself: while x and dy stay in the L2 cache and a
// thread adds at most 64 rows.  900 x 256 f32: one launch of 6.0 us against 4.5 + 4.7 us.
bool sums_in_one_launch(int64_t rows, int64_t width) { return rows <= 2048 && rows * width <= (1 << 20); }

// The forward launch; the backward launch, and into p.row_blocks how many partial rows it writes (with
// `columns` more blocks that sum columns).
template <typename T, int W, int VEC, int K>
int launch_norm(bool backward, NormParams& p, int64_t columns, cudaStream_t st) {
  static int cache[2][64] = {};
  constexpr int kThreads = Group<W>::kThreads;
  const int64_t need = (p.rows + Group<W>::kRows - 1) / Group<W>::kRows;
  if (backward) {
    const int64_t fill = filling_blocks(norm_backward_kernel<T, W, VEC, K>, kThreads, cache[1]);
    p.row_blocks = int(std::min(std::min(need, fill), most_row_blocks(p.rows, p.width)));
    norm_backward_kernel<T, W, VEC, K><<<dim3(unsigned(p.row_blocks + columns)), kThreads, 0, st>>>(p);
    return cuda_check(cudaGetLastError(), "norm_backward_kernel launch");
  }
  const int64_t fill = filling_blocks(norm_forward_kernel<T, W, VEC, K>, kThreads, cache[0]);
  norm_forward_kernel<T, W, VEC, K><<<dim3(unsigned(std::min(need, fill))), kThreads, 0, st>>>(p);
  return cuda_check(cudaGetLastError(), "norm_forward_kernel launch");
}

template <typename T, int VEC>
int dispatch_width(bool backward, NormParams& p, int64_t columns, cudaStream_t st) {
  constexpr int K = kEpt / VEC;
  if constexpr (VEC == 1) {
    // Rows that cannot be read as vectors are read an element at a time: half as many a thread and twice the
    // warps keep more of them under way (7,213 x 1,001 f16 forward 13.7 against 12.4 us, backward
    // 26.9 against 17.5 us).
    if (p.width <= 256) return launch_norm<T, 1, 1, 8>(backward, p, columns, st);
    switch (warps_for(p.width)) {
      case 1: return launch_norm<T, 2, 1, 8>(backward, p, columns, st);
      case 2: return launch_norm<T, 4, 1, 8>(backward, p, columns, st);
      case 4: return launch_norm<T, 8, 1, 8>(backward, p, columns, st);
      case 8: return launch_norm<T, 16, 1, 8>(backward, p, columns, st);
      case 16: return launch_norm<T, 32, 1, 8>(backward, p, columns, st);
      default: return launch_norm<T, 32, 1, 16>(backward, p, columns, st);
    }
  } else {
    switch (warps_for(p.width)) {
      case 1:
        // narrow rows: only as many chunks as the width needs (a decoder row of 256 is half of 512)
        if (p.width <= 32 * kEpt / 2) return launch_norm<T, 1, VEC, K / 2>(backward, p, columns, st);
        return launch_norm<T, 1, VEC, K>(backward, p, columns, st);
      case 2: return launch_norm<T, 2, VEC, K>(backward, p, columns, st);
      case 4: return launch_norm<T, 4, VEC, K>(backward, p, columns, st);
      case 8: return launch_norm<T, 8, VEC, K>(backward, p, columns, st);
      case 16: return launch_norm<T, 16, VEC, K>(backward, p, columns, st);
      default: return launch_norm<T, 32, VEC, K>(backward, p, columns, st);
    }
  }
}

bool vector_rows(const void* p, int64_t ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0;
}

template <typename T>
int dispatch_vector(bool backward, NormParams& p, int64_t columns, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = p.width % VEC == 0 && vector_rows(p.x, p.x_ld, sizeof(T)) && vector_rows(p.y, p.y_ld, sizeof(T)) &&
                   vector_rows(p.dy, p.dy_ld, sizeof(T)) && vector_rows(p.weight, 0, 4) && vector_rows(p.bias, 0, 4);
  return vec ? dispatch_width<T, VEC>(backward, p, columns, st) : dispatch_width<T, 1>(backward, p, columns, st);
}

int dispatch_type(bool backward, int dtype, NormParams& p, int64_t columns, cudaStream_t st) {
  switch (dtype) {
    case S4D_DTYPE_F32: return dispatch_vector<float>(backward, p, columns, st);
    case S4D_DTYPE_BF16: return dispatch_vector<__nv_bfloat16>(backward, p, columns, st);
    default: return dispatch_vector<__half>(backward, p, columns, st);
  }
}

int type_size(int dtype) { return dtype == S4D_DTYPE_F32 ? 4 : 2; }

bool aligned_to(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(size) == 0; }

// The checks both directions share (fn names the entry point).
int check_norm(const char* fn, int dtype, int param_dtype, int64_t rows, int64_t width, int64_t ld_a, int64_t ld_b,
               int64_t ld_out) {
  if (dtype != S4D_DTYPE_F32 && dtype != S4D_DTYPE_BF16 && dtype != S4D_DTYPE_F16) {
    set_error("%s: unknown dtype", fn);
    return S4D_ERR_INVALID_ARG;
  }
  if (param_dtype != S4D_DTYPE_F32 && param_dtype != dtype) {
    set_error("%s: weight and bias must be f32 or of the input's dtype", fn);
    return S4D_ERR_INVALID_ARG;
  }
  if (rows < 0 || width <= 0) {
    set_error("%s: rows must be >= 0 and width >= 1", fn);
    return S4D_ERR_INVALID_ARG;
  }
  if (width > kNormMaxWidth) {
    set_error("%s: width must be <= %d", fn, kNormMaxWidth);
    return S4D_ERR_UNSUPPORTED_SHAPE;
  }
  int64_t span = 0;
  if (ld_a < 0 || ld_b < 0 || (rows > 1 && ld_out < width)) {
    set_error("%s: row strides must be >= 0, the output's >= width", fn);
    return S4D_ERR_INVALID_ARG;
  }
  if (rows > 0x7fffffff || !size_product({rows, ld_a}, int64_t(1) << 46, &span) ||
      !size_product({rows, ld_b}, int64_t(1) << 46, &span) || !size_product({rows, ld_out}, int64_t(1) << 46, &span)) {
    set_error("%s: too many rows or elements", fn);
    return S4D_ERR_UNSUPPORTED_SHAPE;
  }
  return S4D_OK;
}

}  // namespace
}  // namespace s4d

using namespace s4d;

extern "C" {

int s4d_norm_forward(const void* x, int64_t x_ld, int dtype, const void* weight, const void* bias, int param_dtype,
                     void* y, int64_t y_ld, float* mean, float* rstd, int64_t rows, int64_t width, float eps,
                     void* stream) {
  set_error("%s", "");
  const int st = check_norm("s4d_norm_forward", dtype, param_dtype, rows, width, x_ld, 0, y_ld);
  if (st != S4D_OK) return st;
  if (!(eps >= 0.0f)) return fail(S4D_ERR_INVALID_ARG, "s4d_norm_forward: eps must be >= 0");
  if (rows == 0) return S4D_OK;
  if (x == nullptr || y == nullptr) return fail(S4D_ERR_INVALID_ARG, "s4d_norm_forward: null pointer");
  if ((mean == nullptr) != (rstd == nullptr))
    return fail(S4D_ERR_INVALID_ARG, "s4d_norm_forward: mean and rstd go together");
  const int size = type_size(dtype), psize = type_size(param_dtype);
  if (!aligned_to(x, size) || !aligned_to(y, size) || !aligned_to(weight, psize) || !aligned_to(bias, psize) ||
      !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return fail(S4D_ERR_INVALID_ARG, "s4d_norm_forward: misaligned pointer");
  NormParams p{};
  p.x = x, p.x_ld = x_ld, p.weight = weight, p.bias = bias, p.y = y, p.y_ld = y_ld;
  p.mean = mean, p.rstd = rstd, p.rows = rows, p.width = int(width), p.eps = eps;
  p.param_f32 = param_dtype == S4D_DTYPE_F32;
  return dispatch_type(false, dtype, p, 0, static_cast<cudaStream_t>(stream));
}

size_t s4d_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0 || width > kNormMaxWidth || rows > 0x7fffffff || sums_in_one_launch(rows, width)) return 0;
  return size_t(most_row_blocks(rows, width)) * 2 * size_t(width) * sizeof(float);
}

int s4d_norm_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype, const void* weight,
                      int param_dtype, const float* mean, const float* rstd, void* dx, int64_t dx_ld, void* dweight,
                      void* dbias, int64_t rows, int64_t width, void* workspace, size_t workspace_bytes, void* stream) {
  set_error("%s", "");
  int st = check_norm("s4d_norm_backward", dtype, param_dtype, rows, width, x_ld, dy_ld, dx == nullptr ? width : dx_ld);
  if (st != S4D_OK) return st;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (rows > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr))
    return fail(S4D_ERR_INVALID_ARG, "s4d_norm_backward: null pointer");
  const int size = type_size(dtype), psize = type_size(param_dtype);
  if (!aligned_to(dy, size) || !aligned_to(x, size) || !aligned_to(dx, size) || !aligned_to(weight, psize) ||
      !aligned_to(dweight, psize) || !aligned_to(dbias, psize) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return fail(S4D_ERR_INVALID_ARG, "s4d_norm_backward: misaligned pointer");
  int blocks = 0;  // partial rows
  const bool one = sums_in_one_launch(rows, width);
  if (sums && rows > 0 && !one &&
      (workspace == nullptr || !aligned_to(workspace, 16) ||
       workspace_bytes < s4d_norm_backward_workspace_bytes(rows, width)))
    return fail(S4D_ERR_INVALID_ARG, "s4d_norm_backward: missing, misaligned or small workspace");
  cudaStream_t stm = static_cast<cudaStream_t>(stream);
  if (rows > 0 && (sums || dx != nullptr)) {
    NormParams p{};
    p.x = x, p.x_ld = x_ld, p.dy = dy, p.dy_ld = dy_ld, p.weight = weight, p.y = dx, p.y_ld = dx == nullptr ? 0 : dx_ld;
    p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd), p.rows = rows, p.width = int(width);
    p.param_f32 = param_dtype == S4D_DTYPE_F32;
    p.partial = sums && !one ? static_cast<float*>(workspace) : nullptr;
    p.dweight = dweight, p.dbias = dbias;
    st = dispatch_type(true, dtype, p, sums && one ? (width + 7) / 8 : 0, stm);
    if (st != S4D_OK) return st;
    blocks = p.row_blocks;
  }
  if (!sums || (one && rows > 0)) return S4D_OK;
  const dim3 grid(unsigned((width + 31) / 32), 2);
  const float* partial = static_cast<const float*>(workspace);
  cudaError_t e;
  if (param_dtype == S4D_DTYPE_F32)
    e = launch_pdl(blocks > 0, norm_reduce_kernel<float>, grid, dim3(1024), 0, stm, partial, blocks, int(width),
                   static_cast<float*>(dweight), static_cast<float*>(dbias));
  else if (param_dtype == S4D_DTYPE_BF16)
    e = launch_pdl(blocks > 0, norm_reduce_kernel<__nv_bfloat16>, grid, dim3(1024), 0, stm, partial, blocks,
                   int(width), static_cast<__nv_bfloat16*>(dweight), static_cast<__nv_bfloat16*>(dbias));
  else
    e = launch_pdl(blocks > 0, norm_reduce_kernel<__half>, grid, dim3(1024), 0, stm, partial, blocks, int(width),
                   static_cast<__half*>(dweight), static_cast<__half*>(dbias));
  return cuda_check(e, "norm_reduce_kernel launch");
}

}  // extern "C"
