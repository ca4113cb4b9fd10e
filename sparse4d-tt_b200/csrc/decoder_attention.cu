// extern "C" entry points of the decoder's attention (include/s4d_decoder.h): argument validation on
// the host, tensor maps and the choice of launches.
#include <cmath>
#include <mutex>

#include "decoder_attention.cuh"

namespace s4d {

unsigned long long decoder_wait_limit_ns();  // decoder_capi.cu

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}

bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Strides of [batch, rows, heads] for addressing: those of an axis with one entry (or none) are 0.
struct Strides {
  int64_t b, n, h;
  Strides(const int64_t* s, int64_t batch, int64_t rows, int64_t heads)
      : b(batch > 1 ? s[0] : 0), n(rows > 1 ? s[1] : 0), h(heads > 1 ? s[2] : 0) {}
  // Positive multiples of 8 elements below 2^37 where the axis has more than one entry, and an extent
  // that stays below 2^46 elements.
  bool ok(int64_t batch, int64_t rows, int64_t heads) const {
    const int64_t st[3] = {b, n, h}, ext[3] = {batch, rows, heads};
    for (int i = 0; i < 3; ++i) {
      int64_t span = 0;
      if (ext[i] > 1 && (st[i] <= 0 || st[i] % 8 != 0 || st[i] >= (int64_t(1) << 37) ||
                         !size_product({ext[i], st[i]}, int64_t(1) << 46, &span)))
        return false;
    }
    return true;
  }
};

// Tensor map of [B, N, heads, D] 16-bit elements, loaded in boxes of 64 columns x box_heads heads x box_rows
// rows with the 128-byte swizzle; columns past D and rows past N are zero.
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t dim, int64_t heads, int64_t rows, int64_t batch,
             const Strides& s, int box_rows, int box_heads = 1) {
  EncodeTiledFn fn = encode_tiled();
  if (fn == nullptr) return fail(S4D_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the CUDA driver");
  // an axis of one entry still needs a stride the encoder takes
  const int64_t row_bytes = dim * 2 >= 16 ? (dim * 2 + 15) / 16 * 16 : 16;
  const cuuint64_t dims[4] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(rows), cuuint64_t(batch)};
  const cuuint64_t strides[3] = {cuuint64_t(s.h > 0 ? s.h * 2 : row_bytes), cuuint64_t(s.n > 0 ? s.n * 2 : row_bytes),
                                 cuuint64_t(s.b > 0 ? s.b * 2 : row_bytes)};
  const cuuint32_t box[4] = {64, cuuint32_t(box_heads), cuuint32_t(box_rows), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(map, dtype == S4D_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (CUresult %d) for [%lld, %lld, %lld, %lld]", int(r), (long long)batch,
              (long long)rows, (long long)heads, (long long)dim);
    return S4D_ERR_CUDA;
  }
  return S4D_OK;
}

constexpr int64_t kMaxRows = int64_t(1) << 31;
constexpr float kMaxSoftcap = 1024.0f;
constexpr int kKeyTile = 64;       // keys of a forward tile
constexpr int kBackwardTile = 64;  // queries or keys of a backward tile

// Checks of sizes and of the arguments that forward and backward share; fn names the entry point.
int check_args(const char* fn, const s4d_attention_args* a) {
#define S4D_BAD(status, text)         \
  do {                                \
    set_error("%s: %s", fn, text);    \
    return status;                    \
  } while (0)
  if (a == nullptr) S4D_BAD(S4D_ERR_INVALID_ARG, "null args");
  if (a->dtype != S4D_DTYPE_BF16 && a->dtype != S4D_DTYPE_F16) S4D_BAD(S4D_ERR_INVALID_ARG, "dtype must be bf16 or f16");
  if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads <= 0 || a->kv_heads <= 0)
    S4D_BAD(S4D_ERR_INVALID_ARG, "bad sizes");
  if (a->heads % a->kv_heads != 0) S4D_BAD(S4D_ERR_INVALID_ARG, "heads must be a multiple of kv_heads");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8 != 0)
    S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "dim must be a multiple of 8 from 8 to 128");
  if (a->pos_dim < 0 || a->pos_dim > 2) S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "pos_dim must be 0, 1 or 2");
  if (!(a->scale > -INFINITY && a->scale < INFINITY)) S4D_BAD(S4D_ERR_INVALID_ARG, "scale must be finite");
  // a capped score is cap - cap * (1 - tanh), off by a few 2^-23 cap: above the limit that is no longer small
  // beside the rounding of the weights to 16 bits
  if (!(a->softcap >= 0.0f && a->softcap <= kMaxSoftcap))
    S4D_BAD(S4D_ERR_INVALID_ARG, "softcap must be 0 (none) or at most 1024");
  if (!std::isfinite(ScoreConst(a->scale, a->softcap).k1))
    S4D_BAD(S4D_ERR_INVALID_ARG, "scale, or scale / softcap, is too large for fp32");
  int64_t n = 0;
  if (!size_product({a->queries, a->heads / a->kv_heads}, kMaxRows, &n) || a->keys >= kMaxRows ||
      a->batch >= kMaxRows || a->heads >= (1 << 20) ||
      !size_product({a->batch, a->queries, a->heads, a->dim}, int64_t(1) << 46, &n) ||
      !size_product({a->batch, a->keys, a->kv_heads, a->dim}, int64_t(1) << 46, &n))
    S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "too many rows or elements");
  if ((a->q_segment == nullptr) != (a->k_segment == nullptr))
    S4D_BAD(S4D_ERR_INVALID_ARG, "q_segment and k_segment go together");
  if (a->batch == 0) return S4D_OK;
  if (!aligned_to(a->q, 16) || !aligned_to(a->k, 16) || !aligned_to(a->v, 16) || !aligned_to(a->out, 16) ||
      !aligned_to(a->lse, 4) || !aligned_to(a->slopes, 4) || !aligned_to(a->q_pos, 4) || !aligned_to(a->k_pos, 4) ||
      !aligned_to(a->q_segment, 4) || !aligned_to(a->k_segment, 4) || !aligned_to(a->k_len, 4) ||
      !aligned_to(a->error_flag, 4))
    S4D_BAD(S4D_ERR_INVALID_ARG, "misaligned pointer");
  if (a->queries > 0 && (a->q == nullptr || a->out == nullptr)) S4D_BAD(S4D_ERR_INVALID_ARG, "null q or out");
  if (a->keys > 0 && (a->k == nullptr || a->v == nullptr)) S4D_BAD(S4D_ERR_INVALID_ARG, "null k or v");
  if (a->pos_dim > 0 && ((a->queries > 0 && (a->q_pos == nullptr || a->slopes == nullptr)) ||
                         (a->keys > 0 && a->k_pos == nullptr)))
    S4D_BAD(S4D_ERR_INVALID_ARG, "null slopes or positions");
  if (!Strides(a->q_stride, a->batch, a->queries, a->heads).ok(a->batch, a->queries, a->heads) ||
      !Strides(a->k_stride, a->batch, a->keys, a->kv_heads).ok(a->batch, a->keys, a->kv_heads) ||
      !Strides(a->v_stride, a->batch, a->keys, a->kv_heads).ok(a->batch, a->keys, a->kv_heads))
    S4D_BAD(S4D_ERR_INVALID_ARG, "strides of q, k and v must be positive multiples of 8 elements");
  return S4D_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Parts of the keys.  A tile of 128 rows and one shared head is one CTA.  With fewer CTAs than SMs the keys
// are cut until every SM has one, or two when with one a part has 16 tiles of 64 keys or more: the two on
// an SM keep more loads under way, but each of its tiles takes longer, and more parts take longer to join.
// (Graph times: 2 x 16 queries over 30,000 keys, 2 heads of 64 29.4 us with one CTA an SM, 36.2 with two; one
// query over 4 x 65,536 keys, 32 heads of 128 on 8, 1-D distance 268 us with one, 178 with two.)  A part is not
// cut below two tiles, one for each stream of row warps.  Up to 11 parts become at most 8, which
// one cluster joins in shared memory: a second launch and its pass over memory cost more than a quarter
// of the CTAs brings.
int64_t key_splits(const s4d_attention_args& a) {
  const int64_t ctas = a.batch * a.kv_heads * ceil_div(a.queries * (a.heads / a.kv_heads), kAttnRows);
  const int64_t tiles = ceil_div(a.keys, kKeyTile), sms = device_sms();
  const int64_t least = ceil_div(tiles, kAttnMaxTiles);
  if (ctas == 0 || tiles == 0) return 1;
  int64_t splits = sms / ctas > 1 ? sms / ctas : 1;
  if (tiles / splits >= 16 && 2 * sms / ctas > splits) splits = 2 * sms / ctas;
  if (splits > tiles / 2) splits = tiles / 2;
  if (splits > 8 && splits < 12) splits = 8;
  if (splits < least) splits = least;
  if (splits < 1) splits = 1;
  // as many parts as there are after each got the same number of tiles
  return ceil_div(tiles, ceil_div(tiles, splits));
}

int cluster_of(int64_t splits) { return splits <= 8 ? int(splits) : 1; }

size_t forward_workspace(const s4d_attention_args& a) {
  const int64_t splits = key_splits(a);
  return splits == cluster_of(splits) ? 0 : size_t(splits) * size_t(a.batch * a.queries * a.heads) * size_t(a.dim + 1) * sizeof(float);
}

AttnParams fill(const s4d_attention_args& a) {
  AttnParams p{};
  const Strides q(a.q_stride, a.batch, a.queries, a.heads);
  p.q = a.q, p.q_sb = q.b, p.q_sn = q.n, p.q_sh = q.h;
  const Strides v(a.v_stride, a.batch, a.keys, a.kv_heads);
  p.v = a.v, p.v_sb = v.b, p.v_sn = v.n, p.v_sh = v.h;
  p.out = a.out, p.lse = a.lse;
  p.slopes = a.slopes, p.sl_b = a.slope_stride[0], p.sl_n = a.slope_stride[1], p.sl_h = a.slope_stride[2];
  p.q_pos = a.q_pos, p.k_pos = a.k_pos, p.q_seg = a.q_segment, p.k_seg = a.k_segment, p.k_len = a.k_len;
  p.nq = a.queries, p.nk = a.keys;
  p.batch = int(a.batch), p.heads = int(a.heads), p.kv_heads = int(a.kv_heads), p.rep = int(a.heads / a.kv_heads);
  p.dim = int(a.dim), p.scale = a.scale, p.cap = a.softcap;
  p.error_flag = a.error_flag;
  p.wait_limit_ns = decoder_wait_limit_ns();
  return p;
}

// A map of k or v; without keys one of q's memory, which no kernel then reads.
int key_map(CUtensorMap* map, const s4d_attention_args& a, const void* base, const int64_t* stride, int box_rows) {
  if (a.keys == 0) return make_map(map, a.q, a.dtype, a.dim, 1, 1, 1, Strides(stride, 1, 1, 1), box_rows);
  return make_map(map, base, a.dtype, a.dim, a.kv_heads, a.keys, a.batch, Strides(stride, a.batch, a.keys, a.kv_heads),
                  box_rows);
}

// A map of q or dout; without queries one of k's memory, which no kernel then reads.
int query_map(CUtensorMap* map, const s4d_attention_args& a, const void* base, const int64_t* stride, int box_rows,
              int box_heads = 1) {
  if (a.queries == 0) return make_map(map, a.k, a.dtype, a.dim, 1, 1, 1, Strides(stride, 1, 1, 1), box_rows);
  return make_map(map, base, a.dtype, a.dim, a.heads, a.queries, a.batch, Strides(stride, a.batch, a.queries, a.heads),
                  box_rows, box_heads);
}

// dslopes of one slope per head: the sum of every row's ([B, H, Nq]), one head a block, its rows added
// in an order that depends on the sizes alone.
__global__ void __launch_bounds__(1024) slope_sum_kernel(const float* rows, int batch, int64_t nq, int heads, float* out) {
  __shared__ float part[32];
  const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float s[8] = {};
  griddep_wait();
  for (int b = 0; b < batch; ++b) {
    const float* src = rows + (int64_t(b) * heads + h) * nq;
    for (int64_t r = threadIdx.x; r < nq; r += 8 * 1024)
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r + u * 1024 < nq) s[u] += src[r + u * 1024];
  }
  float v = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0f;
    for (int w = 0; w < 32; ++w) v += part[w];
    out[h] = v;
  }
}

int launch_slope_sum(const float* rows, const s4d_attention_args& a, cudaStream_t st) {
  return cuda_check(launch_pdl(true, slope_sum_kernel, dim3(unsigned(a.heads)), dim3(1024), 0, st, rows, int(a.batch),
                               a.queries, int(a.heads), a.dslopes),
                    "slope_sum_kernel launch");
}

size_t backward_workspace(const s4d_attention_args& a) {
  const size_t rows = size_t(a.batch) * size_t(a.heads);
  const bool sum = a.dslopes != nullptr && !a.dslopes_per_row;
  return rows * size_t(ceil_div(a.queries, kRecordTile)) * kRecordBytes + (sum ? rows * size_t(a.queries) * sizeof(float) : 0);
}

}  // namespace
}  // namespace s4d

using namespace s4d;

extern "C" {

size_t s4d_attention_forward_workspace_bytes(const s4d_attention_args* args) {
  if (args == nullptr || args->batch <= 0 || args->queries <= 0 || args->keys < 0 || args->heads <= 0 ||
      args->kv_heads <= 0 || args->heads % args->kv_heads != 0 || args->dim <= 0 || args->dim > 128)
    return 0;
  int64_t n = 0;
  if (!size_product({args->batch, args->queries, args->heads, args->dim}, int64_t(1) << 46, &n) || args->keys >= kMaxRows)
    return 0;
  return forward_workspace(*args);
}

int s4d_attention_forward(const s4d_attention_args* args, void* stream) {
  const char* fn = "s4d_attention_forward";
  set_error("%s", "");
  int st = check_args(fn, args);
  if (st != S4D_OK) return st;
  const s4d_attention_args& a = *args;
  if (a.batch == 0 || a.queries == 0) return S4D_OK;
  AttnParams p = fill(a);
  const int64_t splits = key_splits(a), tiles = ceil_div(a.keys, kKeyTile);
  int64_t ctas = 0;
  if (!size_product({a.batch, a.kv_heads, ceil_div(a.queries * p.rep, kAttnRows), splits}, kMaxRows, &ctas) ||
      ceil_div(a.batch * a.queries * a.heads, 8) >= kMaxRows)
    S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "too many row tiles");
  const size_t need = forward_workspace(a);
  if (need > 0 && (a.workspace == nullptr || !aligned_to(a.workspace, 16) || a.workspace_bytes < need))
    S4D_BAD(S4D_ERR_INVALID_ARG, "missing, misaligned or small workspace");
  p.splits = int(splits);
  p.cluster = cluster_of(splits);
  p.tiles_per_split = tiles > 0 ? ceil_div(tiles, splits) : 0;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_lse = p.part_o + (need > 0 ? splits * a.batch * a.queries * a.heads * a.dim : 0);
  AttnForwardMaps m;
  st = key_map(&m.k, a, a.k, a.k_stride, kKeyTile);
  if (st == S4D_OK) st = key_map(&m.v, a, a.v, a.v_stride, kKeyTile);
  // a box of 128 / rep queries of all the heads that share keys (the kernel gathers Q itself for a rep
  // that does not divide 128: the map is then not used)
  const bool whole = kAttnRows % p.rep == 0;
  if (st == S4D_OK)
    st = query_map(&m.q, a, a.q, a.q_stride, whole ? kAttnRows / p.rep : 1, whole ? p.rep : 1);
  if (st != S4D_OK) return st;
  cudaStream_t stm = static_cast<cudaStream_t>(stream);
  return a.dim <= 64 ? launch_attention_forward_d64(a.dtype, int(a.pos_dim), p, m, stm)
                     : launch_attention_forward_d128(a.dtype, int(a.pos_dim), p, m, stm);
}

size_t s4d_attention_backward_workspace_bytes(const s4d_attention_args* args) {
  int64_t n = 0;
  if (args == nullptr || args->batch <= 0 || args->queries <= 0 || args->heads <= 0 ||
      !size_product({args->batch, args->queries, args->heads}, int64_t(1) << 46, &n))
    return 0;
  return backward_workspace(*args);
}

int s4d_attention_backward(const s4d_attention_args* args, void* stream) {
  const char* fn = "s4d_attention_backward";
  set_error("%s", "");
  int st = check_args(fn, args);
  if (st != S4D_OK) return st;
  const s4d_attention_args& a = *args;
  if (a.dtype != S4D_DTYPE_BF16) S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "implemented for bf16");
  if (ceil_div(a.queries, kBackwardTile) > kAttnMaxTiles || ceil_div(a.keys, kBackwardTile) > kAttnMaxTiles)
    S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "implemented for at most 524288 queries and keys");
  const bool sum = a.dslopes != nullptr && !a.dslopes_per_row;
  cudaStream_t stm = static_cast<cudaStream_t>(stream);
  if (a.dslopes != nullptr && a.pos_dim == 0) S4D_BAD(S4D_ERR_INVALID_ARG, "dslopes without a distance bias");
  if (!aligned_to(a.dslopes, 4)) S4D_BAD(S4D_ERR_INVALID_ARG, "misaligned pointer");
  if (a.batch == 0) return sum ? launch_slope_sum(nullptr, a, stm) : S4D_OK;  // zeros
  if ((a.dk == nullptr) != (a.dv == nullptr)) S4D_BAD(S4D_ERR_INVALID_ARG, "dk and dv go together");
  if (!aligned_to(a.dout, 16) || !aligned_to(a.dq, 16) || !aligned_to(a.dk, 16) || !aligned_to(a.dv, 16))
    S4D_BAD(S4D_ERR_INVALID_ARG, "misaligned pointer");
  if (a.queries > 0 && (a.dout == nullptr || a.dq == nullptr || a.lse == nullptr))
    S4D_BAD(S4D_ERR_INVALID_ARG, "null dout, dq or lse");
  if (!Strides(a.dout_stride, a.batch, a.queries, a.heads).ok(a.batch, a.queries, a.heads))
    S4D_BAD(S4D_ERR_INVALID_ARG, "strides of dout must be positive multiples of 8 elements");
  const size_t need = backward_workspace(a);
  if (a.queries > 0 && (a.workspace == nullptr || !aligned_to(a.workspace, 16) || a.workspace_bytes < need))
    S4D_BAD(S4D_ERR_INVALID_ARG, "missing, misaligned or small workspace");
  AttnParams p = fill(a);
  int64_t ctas = 0;
  if (!size_product({a.batch, a.kv_heads, ceil_div(a.queries * p.rep, kAttnRows)}, kMaxRows, &ctas) ||
      !size_product({a.batch, a.kv_heads, ceil_div(a.keys, kAttnRows)}, kMaxRows, &ctas))
    S4D_BAD(S4D_ERR_UNSUPPORTED_SHAPE, "too many row tiles");
  const Strides d(a.dout_stride, a.batch, a.queries, a.heads);
  p.dout = a.dout, p.do_sb = d.b, p.do_sn = d.n, p.do_sh = d.h;
  p.dq = a.dq, p.dk = a.dk, p.dv = a.dv;
  p.splits = 1;
  p.records = static_cast<float*>(a.workspace);
  p.dslopes = sum ? p.records + a.batch * a.heads * ceil_div(a.queries, kRecordTile) * (kRecordBytes / 4) : a.dslopes;
  p.dslopes_by_head = sum;
  if (a.queries > 0 || a.keys > 0) {
    AttnBackwardMaps m;
    st = key_map(&m.k_tile, a, a.k, a.k_stride, kBackwardTile);
    if (st == S4D_OK) st = key_map(&m.v_tile, a, a.v, a.v_stride, kBackwardTile);
    if (st == S4D_OK) st = key_map(&m.k_rows, a, a.k, a.k_stride, kAttnRows);
    if (st == S4D_OK) st = key_map(&m.v_rows, a, a.v, a.v_stride, kAttnRows);
    if (st == S4D_OK) st = query_map(&m.q_tile, a, a.q, a.q_stride, kBackwardTile);
    if (st == S4D_OK) st = query_map(&m.do_tile, a, a.dout, a.dout_stride, kBackwardTile);
    // as in the forward pass: not used for a rep that does not divide 128
    const bool whole = kAttnRows % p.rep == 0;
    const int own_rows = whole ? kAttnRows / p.rep : 1, own_heads = whole ? p.rep : 1;
    if (st == S4D_OK) st = query_map(&m.q_rows, a, a.q, a.q_stride, own_rows, own_heads);
    if (st == S4D_OK) st = query_map(&m.do_rows, a, a.dout, a.dout_stride, own_rows, own_heads);
    if (st == S4D_OK)
      st = a.dim <= 64 ? launch_attention_backward_d64(int(a.pos_dim), p, m, stm)
                       : launch_attention_backward_d128(int(a.pos_dim), p, m, stm);
    if (st != S4D_OK) return st;
  }
  return sum ? launch_slope_sum(p.dslopes, a, stm) : S4D_OK;
}

}  // extern "C"
