// layer.cu -- what a layer does around its attention block: ca_rms_norm,
// ca_linear_q8, ca_gated_linear (include/canvas_attn.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "canvas_attn.h"
#include "host_util.cuh"
#include "rows.cuh"
#include "pair.cuh"
#include "skinny.cuh"

namespace ca {

int layer_device_error() {
  int e = 0;
  if (cudaMemcpyFromSymbol(&e, g_device_error, sizeof(int)) != cudaSuccess) return CA_ERR_CUDA;
  if (e != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  }
  return e;
}

namespace {

int type_size(int t) {
  return t == CA_TYPE_BF16 ? 2 : t == CA_TYPE_F32 ? 4 : t == CA_TYPE_E4M3 ? 1 : 0;
}

bool aligned_to(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) == 0;
}

template <bool XF32, int RES, int OUT>
int launch_rows(const RowsParams& p, cudaStream_t st) {
  const int chunks = p.cols / 8;
  auto threads = [&](int c) { return ((chunks + c - 1) / c + 31) / 32 * 32; };
  auto grid = [&](int threads) {
    return dim3(static_cast<unsigned>(
        std::min<int64_t>(p.rows, static_cast<int64_t>(kSms) * std::min(32, 1024 / threads))));
  };
  // A chunk a thread where rows are few (the shortest way through one: 888 rows
  // of 4096 in bf16 6.5 us, two chunks 7.1; 1184 rows 8.1 and 7.2) and where a
  // chunk of fp32 takes twice the registers (2000 rows of 3584 12.8 us, two
  // chunks 15.3).
  if (chunks <= 1024 && (p.rows <= 6 * kSms || XF32 || RES == 2 || chunks <= 64)) {
    const int t = threads(1);
    return launch_after(rows_kernel<XF32, RES, OUT, 1>, grid(t), t, 0, st, p);
  }
  if constexpr (!XF32 && RES != 2) {
    if (chunks <= 1024) {
      const int t = threads(2);
      return launch_after(rows_kernel<XF32, RES, OUT, 2>, grid(t), t, 0, st, p);
    }
  }
  if (chunks <= 1536) {
    const int t = threads(3);
    return launch_after(rows_kernel<XF32, RES, OUT, 3>, grid(t), t, 0, st, p);
  }
  const int t = threads(5);
  return launch_after(rows_kernel<XF32, RES, OUT, 5>, grid(t), t, 0, st, p);
}

template <bool XF32, int RES>
int launch_rows_out(const RowsParams& p, cudaStream_t st) {
  if (p.out_type == kOutE4m3) return launch_rows<XF32, RES, kOutE4m3>(p, st);
  if (p.out_type == kOutF32) return launch_rows<XF32, RES, kOutF32>(p, st);
  return launch_rows<XF32, RES, kOutBf16>(p, st);
}

template <bool XF32>
int launch_rows_res(const RowsParams& p, cudaStream_t st) {
  if (!p.res) return launch_rows_out<XF32, 0>(p, st);
  return p.res_f32 ? launch_rows_out<XF32, 2>(p, st) : launch_rows_out<XF32, 1>(p, st);
}

int rms_norm_impl(const ca_rms_norm_args* a, cudaStream_t st) {
  if (!a || a->rows < 0 || a->cols <= 0) return CA_ERR_INVALID;
  // No rows: there is nothing that a pointer could point to.
  if (a->rows > 0 && (!a->x || !a->out)) return CA_ERR_INVALID;
  if (a->x_type != CA_TYPE_BF16 && a->x_type != CA_TYPE_F32) return CA_ERR_INVALID;
  if (type_size(a->out_type) == 0) return CA_ERR_INVALID;
  if (a->rows == 0) return CA_OK;
  if (a->residual && ((a->residual_type != CA_TYPE_BF16 && a->residual_type != CA_TYPE_F32) ||
                      !a->sum_out))
    return CA_ERR_INVALID;
  if (!a->residual && a->sum_out) return CA_ERR_INVALID;
  if (a->out_type == CA_TYPE_E4M3 && !a->out_scale) return CA_ERR_INVALID;
  if (a->norm && !(a->eps >= 0.f)) return CA_ERR_INVALID;
  RowsParams p{};
  auto stride = [&](int64_t s) { return s ? s : a->cols; };
  p.x_stride = stride(a->x_stride);
  p.res_stride = stride(a->residual_stride);
  p.sum_stride = stride(a->sum_stride);
  p.out_stride = stride(a->out_stride);
  if (p.x_stride < a->cols || p.res_stride < a->cols || p.sum_stride < a->cols ||
      p.out_stride < a->cols)
    return CA_ERR_INVALID;
  const int xs = type_size(a->x_type), os = type_size(a->out_type);
  const int rs = a->residual ? type_size(a->residual_type) : 4;
  if (!aligned_to(a->x, xs) || !aligned_to(a->out, os) || !aligned_to(a->w, 4) ||
      !aligned_to(a->residual, rs) || !aligned_to(a->sum_out, rs) || !aligned_to(a->out_scale, 4))
    return CA_ERR_INVALID;
  if (a->cols > INT_MAX - 1024) return CA_ERR_UNSUPPORTED;
  p.x = a->x;
  p.res = a->residual;
  p.sum = a->sum_out;
  p.w = a->w;
  p.out = a->out;
  p.out_scale = a->out_type == CA_TYPE_E4M3 ? a->out_scale : nullptr;
  p.rows = a->rows;
  p.cols = static_cast<int>(a->cols);
  p.x_f32 = a->x_type == CA_TYPE_F32;
  p.res_f32 = a->residual_type == CA_TYPE_F32;
  p.out_type = a->out_type;
  p.norm = a->norm ? 1 : 0;
  p.eps = a->eps;
  auto rows16 = [](const void* q, int64_t bytes) { return !q || (aligned16(q) && bytes % 16 == 0); };
  const bool vec = p.cols % 8 == 0 && rows16(p.x, p.x_stride * xs) &&
                   rows16(p.res, p.res_stride * rs) && rows16(p.sum, p.sum_stride * rs) &&
                   aligned16(p.w) &&
                   (os == 1 ? aligned_to(p.out, 8) && p.out_stride % 8 == 0
                            : rows16(p.out, p.out_stride * os));
  // Registers hold 20480 columns.
  if (vec && p.cols <= 20480)
    return p.x_f32 ? launch_rows_res<true>(p, st) : launch_rows_res<false>(p, st);
  if (p.cols <= 20480) {
    auto odd = [&](auto kernel, int n) {
      const int t = ((p.cols + n - 1) / n + 31) / 32 * 32;
      const int64_t most = static_cast<int64_t>(kSms) * std::min(32, std::max(1, (n == 4 ? 2048 : 1024) / t));
      return launch_after(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, most))), t,
                          0, st, p);
    };
    if (p.cols <= 4096) return odd(rows_odd_kernel<4>, 4);
    if (p.cols <= 8192) return odd(rows_odd_kernel<8>, 8);
    return odd(rows_odd_kernel<20>, 20);
  }
  return launch_after(rows_any_kernel,
                      dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, 4 * kSms))), 256, 0, st,
                      p);
}

// A row-major matrix of 1- or 2-byte elements in boxes of 128 bytes of
// box_rows rows, 128-byte swizzle; what lies outside reads as zero.
int make_tmap_2d(CUtensorMap* m, const void* base, int kind, int64_t cols, int64_t rows,
                 int64_t stride, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return CA_ERR_CUDA;
  const int es = kind == kKindBf16 ? 2 : 1;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * es};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), box_rows};
  cuuint32_t elem[2] = {1, 1};
  const CUresult r =
      fn(m, kind == kKindBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
         const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CA_OK : CA_ERR_INVALID;
}

// A product as both entry points ask for it.
struct Product {
  const void* act;
  const void* w;
  const void* up;  // gated: the second matrix
  int64_t act_stride, cols;
  LinearParams p;
};

// How many pieces of 128 bytes of the columns (four additions each) an
// accumulator takes where the output is fp32, see pair.cuh: 1024 columns of
// bf16, 4096 of e4m3, whose products have eight bits and leave less to cut off
// (sums of one sign over 4096 columns 5e-7 off in 2-norm, over 18944 9e-6).
constexpr int pieces_of_an_accumulator(int kind) { return kind == kKindBf16 ? 16 : 32; }

// tiles x tok tiles of 128 rows by NT tokens, each by a cluster of S CTAs.
template <class C>
int launch_skinny_as(const Product& q, int64_t tiles, int64_t tok, int S, cudaStream_t st) {
  constexpr int KIND = C::KIND, G = C::G, NT = C::NT;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CA_ERR_CUDA;
  CUtensorMap tw, tu, tx;
  int rc;
  if ((rc = make_tmap_2d(&tw, q.w, KIND, q.cols, q.p.rows, q.cols, 128)) != CA_OK) return rc;
  tu = tw;
  if (G == 2 && (rc = make_tmap_2d(&tu, q.up, KIND, q.cols, q.p.rows, q.cols, 128)) != CA_OK)
    return rc;
  if ((rc = make_tmap_2d(&tx, q.act, KIND, q.cols, q.p.n, q.act_stride, NT)) != CA_OK) return rc;
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(skinny_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::kSmem) != cudaSuccess)
      return CA_ERR_CUDA;
    attr_done[dev] = true;
  }
  return launch_cluster_after(skinny_kernel<C>,
                              dim3(static_cast<unsigned>(tiles * S), static_cast<unsigned>(tok)),
                              C::kThreads, C::kSmem, S, st, tw, tu, tx, q.p);
}

template <int KIND, int G, int NT>
int launch_skinny(const Product& q, cudaStream_t st) {
  const int64_t tiles = (q.p.rows + 127) / 128, tok = (q.p.n + NT - 1) / NT;
  if (tiles > INT_MAX / 8 || tok > 65535) return CA_ERR_UNSUPPORTED;
  // Columns are split until there is a CTA for each SM, down to four pieces a
  // CTA, and once more (two fit on an SM) if that leaves twelve. One token, us at
  // 1, 2, 4 and 8 splits: 4096 x 4096 11.3, 8.1, 6.3, 7.1; 1024 x 4096 11.1, 8.0,
  // 5.9, 5.1; 12288 -> 4096 28, 16.5, 10.5, 9.9; gated 4096 -> 12288 in bf16 51,
  // 36, 40, 38.
  // fp32 outputs: few additions to an accumulator, too, which truncates
  // (pair.cuh), by more splits and, beyond eight, by more accumulators.
  constexpr int kPieces = pieces_of_an_accumulator(KIND);
  const int64_t most = q.p.out_f32 ? kPieces : INT_MAX;
  int S = 1;
  while (S < 8 && q.p.kblocks > most * S) S *= 2;
  while (S < 8 && ((tiles * tok * S * 2 <= kSms && q.p.kblocks >= 8 * S) ||
                   (tiles * tok * S * 2 <= 2 * kSms && q.p.kblocks >= 24 * S)))
    S *= 2;
  if (q.p.kblocks > most * S)
    return launch_skinny_as<SkinnyCfg<KIND, G, NT, kPieces>>(q, tiles, tok, S, st);
  return launch_skinny_as<SkinnyCfg<KIND, G, NT>>(q, tiles, tok, S, st);
}

template <int KIND, int G, int NT, int CHUNK = 0>
int launch_pair(const Product& q, cudaStream_t st) {
  using C = PairCfg<KIND, G, NT, CHUNK>;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CA_ERR_CUDA;
  CUtensorMap tw, tu, tx;
  int rc;
  const uint32_t box = G == 2 ? 64 : 128;
  if ((rc = make_tmap_2d(&tw, q.w, KIND, q.cols, q.p.rows, q.cols, box)) != CA_OK) return rc;
  tu = tw;
  if (G == 2 && (rc = make_tmap_2d(&tu, q.up, KIND, q.cols, q.p.rows, q.cols, box)) != CA_OK)
    return rc;
  if ((rc = make_tmap_2d(&tx, q.act, KIND, q.cols, q.p.n, q.act_stride, NT / 2)) != CA_OK)
    return rc;
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(pair_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::kSmem) != cudaSuccess)
      return CA_ERR_CUDA;
    attr_done[dev] = true;
  }
  LinearParams p = q.p;
  const int64_t rt = (p.rows + C::kRows - 1) / C::kRows, tt = (p.n + NT - 1) / NT;
  if (rt * tt > INT_MAX / 2) return CA_ERR_UNSUPPORTED;
  p.r_tiles = static_cast<int>(rt);
  p.t_tiles = static_cast<int>(tt);
  const int pairs = static_cast<int>(std::min<int64_t>(rt * tt, kSms / 2));
  return launch_after(pair_kernel<C>, dim3(2 * pairs), C::kThreads, C::kSmem, st, tw, tu, tx, p);
}

// Few tokens, or few enough tiles that single CTAs of 128 rows by 64 tokens get
// through them at once (two on an SM; the gated form's, which hold two matrices,
// one on every other SM) where pairs of SMs would leave some idle or pay their
// longer way for little: us, single CTAs and pairs, in e4m3: 128 tokens 4096 ->
// 4096 13.5 and 17.1, 512 tokens 16.0 and 18.1, 768 tokens (384 tiles) 28.6 and
// 21.9; 443 tokens 3584 -> 4608 14.0 and 15.9; 512 tokens 12288 -> 4096 34.9 and
// 40.0; gated in bf16 128 tokens 4096 -> 4096 20.5 and 28.1, 256 tokens (128
// tiles) 31.7 and 28.6.
template <int KIND, int G>
int launch_product(const Product& q, cudaStream_t st) {
  const int64_t tiles = (q.p.rows + 127) / 128 * ((q.p.n + 63) / 64);
  constexpr int kPieces = pieces_of_an_accumulator(KIND);
  const bool pieces = q.p.out_f32 && q.p.kblocks > kPieces;
  // Long sums of e4m3 would need more splits here than tiles leave room for (512
  // tokens 12288 -> 4096 to fp32 87 us in eight, pairs 38); bf16 tokens stay
  // (gated, 128 tokens 8192 -> 1024 23 us, pairs 58).
  if (q.p.n <= 64 || (tiles <= (G == 1 ? 2 * kSms : kSms / 2) &&
                      !(KIND == kKindE4m3 && pieces))) {
    if (q.p.n <= 16) return launch_skinny<KIND, G, 16>(q, st);
    if (q.p.n <= 32) return launch_skinny<KIND, G, 32>(q, st);
    return launch_skinny<KIND, G, 64>(q, st);
  }
  // A tile of 128 tokens takes a pair about as long as one of 256 (0.31 us a
  // piece alone: the weights' way into shared memory is the bound), so that it
  // pays only where there are no more rounds of them: 1536 tokens 4096 -> 4096 in
  // three rounds 40 us, in two of 256 tokens 30.
  const int64_t rt = (q.p.rows + 256 / G - 1) / (256 / G);
  auto rounds = [&](int64_t nt) {
    return (rt * ((q.p.n + nt - 1) / nt) + kSms / 2 - 1) / (kSms / 2);
  };
  const bool small = rounds(128) <= rounds(256);
  if constexpr (KIND == kKindE4m3) {
    if (pieces && !small) return launch_pair<KIND, G, 256, kPieces>(q, st);
  }
  if (pieces) return launch_pair<KIND, G, 128, kPieces>(q, st);
  if (small) return launch_pair<KIND, G, 128>(q, st);
  return launch_pair<KIND, G, 256>(q, st);
}

// Shapes, strides and alignment of a product; es: bytes of an operand's element.
int check_product(Product* q, int es, int out_f32) {
  LinearParams& p = q->p;
  if (!q->w || p.n < 0 || p.rows <= 0 || q->cols <= 0) return CA_ERR_INVALID;
  if (p.n > 0 && (!q->act || !p.out)) return CA_ERR_INVALID;
  if (!q->act_stride) q->act_stride = q->cols;
  if (!p.out_stride) p.out_stride = p.rows;
  if (!p.res_stride) p.res_stride = p.rows;
  if (q->act_stride < q->cols || p.out_stride < p.rows || p.res_stride < p.rows ||
      q->act_stride * es % 16 || !aligned16(q->act) || !aligned16(q->w) ||
      (q->up && !aligned16(q->up)))
    return CA_ERR_INVALID;
  const int os = out_f32 ? 4 : 2;
  if (!aligned_to(p.out, os) || !aligned_to(p.residual, os) || !aligned_to(p.act_scale, 4) ||
      !aligned_to(p.w_scale, 4) || !aligned_to(p.up_scale, 4) || !aligned_to(p.bias, 4) ||
      !aligned_to(p.err, 4))
    return CA_ERR_INVALID;
  if (q->cols * es % 16) return CA_ERR_UNSUPPORTED;
  if (p.n > INT_MAX - 256 || p.rows > INT_MAX - 256 || q->cols > INT_MAX - 256)
    return CA_ERR_UNSUPPORTED;
  p.kblocks = static_cast<int>((q->cols * es + 127) / 128);
  p.out_f32 = out_f32 ? 1 : 0;
  return CA_OK;
}

int linear_q8_impl(const ca_linear_q8_args* a, cudaStream_t st) {
  if (!a) return CA_ERR_INVALID;
  Product q{};
  q.act = a->act;
  q.w = a->w;
  q.act_stride = a->act_stride;
  q.cols = a->cols;
  q.p.act_scale = a->act_scale;
  q.p.w_scale = a->w_scale;
  q.p.bias = a->bias;
  q.p.residual = a->residual;
  q.p.out = a->out;
  q.p.out_stride = a->out_stride;
  q.p.res_stride = a->residual_stride;
  q.p.n = a->n;
  q.p.rows = a->rows;
  q.p.err = a->status;
  const int rc = check_product(&q, 1, a->out_f32);
  if (rc != CA_OK || q.p.n == 0) return rc;
  return launch_product<kKindE4m3, 1>(q, st);
}

int gated_linear_impl(const ca_gated_linear_args* a, cudaStream_t st) {
  if (!a || !a->w_up) return CA_ERR_INVALID;
  if (a->type != CA_TYPE_BF16 && a->type != CA_TYPE_E4M3) return CA_ERR_INVALID;
  if (a->activation != CA_ACT_SILU && a->activation != CA_ACT_GELU) return CA_ERR_INVALID;
  if (a->type == CA_TYPE_BF16 && (a->act_scale || a->gate_scale || a->up_scale))
    return CA_ERR_INVALID;
  Product q{};
  q.act = a->act;
  q.w = a->w_gate;
  q.up = a->w_up;
  q.act_stride = a->act_stride;
  q.cols = a->cols;
  q.p.act_scale = a->act_scale;
  q.p.w_scale = a->gate_scale;
  q.p.up_scale = a->up_scale;
  q.p.act = a->activation;
  q.p.out = a->out;
  q.p.out_stride = a->out_stride;
  q.p.n = a->n;
  q.p.rows = a->rows;
  q.p.err = a->status;
  const int rc = check_product(&q, type_size(a->type), a->out_f32);
  if (rc != CA_OK || q.p.n == 0) return rc;
  return a->type == CA_TYPE_BF16 ? launch_product<kKindBf16, 2>(q, st)
                                 : launch_product<kKindE4m3, 2>(q, st);
}

}  // namespace
}  // namespace ca

extern "C" {

int ca_rms_norm(const ca_rms_norm_args* a, void* stream) {
  return ca::rms_norm_impl(a, static_cast<cudaStream_t>(stream));
}

int ca_linear_q8(const ca_linear_q8_args* a, void* stream) {
  return ca::linear_q8_impl(a, static_cast<cudaStream_t>(stream));
}

int ca_gated_linear(const ca_gated_linear_args* a, void* stream) {
  return ca::gated_linear_impl(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
