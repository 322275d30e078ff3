// kv8_api.cuh -- argument checks and launches of the 8-bit cache's entry
// points (include/canvas_attn.h: ca_kv8_*, ca_attention_kv8_*). Part of the
// library's single translation unit, after canvas_attn.cu's helpers.
#pragma once

#include "attn_kv8_rows.cuh"
#include "attn_kv8_tile.cuh"
#include "kv8.cuh"

namespace ca {
namespace {

constexpr int kSms = 148;

// A launch that may overlap the end of the kernel before it (dependency_wait).
template <class... P, class... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                 A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return CA_ERR_CUDA;
  }
  return CA_OK;
}

// The cache as the kernels see it, or why not.
int kv8_view(const ca_kv8_cache& c, Kv8View* v) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return CA_ERR_INVALID;
  if (c.batch < 0 || c.n_total <= 0 || c.n_head_kv <= 0 || c.head_dim <= 0) return CA_ERR_INVALID;
  if (c.head_dim % 16 || c.head_dim > 512) return CA_ERR_UNSUPPORTED;
  if (c.block_tokens != 16 && c.block_tokens != 32 && c.block_tokens != 64 &&
      c.block_tokens != 128)
    return CA_ERR_UNSUPPORTED;
  const int64_t dense = static_cast<int64_t>(c.n_head_kv) * c.head_dim;
  const int64_t rs = c.row_stride ? c.row_stride : dense;
  if (rs < dense || rs % 16 || !aligned16(c.k) || !aligned16(c.v)) return CA_ERR_INVALID;
  if (dense > INT_MAX) return CA_ERR_UNSUPPORTED;
  v->k = static_cast<uint8_t*>(c.k);
  v->v = static_cast<uint8_t*>(c.v);
  v->k_scale = c.k_scale;
  v->v_scale = c.v_scale;
  v->batch = c.batch;
  v->n_total = c.n_total;
  v->Hkv = c.n_head_kv;
  v->hd = c.head_dim;
  v->T = c.block_tokens;
  v->n_blocks = (c.n_total + c.block_tokens - 1) / c.block_tokens;
  v->row_stride = rs;
  return CA_OK;
}

int kv8_store_impl(const ca_kv8_store_args* a, cudaStream_t st) {
  if (!a || !a->k || !a->v || !a->active_pos) return CA_ERR_INVALID;
  Kv8StoreParams p{};
  const int rc = kv8_view(a->cache, &p.c);
  if (rc != CA_OK) return rc;
  if (!aligned16(a->k) || !aligned16(a->v)) return CA_ERR_INVALID;
  if (a->cu_active ? a->total_active < 0 : a->n_active < 0) return CA_ERR_INVALID;
  p.rows = a->cu_active ? a->total_active : static_cast<int64_t>(p.c.batch) * a->n_active;
  if (p.c.batch == 0 || p.rows == 0) return CA_OK;
  if (p.rows > INT_MAX) return CA_ERR_UNSUPPORTED;
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.pos = a->active_pos;
  p.cu_active = a->cu_active;
  p.kv_len = a->kv_len;
  p.na = a->n_active;
  p.err = a->status;
  if (!p.cu_active && a->n_active == p.c.n_total && p.c.batch <= 65535) {
    const dim3 grid(p.c.n_blocks * 2 * p.c.Hkv, p.c.batch);
    return launch_after(kv8_store_all_kernel, grid, 128, 0, st, p);
  }
  // Entries of the active list a job looks through: one where that leaves
  // half the GPU's warp slots at most one job each, 32 (a lane each) at most.
  // From 8 on, rows are many and mostly side by side: four warps a job.
  const int64_t slots = static_cast<int64_t>(kSms) * 32;
  const int64_t one = p.rows * 2 * p.c.Hkv;
  p.rows_per_job = static_cast<int>(std::min<int64_t>(32, (one + slots - 1) / slots));
  const bool many = p.rows_per_job >= 8;
  if (many) p.rows_per_job = 32;
  const int64_t jobs = (p.rows + p.rows_per_job - 1) / p.rows_per_job * 2 * p.c.Hkv;
  if (many)
    return launch_after(kv8_store_kernel<4, 8>,
                        dim3(static_cast<unsigned>(std::min<int64_t>(jobs, kSms * 1024))), 128, 0,
                        st, p);
  return launch_after(kv8_store_kernel<1, 1>,
                      dim3(static_cast<unsigned>(std::min<int64_t>((jobs + 7) / 8, kSms * 64))),
                      256, 0, st, p);
}

int kv8_load_impl(const ca_kv8_load_args* a, cudaStream_t st) {
  if (!a) return CA_ERR_INVALID;
  Kv8LoadParams p{};
  const int rc = kv8_view(a->cache, &p.c);
  if (rc != CA_OK) return rc;
  if ((!a->k_out && !a->v_out) || a->n_pos < 0 || (!a->pos && a->n_pos > p.c.n_total))
    return CA_ERR_INVALID;
  if ((a->k_out && !aligned16(a->k_out)) || (a->v_out && !aligned16(a->v_out)))
    return CA_ERR_INVALID;
  if (a->n_pos == 0 || p.c.batch == 0) return CA_OK;
  if (p.c.batch > 65535) return CA_ERR_UNSUPPORTED;
  p.k_out = a->k_out;
  p.v_out = a->v_out;
  p.out_f32 = a->out_f32 ? 1 : 0;
  p.pos = a->pos;
  p.n_pos = a->n_pos;
  p.err = a->status;
  // Four rows in flight where that still gives each SM its eight CTAs.
  const int upr = p.c.Hkv * p.c.hd / 16;
  const int rows = upr < 256 ? 256 / upr : 1;
  const int64_t pieces = (static_cast<int64_t>(a->n_pos) + rows - 1) / rows;
  const int64_t tensors = 2ll * p.c.batch;
  const bool many = pieces * tensors >= 4 * 8 * kSms;
  const int64_t blocks =
      many ? std::min<int64_t>((pieces + 3) / 4, std::max<int64_t>(1, 8 * kSms / tensors)) : pieces;
  const dim3 grid(static_cast<unsigned>(blocks), 2, p.c.batch);
  return many ? launch_after(kv8_load_kernel<4>, grid, 256, 0, st, p)
              : launch_after(kv8_load_kernel<1>, grid, 256, 0, st, p);
}

// How a call is laid out: which kernel, row tiles and splits of the keys.
struct Kv8Plan {
  int nr;  // query rows of a CTA: 128 (attn_kv8_tile.cuh), 16 or 8
  int tiles, splits;
  int64_t ws_bytes;
};

int kv8_plan(const ca_attn_kv8_args* a, const Kv8View& c, bool split_ok, Kv8Plan* pl) {
  const int64_t max_sq = a->cu_q ? a->max_sq : a->sq;
  const int64_t G = a->n_head / c.Hkv;
  const int64_t rows = max_sq * G;
  // Rows of the tensor maps are int32, a tile's last ones past the end too.
  if (static_cast<int64_t>(c.batch) * c.n_total > INT_MAX - 128) return CA_ERR_UNSUPPORTED;
  // Measured with 16 sequences of 4128 positions, 4 query heads a kv head, in
  // us, rows kernel against tile kernel: 8 rows 31 and 45 at head_dim 128, 35
  // and 51 at 256, 23 and 40 at 64; 16 rows 47 and 45, 49 and 55, 33 and 39;
  // 20 rows (a tile of 16 more) 89 and 46, 92 and 57, 60 and 40.
  const int tr = rows > 16 && c.hd <= 256 ? 128 : rows > 8 && c.hd <= 128 ? 16 : 8;
  pl->nr = tr;
  const int64_t tiles = (rows + tr - 1) / tr;
  if (tiles > INT_MAX / 1024) return CA_ERR_UNSUPPORTED;
  const int64_t cells = tiles * c.Hkv * c.batch;
  // A key axis is split where the row tiles alone would leave SMs idle, into
  // stretches of at least 256 keys (one chunk a warp; 1001 keys of 4 kv heads
  // took 1.9 us less than with 1024) or 512 (four tiles).
  int64_t splits = 1;
  if (split_ok && cells > 0 && cells < kSms)
    splits = std::max<int64_t>(
        1, std::min<int64_t>(kSms / cells, c.n_total / (tr == 128 ? 512 : 256)));
  pl->tiles = static_cast<int>(tiles);
  pl->splits = static_cast<int>(splits);
  pl->ws_bytes = splits == 1 ? 0
                             : CA_KV8_TICKET_BYTES +
                                   cells * splits * (static_cast<int64_t>(tr) * c.hd + 2 * tr) * 4;
  return CA_OK;
}

int attn_kv8_check(const ca_attn_kv8_args* a, Kv8View* c) {
  if (!a) return CA_ERR_INVALID;
  const int rc = kv8_view(a->cache, c);
  if (rc != CA_OK) return rc;
  if (a->n_head <= 0 || a->n_head % c->Hkv) return CA_ERR_INVALID;
  if (a->cu_q ? (a->max_sq < 0 || a->total_q < 0) : a->sq < 0) return CA_ERR_INVALID;
  if (c->batch > 65535 || c->Hkv > 65535) return CA_ERR_UNSUPPORTED;
  const int64_t total_q = a->cu_q ? a->total_q : static_cast<int64_t>(c->batch) * a->sq;
  if (total_q > INT_MAX) return CA_ERR_UNSUPPORTED;
  // Rows that no sequence could hold would be left unwritten.
  if (a->cu_q && total_q > static_cast<int64_t>(c->batch) * a->max_sq) return CA_ERR_INVALID;
  return CA_OK;
}

// e4m3 rows [tokens][kv heads][head_dim] in boxes of 128 bytes x 1 head x
// `keys` tokens, 128-byte swizzle; what lies outside reads as zero.
int make_tmap_kv8(CUtensorMap* m, const uint8_t* base, const Kv8View& c, uint32_t keys) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return CA_ERR_CUDA;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.hd), static_cast<cuuint64_t>(c.Hkv),
                        static_cast<cuuint64_t>(c.batch) * c.n_total};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.hd), static_cast<cuuint64_t>(c.row_stride)};
  cuuint32_t box[3] = {128, 1, keys};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r =
      fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(base), dims, strides, box, es,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CA_OK : CA_ERR_INVALID;
}

template <class C>
int launch_rows(const Kv8AttnParams& p, cudaStream_t st) {
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CA_ERR_CUDA;
  CUtensorMap tk, tv;
  int rc;
  if ((rc = make_tmap_kv8(&tk, p.c.k, p.c, 16)) != CA_OK) return rc;
  if ((rc = make_tmap_kv8(&tv, p.c.v, p.c, 16)) != CA_OK) return rc;
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(attn_kv8_rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::kSmem) != cudaSuccess)
      return CA_ERR_CUDA;
    attr_done[dev] = true;
  }
  const dim3 grid(p.tiles * p.splits, p.c.Hkv, p.c.batch);
  return launch_after(attn_kv8_rows_kernel<C>, grid, C::kThreads, C::kSmem, st, tk, tv, p);
}

template <class C>
int launch_tile(const Kv8AttnParams& p, cudaStream_t st) {
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CA_ERR_CUDA;
  CUtensorMap tk, tv;
  int rc;
  if ((rc = make_tmap_kv8(&tk, p.c.k, p.c, C::BN)) != CA_OK) return rc;
  if ((rc = make_tmap_kv8(&tv, p.c.v, p.c, C::BN)) != CA_OK) return rc;
  if (!attr_done[dev]) {
    if (C::REGS) {
      // The warpgroups' shares come out of the block's registers at launch
      // (eight a thread at a time): a build with fewer would wait for good.
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, attn_kv8_tile_kernel<C>) != cudaSuccess ||
          (fa.numRegs + 7) / 8 * 8 * C::kThreads < C::kRegsAsked)
        return CA_ERR_CUDA;
    }
    if (cudaFuncSetAttribute(attn_kv8_tile_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::kSmem) != cudaSuccess)
      return CA_ERR_CUDA;
    attr_done[dev] = true;
  }
  const dim3 grid(p.tiles * p.splits, p.c.Hkv, p.c.batch);
  return launch_after(attn_kv8_tile_kernel<C>, grid, C::kThreads, C::kSmem, st, tk, tv, p);
}

// `check_only`: says whether the call would be taken, and launches nothing.
int attn_kv8_impl(const ca_attn_kv8_args* a, cudaStream_t st, bool check_only = false) {
  Kv8AttnParams p{};
  int rc = attn_kv8_check(a, &p.c);
  if (rc != CA_OK) return rc;
  if (!a->q || !a->out) return CA_ERR_INVALID;
  const int H = a->n_head, hd = p.c.hd;
  const int64_t dense = static_cast<int64_t>(H) * hd;
  p.q_row_stride = a->q_row_stride ? a->q_row_stride : dense;
  p.out_row_stride = a->out_row_stride ? a->out_row_stride : dense;
  if (p.q_row_stride < dense || p.out_row_stride < dense || p.q_row_stride % 8 ||
      p.out_row_stride % (a->out_f32 ? 4 : 8) || !aligned16(a->q) || !aligned16(a->out))
    return CA_ERR_INVALID;
  const int64_t max_sq = a->cu_q ? a->max_sq : a->sq;
  const int64_t total_q = a->cu_q ? a->total_q : static_cast<int64_t>(p.c.batch) * a->sq;
  if (p.c.batch == 0 || total_q == 0 || max_sq == 0) return CA_OK;
  Kv8Plan pl;
  if ((rc = kv8_plan(a, p.c, a->workspace != nullptr, &pl)) != CA_OK) return rc;
  if (a->workspace && (!aligned16(a->workspace) || a->workspace_bytes < pl.ws_bytes))
    return CA_ERR_INVALID;
  if (check_only) return CA_OK;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = a->out;
  p.out_f32 = a->out_f32 ? 1 : 0;
  p.sq = a->sq;
  p.cu_q = a->cu_q;
  p.q_pos = a->q_pos;
  p.kv_len = a->kv_len;
  p.seq_prefix = a->seq_prefix;
  p.causal_prefix = clamp_opt(a->causal_prefix);
  p.window = a->sliding_window < 0 ? kNoWindow
                                   : static_cast<int>(std::min<int64_t>(a->sliding_window,
                                                                        INT_MAX - 1));
  p.H = H;
  p.G = H / p.c.Hkv;
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.softcap = a->softcap > 0.f ? a->softcap : 0.f;
  p.splits = pl.splits;
  p.tiles = pl.tiles;
  p.err = a->status;
  if (pl.splits > 1) {
    const int64_t cells = static_cast<int64_t>(pl.tiles) * p.c.Hkv * p.c.batch;
    p.tickets = static_cast<int*>(a->workspace);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + CA_KV8_TICKET_BYTES);
    p.part_o = p.part_ml + cells * pl.splits * 2 * pl.nr;
  }
  if (pl.nr == 128) {
    if (p.softcap != 0.f) {
      if (hd <= 64) return launch_tile<TileCfg<64, 1, true>>(p, st);
      if (hd <= 128) return launch_tile<TileCfg<128, 1, true>>(p, st);
      return launch_tile<TileCfg<256, 2, true>>(p, st);
    }
    if (hd <= 64) return launch_tile<TileCfg<64, 1, false>>(p, st);
    if (hd <= 128) return launch_tile<TileCfg<128, 1, false>>(p, st);
    return launch_tile<TileCfg<256, 2, false>>(p, st);
  }
  if (pl.nr == 16)
    return hd <= 64 ? launch_rows<RowsCfg<64, 16>>(p, st) : launch_rows<RowsCfg<128, 16>>(p, st);
  if (hd <= 64) return launch_rows<RowsCfg<64, 8>>(p, st);
  if (hd <= 128) return launch_rows<RowsCfg<128, 8>>(p, st);
  if (hd <= 256) return launch_rows<RowsCfg<256, 8>>(p, st);
  return launch_rows<RowsCfg<512, 8>>(p, st);
}

int block_kv8_impl(const ca_block_kv8_args* a, cudaStream_t st) {
  if (!a || !a->q || !a->k || !a->v || !a->active_pos || !a->rope || !a->work || !a->out)
    return CA_ERR_INVALID;
  Kv8View c;
  int rc = kv8_view(a->cache, &c);
  if (rc != CA_OK) return rc;
  const int H = a->n_head;
  if (H <= 0 || H % c.Hkv || !aligned16(a->work)) return CA_ERR_INVALID;
  if (a->cu_active ? (a->total_active < 0 || a->max_active < 0) : a->n_active < 0)
    return CA_ERR_INVALID;
  if (a->rope_dim < 0 || a->rope_dim > c.hd || a->rope_dim % 2 || a->rope_len < c.n_total)
    return CA_ERR_INVALID;
  const int64_t rows = a->cu_active ? a->total_active : static_cast<int64_t>(c.batch) * a->n_active;
  if (rows > INT_MAX) return CA_ERR_UNSUPPORTED;
  // The three parts are checked before the first is launched.
  __nv_bfloat16* wq = static_cast<__nv_bfloat16*>(a->work);
  __nv_bfloat16* wk = wq + rows * H * c.hd;
  __nv_bfloat16* wv = wk + rows * c.Hkv * c.hd;
  ca_kv8_store_args s{};
  s.cache = a->cache;
  s.k = wk;
  s.v = wv;
  s.n_active = a->n_active;
  s.active_pos = a->active_pos;
  s.cu_active = a->cu_active;
  s.total_active = a->total_active;
  s.kv_len = a->held;
  s.status = a->status;
  ca_attn_kv8_args t{};
  t.cache = a->cache;
  t.q = wq;
  t.out = a->out;
  t.out_f32 = a->out_f32;
  t.out_row_stride = a->out_row_stride;
  t.n_head = H;
  t.sq = a->n_active;
  t.cu_q = a->cu_active;
  t.max_sq = a->max_active;
  t.total_q = a->total_active;
  t.q_pos = a->active_pos;
  t.kv_len = a->kv_len;
  t.sliding_window = a->sliding_window;
  t.causal_prefix = a->causal_prefix;
  t.seq_prefix = a->seq_prefix;
  t.scale = a->scale;
  t.softcap = a->softcap;
  t.status = a->status;
  t.workspace = a->workspace;
  t.workspace_bytes = a->workspace_bytes;
  if ((rc = attn_kv8_impl(&t, st, true)) != CA_OK) return rc;
  if (c.batch == 0 || rows == 0) return CA_OK;
  PrepParams pp{};
  pp.q = static_cast<const __nv_bfloat16*>(a->q);
  pp.k = static_cast<const __nv_bfloat16*>(a->k);
  pp.v = static_cast<const __nv_bfloat16*>(a->v);
  pp.pos = a->active_pos;
  pp.q_norm_w = a->q_norm_w;
  pp.k_norm_w = a->k_norm_w;
  pp.v_norm = a->v_norm;
  pp.eps = a->rms_eps;
  pp.rope = a->rope;
  pp.rope_len = a->rope_len;
  pp.rope_dim = a->rope_dim;
  pp.q_out = wq;
  pp.cache_k = wk;
  pp.cache_v = wv;
  pp.kv_rows = 1;
  pp.batch = c.batch;
  pp.na = a->n_active;
  pp.n_total = c.n_total;
  pp.cu_active = a->cu_active;
  pp.total_active = a->total_active;
  pp.err = a->status;
  pp.H = H;
  pp.Hkv = c.Hkv;
  pp.hd = c.hd;
  const bool vec = aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->rope) &&
                   (!a->q_norm_w || aligned16(a->q_norm_w)) &&
                   (!a->k_norm_w || aligned16(a->k_norm_w)) && a->rope_dim % 16 == 0;
  if ((rc = launch_prep(pp, rows, vec, st)) != CA_OK) return rc;
  if ((rc = kv8_store_impl(&s, st)) != CA_OK) return rc;
  return attn_kv8_impl(&t, st);
}

}  // namespace
}  // namespace ca

extern "C" {

int ca_attention_block_kv8_dev(const ca_block_kv8_args* a, void* stream) {
  return ca::block_kv8_impl(a, static_cast<cudaStream_t>(stream));
}

int ca_kv8_store(const ca_kv8_store_args* a, void* stream) {
  return ca::kv8_store_impl(a, static_cast<cudaStream_t>(stream));
}

int ca_kv8_load(const ca_kv8_load_args* a, void* stream) {
  return ca::kv8_load_impl(a, static_cast<cudaStream_t>(stream));
}

int ca_attention_kv8_dev(const ca_attn_kv8_args* a, void* stream) {
  return ca::attn_kv8_impl(a, static_cast<cudaStream_t>(stream));
}

int64_t ca_attention_kv8_workspace(const ca_attn_kv8_args* a) {
  ca::Kv8View c;
  const int rc = ca::attn_kv8_check(a, &c);
  if (rc != CA_OK) return rc;
  ca::Kv8Plan pl;
  const int rp = ca::kv8_plan(a, c, true, &pl);
  return rp != CA_OK ? rp : pl.ws_bytes;
}

}  // extern "C"
