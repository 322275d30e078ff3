// sample.cu -- ca_sample (include/canvas_attn.h): argument checks and launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "canvas_attn.h"
#include "host_util.cuh"
#include "sample.cuh"

namespace ca {
namespace {

template <class T>
int launch_sample(const ca_sample_args* a, SampleParams p, cudaStream_t st) {
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CA_ERR_CUDA;
  constexpr int most = kSampleSegBytes / sizeof(T);
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kSampleSegBytes + kSampleExtra) != cudaSuccess)
      return CA_ERR_CUDA;
    attr_done[dev] = true;
  }
  // As many CTAs a row as leave two on an SM (one loads while the other
  // computes), and more while SMs would idle and a thread has four entries.
  constexpr int two = 80 * 1024 / sizeof(T);
  int c = 1;
  while (c < 8 && (p.n_vocab > c * two || (a->n_cand * 2ll * c <= 2 * kSms &&
                                           p.n_vocab >= 2 * c * 4 * kSampleThreads)))
    c *= 2;
  if (p.n_vocab > static_cast<int64_t>(c) * most) return CA_ERR_UNSUPPORTED;
  p.seg = ((p.n_vocab + c - 1) / c + 127) / 128 * 128;
  return launch_cluster_after(sample_kernel<T>, dim3(static_cast<unsigned>(a->n_cand) * c),
                              kSampleThreads, p.seg * sizeof(T) + kSampleExtra, c, st, p);
}

int sample_impl(const ca_sample_args* a, cudaStream_t st) {
  if (!a || a->n_cand < 0 || a->n_vocab <= 0 || a->n_rows < 0 || a->n_suppress < 0 ||
      (a->n_suppress > 0 && !a->suppress))
    return CA_ERR_INVALID;
  if (a->n_cand == 0) return CA_OK;
  if (!a->logits || !a->u || !a->token) return CA_ERR_INVALID;
  if (a->n_vocab > INT_MAX || a->n_cand > INT_MAX / 8) return CA_ERR_UNSUPPORTED;
  const int64_t rs = a->row_stride ? a->row_stride : a->n_vocab;
  if (rs < a->n_vocab) return CA_ERR_INVALID;
  if (!a->rows && a->n_cand > a->n_rows) return CA_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->logits_bf16 ? 1u : 3u)) return CA_ERR_INVALID;
  for (const void* q : {static_cast<const void*>(a->rows), static_cast<const void*>(a->suppress),
                        static_cast<const void*>(a->u), static_cast<const void*>(a->token),
                        static_cast<const void*>(a->prob),
                        static_cast<const void*>(a->temperature_row),
                        static_cast<const void*>(a->top_k_row),
                        static_cast<const void*>(a->top_p_row),
                        static_cast<const void*>(a->min_p_row)})
    if (reinterpret_cast<uintptr_t>(q) & 3u) return CA_ERR_INVALID;
  if (a->n_vocab > 8ll * kSampleSegBytes / (a->logits_bf16 ? 2 : 4)) return CA_ERR_UNSUPPORTED;
  SampleParams p{};
  p.logits = a->logits;
  p.row_stride = rs;
  p.n_rows = a->n_rows;
  p.n_vocab = static_cast<int>(a->n_vocab);
  p.rows = a->rows;
  p.mask_id = a->mask_id;
  p.suppress = a->suppress;
  p.n_suppress = a->n_suppress;
  p.u = a->u;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.temperature_row = a->temperature_row;
  p.top_k_row = a->top_k_row;
  p.top_p_row = a->top_p_row;
  p.min_p_row = a->min_p_row;
  p.token = a->token;
  p.prob = a->prob;
  return a->logits_bf16 ? launch_sample<uint16_t>(a, p, st) : launch_sample<float>(a, p, st);
}

}  // namespace
}  // namespace ca

extern "C" int ca_sample(const ca_sample_args* a, void* stream) {
  return ca::sample_impl(a, static_cast<cudaStream_t>(stream));
}
