// sample.cuh -- a token for each candidate row of a denoising step's logits:
// temperature, top-k, top-p and min-p, from a given random number.
//
//   w_j = exp((l_j - m) / T), m the row's maximum
//   kept: a prefix of the row in the order (value descending, index
//   ascending), cut by top_k, by the weights before an entry reaching top_p of
//   those of the top_k, and by w_j >= min_p
//   token: the first kept j whose kept weights up to j exceed u * all of them
//
// Every cut is a border (key K, index I): an entry is before it if its key is
// above K, or equal with an index of at most I. Sums decide which side of a
// border a number falls on, so they are exact whatever their order: weights
// are taken in 64 bits and rounded to steps of 2^-44 (a row's largest is 1),
// and whole numbers are added.
//
// A cluster of 1 to 8 CTAs takes a row: its segments stay in shared memory,
// so HBM sees the logits once, and what the CTAs have to tell each other goes
// through distributed shared memory.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>

#include "cluster.cuh"

namespace ca {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleSegBytes = 208 * 1024;  // of a row, a CTA

struct SampleParams {
  const void* logits;
  long long row_stride, n_rows;
  int n_vocab, seg;  // entries of a CTA
  const int* rows;
  int mask_id;
  const int* suppress;
  int n_suppress;
  const float* u;
  float temperature, top_p, min_p;
  int top_k;
  const float* temperature_row;
  const float* top_p_row;
  const float* min_p_row;
  const int* top_k_row;
  int* token;
  float* prob;
};

typedef unsigned long long u64;

// Keys in the order of the values.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// Weights in steps of 2^-44, by the alignment of a sum with 256.
__device__ __forceinline__ u64 fixed44(double w) {
  return static_cast<u64>(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0));
}

struct SampleShared {
  u64 warp_sum[kSampleWarps];
  u64 cta_sum[2];
  uint32_t found[2];
  float max_v[kSampleWarps];
  float cta_max;
};

template <class T>
struct SampleRow {
  const T* seg;
  int len, first;  // entries of this CTA's segment, the first one's index
  int lo, hi;      // this warp's entries in it
  int lane, warp;
  uint32_t rank, n_ranks;
  SampleShared* sh;
  int turn = 0;

  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4)
      return seg[i];
    else
      return __uint_as_float(static_cast<uint32_t>(seg[i]) << 16);
  }

  // The sum of q(value, index) over the row; `before`: over the entries of
  // lower ranks, `mine`: over this warp's.
  template <class Q>
  __device__ __forceinline__ u64 total(Q q, u64& before, u64& mine) {
    u64 s = 0;
    for (int i = lo + lane; i < hi; i += 32) s += q(at(i), first + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    mine = s;
    if (lane == 0) sh->warp_sum[warp] = s;
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      u64 c = sh->warp_sum[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
      if (lane == 0) sh->cta_sum[turn] = c;
    }
    __syncwarp();
    cluster_sync_all();
    u64 all = 0;
    before = 0;
    for (uint32_t r = 0; r < n_ranks; ++r) {
      const u64 c = ld_cluster_u64(map_to_rank(smem_addr(&sh->cta_sum[turn]), r));
      if (r < rank) before += c;
      all += c;
    }
    return all;
  }
  template <class Q>
  __device__ __forceinline__ u64 total(Q q) {
    u64 a, b;
    return total(q, a, b);
  }

  // The first index up to which q sums to more than target(sum over the row).
  template <class Q, class F>
  __device__ __forceinline__ int find(Q q, F target_of) {
    u64 before, mine;
    const u64 all = total(q, before, mine);
    const u64 target = target_of(all);
    u64 s = before;
    for (int w = 0; w < warp; ++w) s += sh->warp_sum[w];
    if (s <= target && target < s + mine) {
      for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        u64 c = i < hi ? q(at(i), first + i) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 t = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += t;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, s + c > target);
        if (over) {
          const int k = __ffs(over) - 1;
          if (static_cast<uint32_t>(lane) < n_ranks)
            st_cluster_u32(map_to_rank(smem_addr(&sh->found[turn]), lane),
                           static_cast<uint32_t>(first + i0 + k));
          break;
        }
        s += __shfl_sync(0xffffffffu, c, 31);
      }
    }
    __syncwarp();
    cluster_sync_all();
    return static_cast<int>(sh->found[turn]);
  }

  __device__ __forceinline__ static uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
  }
};

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t raw_smem[];
  __shared__ SampleShared sh;
  T* seg = reinterpret_cast<T*>(raw_smem);
  const int tid = threadIdx.x;
  wait_prior_kernel();
  let_next_kernel();

  SampleRow<T> row;
  row.rank = cluster_rank();
  row.n_ranks = cluster_size();
  const int cand = static_cast<int>(blockIdx.x / row.n_ranks);
  const long long at = p.rows ? p.rows[cand] : cand;
  if (at < 0 || at >= p.n_rows) {  // the same for the whole cluster
    if (tid == 0 && row.rank == 0) {
      p.token[cand] = -1;
      if (p.prob) p.prob[cand] = 0.f;
    }
    return;
  }
  row.seg = seg;
  row.first = static_cast<int>(row.rank) * p.seg;
  row.len = max(0, min(p.seg, p.n_vocab - row.first));
  row.lane = tid & 31;
  row.warp = tid >> 5;
  row.sh = &sh;
  const int share = ((row.len + kSampleThreads - 1) / kSampleThreads) * 32;
  row.lo = min(row.len, row.warp * share);
  row.hi = min(row.len, row.lo + share);

  // The segment, NaN as -inf and -0 as +0, so that equal values have equal keys.
  constexpr int V = 16 / sizeof(T);
  const T* src = static_cast<const T*>(p.logits) + at * p.row_stride + row.first;
  auto clean = [](T x) -> T {
    if constexpr (sizeof(T) == 4) {
      return x == x ? x + 0.f : -INFINITY;
    } else {
      if ((x & 0x7fff) > 0x7f80) return 0xff80;
      return x == 0x8000 ? 0 : x;
    }
  };
  int i0 = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
    i0 = row.len / V * V;
    for (int i = tid * V; i < i0; i += kSampleThreads * V) {
      uint4 raw = *reinterpret_cast<const uint4*>(src + i);
      T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = clean(v[j]);
      *reinterpret_cast<uint4*>(seg + i) = raw;
    }
  }
  for (int i = i0 + tid; i < row.len; i += kSampleThreads) seg[i] = clean(src[i]);
  __syncthreads();
  auto drop = [&](int id) {
    const int i = id - row.first;
    if (id >= 0 && i >= 0 && i < row.len) {
      if constexpr (sizeof(T) == 4)
        seg[i] = -INFINITY;
      else
        seg[i] = 0xff80;
    }
  };
  if (tid == 0) drop(p.mask_id);
  for (int i = tid; i < p.n_suppress; i += kSampleThreads) drop(p.suppress[i]);
  __syncthreads();

  float m = -INFINITY;
  for (int i = row.lo + row.lane; i < row.hi; i += 32) m = fmaxf(m, row.at(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (row.lane == 0) sh.max_v[row.warp] = m;
  __syncthreads();
  if (row.warp == 0) {
    m = sh.max_v[row.lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (row.lane == 0) sh.cta_max = m;
  }
  __syncwarp();
  cluster_sync_all();
  m = -INFINITY;
  for (uint32_t r = 0; r < row.n_ranks; ++r)
    m = fmaxf(m, ld_cluster_f32(map_to_rank(row.smem_addr(&sh.cta_max), r)));

  const float T0 = p.temperature_row ? p.temperature_row[cand] : p.temperature;
  const int k0 = p.top_k_row ? p.top_k_row[cand] : p.top_k;
  const float tp = p.top_p_row ? p.top_p_row[cand] : p.top_p;
  const float mp = p.min_p_row ? p.min_p_row[cand] : p.min_p;

  int token = 0;
  if (m != -INFINITY) {
    if (!(T0 > 0.f)) {
      token = row.find([&](float l, int) -> u64 { return l == m; }, [](u64) -> u64 { return 0; });
    } else {
      const double inv_t = 1.0 / static_cast<double>(T0), md = m;
      auto weight = [&](float l) -> double {
        if (l == m) return 1.0;
        if (l == -INFINITY) return 0.0;
        return exp((static_cast<double>(l) - md) * inv_t);
      };
      uint32_t K = 0;
      int I = 0x7fffffff;
      auto before = [&](float l, int i) {
        const uint32_t k = key_of(l);
        return k > K || (k == K && i <= I);
      };
      if (k0 > 0 && k0 < p.n_vocab) {
        uint32_t key = 0;  // the largest key that k0 entries reach
        for (int b = 31; b >= 0; --b) {
          const uint32_t t = key | (1u << b);
          if (row.total([&](float l, int) -> u64 { return key_of(l) >= t; }) >=
              static_cast<u64>(k0))
            key = t;
        }
        const u64 above = row.total([&](float l, int) -> u64 { return key_of(l) > key; });
        const int last = row.find([&](float l, int) -> u64 { return key_of(l) == key; },
                                  [&](u64) -> u64 { return k0 - above - 1; });
        K = key;
        I = last;
      }
      if (tp < 1.f) {
        auto q = [&](float l, int i) -> u64 { return before(l, i) ? fixed44(weight(l)) : 0; };
        const double share_d = static_cast<double>(fmaxf(tp, 0.f)) * static_cast<double>(row.total(q));
        u64 need = static_cast<u64>(share_d);
        if (static_cast<double>(need) < share_d) ++need;
        if (need == 0) need = 1;
        uint32_t key = 0;  // the largest key whose entries and those above weigh `need`
        for (int b = 31; b >= 0; --b) {
          const uint32_t t = key | (1u << b);
          if (row.total([&](float l, int i) -> u64 { return key_of(l) >= t ? q(l, i) : 0; }) >= need)
            key = t;
        }
        const u64 above =
            row.total([&](float l, int i) -> u64 { return key_of(l) > key ? q(l, i) : 0; });
        const int last =
            row.find([&](float l, int i) -> u64 { return key_of(l) == key ? q(l, i) : 0; },
                     [&](u64) -> u64 { return need - above - 1; });
        K = key;
        I = last;
      }
      const double least = mp > 0.f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
      float u = p.u[cand];
      u = u >= 0.f ? fminf(u, 0.99999994f) : 0.f;
      token = row.find(
          [&](float l, int i) -> u64 {
            if (!before(l, i)) return 0;
            const double w = weight(l);
            return w >= least ? fixed44(w) : 0;
          },
          [&](u64 all) -> u64 {
            return static_cast<u64>(static_cast<double>(u) * static_cast<double>(all));
          });
    }
  }
  if (p.prob) {
    float pr = 0.f;
    if (m != -INFINITY) {
      auto e = [&](float l) { return l == m ? 1.f : expf(l - m); };
      const u64 all = row.total([&](float l, int) -> u64 { return fixed44(e(l)); });
      const int i = token - row.first;
      if (i >= 0 && i < row.len && tid == 0)
        p.prob[cand] = static_cast<float>(e(row.at(i)) / (static_cast<double>(all) * 0x1p-44));
    } else if (tid == 0 && row.rank == 0) {
      p.prob[cand] = pr;
    }
  }
  if (tid == 0 && row.rank == 0) p.token[cand] = token;
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

}  // namespace ca
