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
// are taken in 64 bits, rounded to steps of 2^-44 (a row's largest is 1), and
// whole numbers are added.
//
// A cluster of 1 to 8 CTAs takes a row: its segments stay in shared memory,
// so HBM sees the logits once, and what the CTAs have to tell each other goes
// through distributed shared memory.
//
// Borders are found in two steps. A histogram over log2 w (bins of 1/32,
// weights within a factor of 2^(1/32) of one another) tells which bins lie
// before a border for certain and which may hold it. Then either every entry
// up to there fits a list of the cluster's first CTA, which settles the rest
// by itself (a top-k, a sharp nucleus), or the entries of the doubtful bins do
// (a wide nucleus); doubtful bins that hold too many get a histogram of their
// own, finer by their number (32 rows of 250000 flat logits at top-p 0.9 189 us,
// bisected 1.5 ms). What fits none of these (thousands of equal logits; in fp32
// a top_k of more entries than the list has, together with top_p) is settled by
// bisection of the keys over the whole row, 32 sums a border (1.5 ms).
//
// A small top_k needs no histogram: each thread's maximum gives a value that
// at least top_k entries reach, and the entries from there on go to the list.
//
// bf16 logits take few values, so that their rows need less: a histogram over
// the values themselves (those of the 17 largest binades that count; smaller
// ones, next to zero, are few and weighed one by one) gives every sum of the
// row exactly from one weight a value, and the border's value with it. Only a
// border next to zero goes the general way.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>

#include "cluster.cuh"
#include "sm100.cuh"

namespace ca {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleSegBytes = 184 * 1024;  // of a row, a CTA
constexpr int kBins = 1536;                  // 1/32 each: beyond 2^-45 there is no weight
constexpr int kBinsEach = 4;                 // of a thread
static_assert(kBins / kBinsEach <= kSampleThreads, "bins");
constexpr float kBinsPerOctave = 32.f;
constexpr float kNowhere = 8388608.f + 46.f * kBinsPerOctave;  // of SampleWeights::place
constexpr int kListEach = 6;                 // entries of a thread
constexpr int kList = kListEach * kSampleThreads;
constexpr int kQueue = 160;                  // values a warp holds back
constexpr int kSampleExtra = kBins * 4 + kList * 8;
constexpr int kSide = 17 * 128;              // bf16 magnitudes of 17 binades
constexpr int kValues = 2 * kSide + 1;       // in order: positive, next to zero, negative
constexpr int kValuesEach = (kValues + kSampleThreads - 1) / kSampleThreads;
static_assert(kValuesEach * kSampleThreads * 4 <= kSampleExtra, "over the histogram and the list");
static_assert(kSampleWarps * kQueue * 4 <= kList * 8, "the queues lie over the list");

typedef unsigned long long u64;

struct SampleParams {
  const void* logits;
  long long row_stride, n_rows;
  int n_vocab, seg;  // entries of a CTA, a multiple of 128
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

// Keys in the order of the values, NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(fmaxf(l, -INFINITY) + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// A weight of at most 1 in steps of 2^-44, by the alignment of a sum with 256.
__device__ __forceinline__ u64 fixed44(double w) {
  return static_cast<u64>(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0));
}

// 2^a for -1000 < a < 1000 to 5e-16 and the roundings of its sums: a = n + f
// with n the nearest whole number (the low bits of a sum with 1.5 * 2^52), 2^f
// by the Chebyshev interpolation of degree 10 on [-1/2, 1/2], n added to the
// exponent. Its eleven nodes hold 0, so that 2^0 is 1 to the bit: a row's
// largest entry weighs exactly 1, which is what min_p counts on. The
// coefficients stand in constant memory, where an instruction takes them from
// directly: as immediates they cost two moves each, more than the arithmetic.
__constant__ double kExp2[11] = {
    1.0,                    0.69314718055995,       0.24022650695910097,   0.05550410866444772,
    0.009618129107606888,   0.0013333558230164974,  0.0001540353044173605, 1.5252657260200837e-05,
    1.321544258792169e-06,  1.0208690299958306e-07, 7.072585949269223e-09};
__device__ __forceinline__ double exp2_64(double a) {
  const double t = a + 6755399441055744.0;
  const double f = a - (t - 6755399441055744.0);
  double p = kExp2[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) p = fma(p, f, kExp2[i]);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

struct SampleShared {
  u64 warp_sum[kSampleWarps], warp_second[kSampleWarps];
  u64 cta_sum[2][8], cta_second[2][8];  // of every rank
  uint32_t found[2], first_found[2][8];
  float max_v[kSampleWarps], cta_max[8];
  uint32_t cta_cut[8];
  u64 equal_before[kSampleWarps];       // bf16: entries of the border's value
  uint32_t equal[kSampleWarps];
  double warp_d[kSampleWarps];
  uint32_t warp_u[kSampleWarps];
  uint32_t bin_lo, bin_hi, n_lo, n_hi;  // of the first CTA, and what it tells the others:
  uint32_t told[4];
  uint32_t border[3];              // key and index; bf16: value, how many of it, whether it holds
  uint32_t answer;
  u64 list_sum[kSampleWarps];
  u64 tiny_weight, tiny_one;       // of the values next to zero
  u64 range_sum[8 * kSampleWarps]; // of the first CTA: kept doubtful entries of every warp
};

// What a row's weights are made of.
struct SampleWeights {
  float m;
  float bin_c;    // place = -bin_c (l - m) + 2^23, whose low bits are the bin
  double c, top;  // log2 w = c (l - top), top: m in 64 bits
  double least;   // min_p

  // To the nearest bin; not below kNowhere for an entry without a weight (NaN
  // for NaN).
  __device__ __forceinline__ float place(float l) const {
    return fmaf(l - m, -bin_c, 8388608.f);
  }
  __device__ __forceinline__ bool none(float l) const { return !(place(l) < kNowhere); }
  __device__ __forceinline__ static uint32_t bin(float place) {
    return __float_as_uint(place) - 0x4B000000u;
  }
  // Of an entry that is not none(). The difference comes first: it is exact or
  // off by 2^-53 of itself, 0 for the maximum. c l - c m would be off by 2^-53 of
  // c m, which at low temperatures or far from 0 is more than there are bits.
  __device__ __forceinline__ double weight(float l) const {
    return exp2_64((static_cast<double>(l) - top) * c);
  }
  __device__ __forceinline__ u64 fixed(float l) const {
    return none(l) ? 0 : fixed44(weight(l));
  }
};

template <class T>
struct SampleRow {
  const T* seg;
  int first;   // index of the segment's first entry
  int share, padded;  // entries of a warp, of the segment: multiples of 128
  int lo, hi;         // this warp's
  int lane, warp;
  uint32_t rank, n_ranks;
  SampleShared* sh;
  uint32_t* hist;
  uint32_t* list_key;
  uint32_t* list_idx;
  int turn = 0;

  __device__ __forceinline__ void load4(int i, float (&v)[4]) const {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(seg + i);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(seg + i);
      v[0] = __uint_as_float(a.x << 16);
      v[1] = __uint_as_float(a.x & 0xffff0000u);
      v[2] = __uint_as_float(a.y << 16);
      v[3] = __uint_as_float(a.y & 0xffff0000u);
    }
  }

  __device__ __forceinline__ static uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
  }

  // Sums over a warp of numbers below 2^59: pieces of 27 bits (32 of them fit
  // 32 bits), each by one reduction instruction.
  __device__ __forceinline__ static u64 warp_total(u64 s) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(s) & 0x7ffffffu);
    const uint32_t b = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(s >> 27) & 0x7ffffffu);
    const uint32_t c = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(s >> 54));
    return a + (static_cast<u64>(b) << 27) + (static_cast<u64>(c) << 54);
  }

  // The sum of the warps' `mine` over the row; `before`: over lower ranks.
  // `second`: another sum, made that of the row. A CTA's sums are written to
  // every CTA before the barrier: reads of one another's after it cost about
  // 1000 clocks each.
  __device__ __forceinline__ u64 gather(u64 mine, u64& before, u64* second = nullptr) {
    __syncthreads();  // the last ones are read
    if (lane == 0) {
      sh->warp_sum[warp] = mine;
      if (second) sh->warp_second[warp] = *second;
    }
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      const u64 c = warp_total(lane < kSampleWarps ? sh->warp_sum[lane] : 0);
      if (lane < n_ranks) st_cluster_u64(map_to_rank(smem_addr(&sh->cta_sum[turn][rank]), lane), c);
      if (second) {
        const u64 d = warp_total(lane < kSampleWarps ? sh->warp_second[lane] : 0);
        if (lane < n_ranks)
          st_cluster_u64(map_to_rank(smem_addr(&sh->cta_second[turn][rank]), lane), d);
      }
    }
    cluster_sync_cta();
    u64 all = 0, all2 = 0;
    before = 0;
#pragma unroll
    for (uint32_t r = 0; r < 8; ++r) {
      if (r < n_ranks) {
        const u64 c = sh->cta_sum[turn][r];
        if (r < rank) before += c;
        all += c;
        if (second) all2 += sh->cta_second[turn][r];
      }
    }
    if (second) *second = all2;
    return all;
  }

  // exp(l - m) in fp32 (NaN as far below the maximum as counts for nothing).
  __device__ __forceinline__ static float term(float l, float m) {
    return ex2_approx(fmaxf(l - m, -200.f) * 1.4426950408889634f);
  }
  // A thread's sum of them as a warp's, in steps of 2^-40.
  __device__ __forceinline__ static u64 terms_total(float s) {
    return warp_total(static_cast<u64>(static_cast<double>(s) * 0x1p40));
  }

  // This warp's part of the sum of q(value, index); `terms`, if given: that of
  // exp(value - m).
  template <class Q>
  __device__ __forceinline__ u64 part(Q q, float m = 0.f, u64* terms = nullptr) {
    u64 s = 0;
    float e = 0.f;
    for (int i = lo + 4 * lane; i < hi; i += 128) {
      float v[4];
      load4(i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += q(v[j], first + i + j);
      if (terms) e += (term(v[0], m) + term(v[1], m)) + (term(v[2], m) + term(v[3], m));
    }
    if (terms) *terms = terms_total(e);
    return warp_total(s);
  }
  template <class Q>
  __device__ __forceinline__ u64 total(Q q) {
    u64 before;
    return gather(part(q), before);
  }

  // The first index up to which q sums to more than `target`, given what the
  // lower ranks hold; the warps' parts are those of the last gather.
  template <class Q>
  __device__ __forceinline__ int find(Q q, u64 target, u64 before) {
    return find_from(target, before, [](int, int, int) {}, q);
  }
  // `begin`(warp, first entry, one behind the last) is called by all threads
  // of the CTA that it falls in, before q is.
  template <class B, class Q>
  __device__ __forceinline__ int find_from(u64 target, u64 before, B begin, Q q) {
    // The warp whose entries it falls in; its CTA's warps then take a part of
    // them each, one warp would take many rounds.
    int owner = -1;
    u64 s = before, at = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) {
      const u64 t = sh->warp_sum[w];
      if (s <= target && target < s + t) {
        owner = w;
        at = s;
      }
      s += t;
    }
    if (owner >= 0) {  // the same for the whole CTA
      const int lo0 = min(owner * share, padded), hi0 = min(lo0 + share, padded);
      begin(owner, lo0, hi0);
      const int sub = (share / 128 + kSampleWarps - 1) / kSampleWarps * 128;
      const int lo1 = min(lo0 + warp * sub, hi0), hi1 = min(lo1 + sub, hi0);
      u64 c = 0;
      for (int i = lo1 + 4 * lane; i < hi1; i += 128) {
        float v[4];
        load4(i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) c += q(v[j], first + i + j);
      }
      c = warp_total(c);
      __syncthreads();  // the sums of whole warps are read
      if (lane == 0) sh->warp_sum[warp] = c;
      __syncthreads();
      u64 s1 = at;
      for (int w = 0; w < warp; ++w) s1 += sh->warp_sum[w];
      if (s1 <= target && target < s1 + c) {
        for (int i0 = lo1; i0 < hi1; i0 += 128) {
          const int i = i0 + 4 * lane;
          float v[4];
          load4(i, v);
          u64 e[4], c4 = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) c4 += e[j] = q(v[j], first + i + j);
          u64 up = c4;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += t;
          }
          const uint32_t over = __ballot_sync(0xffffffffu, s1 + up > target);
          if (over) {
            if (lane == __ffs(over) - 1) {
              u64 t = s1 + up - c4;
              int k = 0;
              while (k < 3 && t + e[k] <= target) t += e[k++];
              for (uint32_t r = 0; r < n_ranks; ++r)
                st_cluster_u32(map_to_rank(smem_addr(&sh->found[turn]), r),
                               static_cast<uint32_t>(first + i + k));
            }
            break;
          }
          s1 += __shfl_sync(0xffffffffu, up, 31);
        }
      }
    }
    cluster_sync_cta();
    return static_cast<int>(sh->found[turn]);
  }
  template <class Q, class F>
  __device__ __forceinline__ int find(Q q, F target_of) {
    u64 before;
    const u64 all = gather(part(q), before);
    return find(q, target_of(all), before);
  }

  // The first index whose value is `m` (there is one).
  __device__ __forceinline__ int first_of(float m) {
    uint32_t best = 0xffffffffu;
    for (int i0 = lo; i0 < hi; i0 += 128) {
      const int i = i0 + 4 * lane;
      float v[4];
      load4(i, v);
      const bool any = v[0] == m || v[1] == m || v[2] == m || v[3] == m;
      const uint32_t who = __ballot_sync(0xffffffffu, any);
      if (who) {
        const int k = v[0] == m ? 0 : v[1] == m ? 1 : v[2] == m ? 2 : 3;
        best = __shfl_sync(0xffffffffu, static_cast<uint32_t>(first + i + k), __ffs(who) - 1);
        break;
      }
    }
    if (lane == 0) sh->warp_u[warp] = best;
    __syncthreads();
    turn ^= 1;
    if (warp == 0) {
      best = __reduce_min_sync(0xffffffffu, lane < kSampleWarps ? sh->warp_u[lane] : 0xffffffffu);
      if (lane < n_ranks)
        st_cluster_u32(map_to_rank(smem_addr(&sh->first_found[turn][rank]), lane), best);
    }
    cluster_sync_cta();
    best = 0xffffffffu;
    for (uint32_t r = 0; r < n_ranks; ++r) best = min(best, sh->first_found[turn][r]);
    return static_cast<int>(best);
  }

  // This warp's part of the sum of q over the entries that `in` holds for:
  // those are queued, so that a warp's lanes have one each to weigh.
  // `equal`, if given: how many entries are `at`.
  template <class P, class Q>
  __device__ __forceinline__ u64 part_of(P in, Q q, float at = 0.f, u64* equal = nullptr) {
    uint32_t same = 0;
    float* queue = reinterpret_cast<float*>(list_key) + warp * kQueue;
    u64 s = 0;
    int n = 0;
    for (int i = lo + 4 * lane; i < hi; i += 128) {
      float v[4];
      load4(i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool t = in(v[j]);
        if (equal) same += v[j] == at ? 1 : 0;
        const uint32_t who = __ballot_sync(0xffffffffu, t);
        if (t) queue[n + __popc(who & ((1u << lane) - 1))] = v[j];
        n += __popc(who);
      }
      __syncwarp();
      while (n >= 32) {
        n -= 32;
        s += q(queue[n + lane]);
      }
      __syncwarp();
    }
    if (lane < n) s += q(queue[lane]);
    __syncwarp();
    if (equal) *equal = __reduce_add_sync(0xffffffffu, same);
    return warp_total(s);
  }

  // The index of the n-th entry of the segment's from .. to - 1 whose value is
  // `at` (there are as many; every warp looks for itself).
  __device__ __forceinline__ uint32_t nth_equal(float at, u64 n, int from, int to) {
    uint32_t last = 0;
    u64 seen = 0;
    for (int i0 = from; i0 < to && seen < n; i0 += 32) {
      const float l = value(i0 + lane);
      const uint32_t who = __ballot_sync(0xffffffffu, l == at);
      const int here = __popc(who);
      if (seen + here >= n)
        last = static_cast<uint32_t>(first + i0 + __fns(who, 0, static_cast<int>(n - seen)));
      seen += here;
    }
    return last;
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4)
      return seg[i];
    else
      return __uint_as_float(static_cast<uint32_t>(seg[i]) << 16);
  }

  // The first k (k < n <= kSampleThreads) of the n entries in this CTA's list,
  // whose keys lie between low and high, in the order of their indices again.
  // An entry a thread: a barrier counts.
  __device__ __forceinline__ void narrow(int n, int k, uint32_t low, uint32_t high) {
    const int tid = threadIdx.x;
    const uint32_t key = tid < n ? list_key[tid] : 0, idx = tid < n ? list_idx[tid] : 0;
    const int bits = low == high ? 0 : 32 - __clz(low ^ high);
    uint32_t K = bits == 32 ? 0 : high >> bits << bits;
#pragma unroll 1
    for (int b = bits - 1; b >= 0; --b) {
      const uint32_t t = K | (1u << b);
      if (__syncthreads_count(key >= t) >= k) K = t;
    }
    const int room = k - __syncthreads_count(key > K);  // for those of key K
    const uint32_t lower = (1u << lane) - 1;
    const uint32_t same = __ballot_sync(0xffffffffu, tid < n && key == K);
    if (lane == 0) sh->warp_u[warp] = __popc(same);
    __syncthreads();
    int at = __popc(same & lower);
    for (int w = 0; w < warp; ++w) at += sh->warp_u[w];
    const bool keep = tid < n && (key > K || (key == K && at < room));
    const uint32_t kept = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) sh->warp_u[warp] = __popc(kept);
    __syncthreads();
    at = __popc(kept & lower);
    for (int w = 0; w < warp; ++w) at += sh->warp_u[w];
    if (keep) {
      list_key[at] = key;
      list_idx[at] = idx;
    }
    __syncthreads();
  }

  // bf16: the place of a value among kValues, by its 15 low bits less those of
  // the smallest counted magnitude (below 0: next to zero; from kSide on: too
  // far down to count).
  __device__ __forceinline__ static int value_place(int i, bool negative) {
    return negative ? kSide + 1 + i : kSide - 1 - i;
  }

  // The entries that `in` holds for, in the order of their indices, into the
  // first CTA's list (at most kList of them; none if there are more).
  template <class P>
  __device__ __forceinline__ int collect(P in, float m = 0.f, u64* terms = nullptr) {
    uint32_t mine = 0;
    float e = 0.f;
    for (int i = lo + 4 * lane; i < hi; i += 128) {
      float v[4];
      load4(i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += in(v[j]) ? 1 : 0;
      if (terms) e += (term(v[0], m) + term(v[1], m)) + (term(v[2], m) + term(v[3], m));
    }
    if (terms) *terms = terms_total(e);
    const u64 n = __reduce_add_sync(0xffffffffu, mine);
    u64 before;
    const int all = static_cast<int>(gather(n, before, terms));
    u64 at = before;
    for (int w = 0; w < warp; ++w) at += sh->warp_sum[w];
    if (n > 0 && all <= kList) {
      const uint32_t keys = map_to_rank(smem_addr(list_key), 0);
      const uint32_t idxs = map_to_rank(smem_addr(list_idx), 0);
      for (int i0 = lo; i0 < hi; i0 += 128) {
        const int i = i0 + 4 * lane;
        float v[4];
        load4(i, v);
        int c = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) c += in(v[j]) ? 1 : 0;
        if (!__any_sync(0xffffffffu, c)) continue;
        int up = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, up, o);
          if (lane >= o) up += t;
        }
        uint32_t to = static_cast<uint32_t>(at) + up - c;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (in(v[j])) {
            st_cluster_u32(keys + 4 * to, key_of(v[j]));
            st_cluster_u32(idxs + 4 * to, static_cast<uint32_t>(first + i + j));
            ++to;
          }
        }
        at += __shfl_sync(0xffffffffu, up, 31);
      }
    }
    cluster_sync_cta();
    return all;
  }
};

// The first CTA's list: a thread holds the entries tid * kListEach and on, in
// the order of their indices. Only the warps that have entries take part.
struct SampleList {
  uint32_t key[kListEach], idx[kListEach];
  u64 w[kListEach];
  bool in[kListEach];
  SampleShared* sh;
  int lane, warp, warps;

  __device__ __forceinline__ void sync() const {
    if (warps > 1)
      named_bar_sync(1, warps * 32);
    else
      __syncwarp();
  }

  // Sum over the threads; of `before` over the lower threads.
  __device__ __forceinline__ u64 sum(u64 v, u64* before = nullptr) {
    u64 up = v;
    if (before) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += t;
      }
    }
    const u64 mine = SampleRow<float>::warp_total(v);
    u64 all = mine, low = 0;
    if (warps > 1) {
      sync();  // the last sum is read
      if (lane == 0) sh->list_sum[warp] = mine;
      sync();
      const u64 c = lane < warps ? sh->list_sum[lane] : 0;
      all = SampleRow<float>::warp_total(c);
      if (before) low = SampleRow<float>::warp_total(lane < warp ? c : 0);
    }
    if (before) *before = low + up - v;
    return all;
  }

  // The border at which `e` of the entries, in order, first sums to `need`
  // (of at most the whole sum): key and index of that entry.
  __device__ __forceinline__ void border(const u64 (&e)[kListEach], u64 need, uint32_t& K,
                                         uint32_t& I) {
    // Bits that all keys have in common need no sum.
    uint32_t hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kListEach; ++j) {
      if (e[j]) {
        hi = max(hi, key[j]);
        lo = min(lo, key[j]);
      }
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if (warps > 1) {
      sync();
      if (lane == 0) sh->list_sum[warp] = (static_cast<u64>(hi) << 32) | lo;
      sync();
      const u64 c = lane < warps ? sh->list_sum[lane] : 0xffffffffull;
      hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(c >> 32));
      lo = __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(c));
    }
    const int bits = hi == lo ? 0 : 32 - __clz(hi ^ lo);
    uint32_t k = bits == 32 ? 0 : hi >> bits << bits;
#pragma unroll 1
    for (int b = bits - 1; b >= 0; --b) {
      const uint32_t t = k | (1u << b);
      u64 s = 0;
#pragma unroll
      for (int j = 0; j < kListEach; ++j) s += key[j] >= t ? e[j] : 0;
      if (sum(s) >= need) k = t;
    }
    u64 above = 0, same = 0, low;
#pragma unroll
    for (int j = 0; j < kListEach; ++j) {
      above += key[j] > k ? e[j] : 0;
      same += key[j] == k ? e[j] : 0;
    }
    above = sum(above);
    sum(same, &low);
    u64 at = above + low;
#pragma unroll
    for (int j = 0; j < kListEach; ++j) {
      const u64 x = key[j] == k ? e[j] : 0;
      if (at < need && at + x >= need) sh->border[1] = idx[j];
      at += x;
    }
    sync();
    K = k;
    I = sh->border[1];
    sync();
#pragma unroll
    for (int j = 0; j < kListEach; ++j)
      in[j] = in[j] && (key[j] > K || (key[j] == K && idx[j] <= I));
  }
};

// Two CTAs an SM: 64 registers, with 80 bytes of spills (44 for bf16 rows).
template <class T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleParams p) {
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
  cluster_arrive_relaxed();  // (waited for before anything is written to another CTA)
  row.seg = seg;
  row.first = static_cast<int>(row.rank) * p.seg;
  auto len_in = [&](int rank) { return max(0, min(p.seg, p.n_vocab - rank * p.seg)); };
  // Entries of a warp of that rank.
  auto share_in = [&](int rank) {
    return ((len_in(rank) + 127) / 128 + kSampleWarps - 1) / kSampleWarps * 128;
  };
  const int len = len_in(static_cast<int>(row.rank));
  const int padded = (len + 127) / 128 * 128;
  row.lane = tid & 31;
  row.warp = tid >> 5;
  row.sh = &sh;
  row.hist = reinterpret_cast<uint32_t*>(raw_smem + p.seg * sizeof(T));
  row.list_key = row.hist + kBins;
  row.list_idx = row.list_key + kList;
  row.padded = padded;
  row.share = share_in(static_cast<int>(row.rank));
  row.lo = min(padded, row.warp * row.share);
  row.hi = min(padded, row.lo + row.share);

  // The segment, filled up with -inf.
  constexpr int V = 16 / sizeof(T);
  const T* src = static_cast<const T*>(p.logits) + at * p.row_stride + row.first;
  T nothing;
  if constexpr (sizeof(T) == 4)
    nothing = -INFINITY;
  else
    nothing = 0xff80;
  int i0 = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
    i0 = len / V * V;
    constexpr int U = 8;  // loads in flight
    constexpr int step = kSampleThreads * V;
    int i = tid * V;
    for (; i + (U - 1) * step < i0; i += U * step) {
      uint4 raw[U];
#pragma unroll
      for (int k = 0; k < U; ++k) raw[k] = *reinterpret_cast<const uint4*>(src + i + k * step);
#pragma unroll
      for (int k = 0; k < U; ++k) *reinterpret_cast<uint4*>(seg + i + k * step) = raw[k];
    }
#pragma unroll 2
    for (; i < i0; i += step)
      *reinterpret_cast<uint4*>(seg + i) = *reinterpret_cast<const uint4*>(src + i);
  }
#pragma unroll 4
  for (int i = i0 + tid; i < len; i += kSampleThreads) seg[i] = src[i];
  for (int i = len + tid; i < padded; i += kSampleThreads) seg[i] = nothing;
  for (int i = tid; i < (sizeof(T) == 2 ? kValuesEach * kSampleThreads : kBins);
       i += kSampleThreads)
    row.hist[i] = 0;
  if (tid == 0) {
    sh.tiny_weight = sh.tiny_one = 0;
    sh.border[0] = __float_as_uint(-INFINITY);  // no border
    sh.border[1] = 0;
    sh.border[2] = 1;
    sh.found[0] = sh.found[1] = sh.answer = 0;
  }
  for (int i = tid; i < 8 * kSampleWarps; i += kSampleThreads) sh.range_sum[i] = 0;
  __syncthreads();
  auto drop = [&](int id) {
    const int i = id - row.first;
    if (id >= 0 && i >= 0 && i < len) seg[i] = nothing;
  };
  if (tid == 0) drop(p.mask_id);
  for (int i = tid; i < p.n_suppress; i += kSampleThreads) drop(p.suppress[i]);
  __syncthreads();

  float m = -INFINITY;
  if constexpr (sizeof(T) == 4) {
    for (int i = 4 * tid; i < padded; i += 4 * kSampleThreads) {
      float v[4];
      row.load4(i, v);
      m = fmaxf(m, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    }
  } else {
    uint32_t mm = 0xff80ff80u;  // two at a time; NaN has no part
    for (int i = 8 * tid; i < padded; i += 8 * kSampleThreads) {
      const uint4 a = *reinterpret_cast<const uint4*>(seg + i);
      asm("max.bf16x2 %0, %0, %1;\n\tmax.bf16x2 %0, %0, %2;\n\tmax.bf16x2 %0, %0, %3;\n\t"
          "max.bf16x2 %0, %0, %4;" : "+r"(mm) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w));
    }
    m = fmaxf(__uint_as_float(mm << 16), __uint_as_float(mm & 0xffff0000u));
  }
  float own_max = m;  // over this thread's share of the segment
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (row.lane == 0) sh.max_v[row.warp] = m;
  __syncthreads();
  cluster_wait();  // every CTA of the cluster has started
  if (row.warp == 0) {
    m = row.lane < kSampleWarps ? sh.max_v[row.lane] : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (row.lane < row.n_ranks)
      st_cluster_u32(map_to_rank(row.smem_addr(&sh.cta_max[row.rank]), row.lane),
                     __float_as_uint(m));
  }
  cluster_sync_cta();
  m = -INFINITY;
  for (uint32_t r = 0; r < row.n_ranks; ++r) m = fmaxf(m, sh.cta_max[r]);

  m += 0.f;  // -0 as +0
  if (m == INFINITY) {
    // Infinite entries share the row: as zeros among -inf they have the same
    // weights and no arithmetic of their own.
    for (int i = tid; i < padded; i += kSampleThreads) {
      if constexpr (sizeof(T) == 4)
        seg[i] = seg[i] == INFINITY ? 0.f : -INFINITY;
      else
        seg[i] = seg[i] == 0x7f80 ? 0 : 0xff80;
    }
    m = 0.f;
    own_max = own_max == INFINITY ? 0.f : -INFINITY;
    __syncthreads();
  }

  const float temp = p.temperature_row ? p.temperature_row[cand] : p.temperature;
  const int top_k = p.top_k_row ? p.top_k_row[cand] : p.top_k;
  const float top_p = p.top_p_row ? p.top_p_row[cand] : p.top_p;
  const float min_p = p.min_p_row ? p.min_p_row[cand] : p.min_p;
  float u = p.u[cand];
  u = u >= 0.f ? fminf(u, 0.99999994f) : 0.f;
  auto share_of = [&](u64 all) -> u64 {
    return static_cast<u64>(static_cast<double>(u) * static_cast<double>(all));
  };
  // The whole numbers below a share of `all`, and at least 1: an entry is kept
  // while what is before it sums to less.
  auto need_of = [&](float part, u64 all) -> u64 {
    const double x = static_cast<double>(fmaxf(part, 0.f)) * static_cast<double>(all);
    u64 n = static_cast<u64>(x);
    if (static_cast<double>(n) < x) ++n;
    return n ? n : 1;
  };

  int token = 0;
  u64 one_all = 0;  // exp(l - m) over the row in steps of 2^-40, once known
  if (m != -INFINITY) {
    SampleWeights wt;
    wt.m = m;
    wt.least = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
    if (!(temp > 0.f)) {
      token = row.first_of(m);
    } else {
      // (Temperatures below 2^-100 as 2^-100.)
      wt.c = 1.4426950408889634 / static_cast<double>(fmaxf(temp, 0x1p-100f));
      wt.top = static_cast<double>(m);
      wt.bin_c = static_cast<float>(wt.c) * kBinsPerOctave;
      uint32_t K = 0, I = 0xffffffffu;
      auto before = [&](float l, int i) {
        const uint32_t k = key_of(l);
        return k > K || (k == K && static_cast<uint32_t>(i) <= I);
      };
      float end = kNowhere;  // places from here on have no weight, or are cut
      auto kept_weight = [&](float l) -> u64 {  // of any entry: 0 without a weight
        const double w = wt.weight(l);
        return wt.place(l) < end && w >= wt.least ? fixed44(w) : 0;
      };
      const bool by_k = top_k > 0 && top_k < p.n_vocab, by_p = top_p < 1.f;
      bool done = false;
      // The first CTA's list of n entries, by its warps that have any: borders
      // (of top_k, if `above` entries not listed come before; of top_p, if
      // entries of weight sure_all do), min_p, and the draw from a list that is
      // whole.
      auto settle = [&](int n, bool whole, u64 above, u64 need, u64 sure_all) {
        if (row.rank == 0 && row.warp * 32 * kListEach < max(n, 1)) {
          SampleList ls;
          ls.sh = &sh;
          ls.lane = row.lane;
          ls.warp = row.warp;
          ls.warps = (max(n, 1) + 32 * kListEach - 1) / (32 * kListEach);
          u64 e[kListEach];
#pragma unroll
          for (int j = 0; j < kListEach; ++j) {
            const int i = tid * kListEach + j;
            ls.in[j] = i < n;
            ls.key[j] = i < n ? row.list_key[i] : 0;
            ls.idx[j] = i < n ? row.list_idx[i] : 0;
            ls.w[j] = 0;
            if (i < n) ls.w[j] = fixed44(wt.weight(value_of(ls.key[j])));
          }
          if (by_k) {
            if (above + n > need) {  // otherwise all of them are kept
#pragma unroll
              for (int j = 0; j < kListEach; ++j) e[j] = ls.in[j];
              ls.border(e, need - above, K, I);
            }
          }
          if (by_p) {
            u64 c = 0;
#pragma unroll
            for (int j = 0; j < kListEach; ++j) c += e[j] = ls.in[j] ? ls.w[j] : 0;
            const u64 here = ls.sum(c);
            if (by_k) need = need_of(top_p, here);
            if (sure_all + here > need) ls.border(e, need - sure_all, K, I);
          }
          // min_p, and the draw: over a whole list in the order of the
          // indices; doubtful entries join what their warps are sure of.
          u64 c = 0, low;
#pragma unroll
          for (int j = 0; j < kListEach; ++j) {
            if (ls.in[j] && wt.least > 0.0 && wt.weight(value_of(ls.key[j])) < wt.least)
              ls.in[j] = false;
            c += e[j] = ls.in[j] ? ls.w[j] : 0;
          }
          if (whole) {
            const u64 sum = ls.sum(c, &low);
            const u64 target = share_of(sum);
#pragma unroll
            for (int j = 0; j < kListEach; ++j) {
              if (low <= target && target < low + e[j])
                for (uint32_t r = 0; r < row.n_ranks; ++r)
                  st_cluster_u32(map_to_rank(row.smem_addr(&sh.answer), r), ls.idx[j]);
              low += e[j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < kListEach; ++j) {
              if (e[j]) {
                const int rank = static_cast<int>(ls.idx[j]) / p.seg;
                const int w = (static_cast<int>(ls.idx[j]) - rank * p.seg) / share_in(rank);
                atomicAdd(&sh.range_sum[rank * kSampleWarps + w], e[j]);
              }
            }
          }
          ls.sync();
          if (tid < row.n_ranks && !whole) {
            st_cluster_u32(map_to_rank(row.smem_addr(&sh.border[0]), tid), K);
            st_cluster_u32(map_to_rank(row.smem_addr(&sh.border[1]), tid), I);
          }
        }
      };
      // Few entries of top_k: no fewer than top_k entries reach the top_k-th largest
      // of the threads' maxima in any CTA (to its upper 24 bits), so all that
      // may be kept is at or above the largest of these; few more if top_k is
      // well below the number of threads (k of t threads in each of c CTAs leave
      // at most -c t ln(1 - k / t) entries of a row without order, 1200 at the
      // limit below).
      if (by_k && top_k <= kSampleThreads / 2 &&
          static_cast<uint32_t>(top_k) * row.n_ranks <= 2 * kSampleThreads) {
        const uint32_t mine = key_of(own_max);
        uint32_t cut = 0;
#pragma unroll 1
        for (int b = 31; b >= 8; --b) {
          const uint32_t t = cut | (1u << b);
          if (__syncthreads_count(mine >= t) >= top_k) cut = t;
        }
        if (tid < row.n_ranks)
          st_cluster_u32(map_to_rank(row.smem_addr(&sh.cta_cut[row.rank]), tid), cut);
        cluster_sync_cta();
        for (uint32_t r = 0; r < row.n_ranks; ++r) cut = max(cut, sh.cta_cut[r]);
        const float least = value_of(max(cut, 0x007fffffu));
        u64 terms = 0;
        const int n = row.collect([&](float l) { return l >= least && wt.place(l) < kNowhere; }, m,
                                  p.prob ? &terms : nullptr);
        one_all = terms;
        if (n <= kList) {
          const bool few = n > top_k && n <= kSampleThreads;
          if (few && row.rank == 0) row.narrow(n, top_k, cut, key_of(m));
          settle(few ? top_k : n, true, 0, top_k, 0);
          cluster_sync_cta();
          token = static_cast<int>(sh.answer);
          done = true;
        }
      }
      if constexpr (sizeof(T) == 2) {
        if (!done && (by_k || by_p)) {
          // What counts lies between m and `far`, for the weights and for prob (whose
          // terms are below 1e-13 from there on); its magnitudes' binades.
          const float far = fmaxf(m - fmaxf(static_cast<float>(46.0 / wt.c), 32.f), -3e38f);
          const int top = static_cast<int>(
              __float_as_uint(fmaxf(fmaxf(fabsf(m), fabsf(far)), 0x1p-100f)) >> 23);
          const int least_bits = (top - 16) << 7;  // of the smallest counted magnitude
          uint32_t* const values = row.hist;
          u64 tiny = 0, tiny_one = 0;
          uint32_t tiny_n = 0;
          auto one_of = [&](float l) -> u64 {  // exp(l - m) in steps of 2^-40
            return static_cast<u64>(static_cast<double>(expf(l - m)) * 0x1p40);
          };
          for (int i = 8 * tid; i < padded; i += 8 * kSampleThreads) {
            const uint4 a = *reinterpret_cast<const uint4*>(seg + i);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t bits = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
              const int k = static_cast<int>(bits & 0x7fffu) - least_bits;
              const bool negative = bits >> 15;
              if (static_cast<uint32_t>(k) < static_cast<uint32_t>(kSide)) {
                atomicAdd(values + row.value_place(k, negative), 1u);
              } else if (k < 0) {
                const float l = __uint_as_float(bits << 16);
                tiny_one += one_of(l);
                if (!wt.none(l)) {
                  ++tiny_n;
                  tiny += fixed44(wt.weight(l));
                }
              }
            }
          }
          if (tiny_n || tiny_one) {
            atomicAdd(&sh.tiny_one, tiny_one);
            atomicAdd(values + kSide, tiny_n);
            atomicAdd(&sh.tiny_weight, tiny);
          }
          cluster_sync_cta();
          // Each CTA takes a share of the values, from the whole row, and of those
          // a thread the `each` from `o0` on.
          const int Q = kValuesEach * kSampleThreads / static_cast<int>(row.n_ranks);
          const int each = (Q + kSampleThreads - 1) / kSampleThreads;
          const int q0 = Q * static_cast<int>(row.rank), o0 = q0 + each * tid;
          if (row.n_ranks > 1) {
            for (int i = q0 + 4 * tid; i < q0 + Q; i += 4 * kSampleThreads) {
              uint4 c = make_uint4(0, 0, 0, 0);
#pragma unroll 4
              for (uint32_t r = 0; r < row.n_ranks; ++r) {
                uint4 t;
                asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w)
                             : "r"(map_to_rank(row.smem_addr(values + i), r)) : "memory");
                c.x += t.x;
                c.y += t.y;
                c.z += t.z;
                c.w += t.w;
              }
              *reinterpret_cast<uint4*>(values + i) = c;
            }
          }
          __syncthreads();
          auto value_at = [&](int o) {
            const int k = o < kSide ? kSide - 1 - o : o - kSide - 1;
            return __uint_as_float((static_cast<uint32_t>(k + least_bits) << 16) |
                                   (o > kSide ? 0x80000000u : 0u));
          };
          uint32_t n[kValuesEach];
          u64 w[kValuesEach], ones = 0, tiny_all = 0;
#pragma unroll
          for (int h = 0; h < kValuesEach; ++h) {
            const int o = o0 + h;
            n[h] = 0;
            w[h] = 0;
            if (h < each && o < q0 + Q && o < kValues) {
              n[h] = values[o];
              if (o == kSide) {
                for (uint32_t r = 0; r < row.n_ranks; ++r) {
                  tiny_all += ld_cluster_u64(map_to_rank(row.smem_addr(&sh.tiny_weight), r));
                  ones += ld_cluster_u64(map_to_rank(row.smem_addr(&sh.tiny_one), r));
                }
              } else if (n[h]) {
                const float l = value_at(o);
                ones += n[h] * one_of(l);
                if (wt.none(l))
                  n[h] = 0;
                else
                  w[h] = fixed44(wt.weight(l));
              }
            }
          }
          // What a value weighs, by how many of it count.
          auto here = [&](int h) -> u64 {
            return o0 + h == kSide ? (n[h] ? tiny_all : 0) : n[h] * w[h];
          };
          // Sum over the row; `low`: over the values before this thread's.
          auto scan = [&](u64 v, u64& low, u64* second) {
            u64 up = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const u64 t = __shfl_up_sync(0xffffffffu, up, o);
              if (row.lane >= o) up += t;
            }
            const u64 all = row.gather(__shfl_sync(0xffffffffu, up, 31), low, second);
            for (int i = 0; i < row.warp; ++i) low += sh.warp_sum[i];
            low += up - v;
            return all;
          };
          auto tell = [&](float value, uint32_t count, bool settled) {
            const uint32_t x[3] = {__float_as_uint(value), count, settled ? 1u : 0u};
            for (uint32_t r = 0; r < row.n_ranks; ++r)
#pragma unroll
              for (int i = 0; i < 3; ++i)
                st_cluster_u32(map_to_rank(row.smem_addr(&sh.border[i]), r), x[i]);
          };
          u64 low, second = row.warp_total(ones);
          if (by_k) {
            u64 c = 0;
#pragma unroll
            for (int h = 0; h < kValuesEach; ++h) c += n[h];
            scan(c, low, &second);
            one_all = second;
            const u64 k = static_cast<u64>(top_k);
#pragma unroll
            for (int h = 0; h < kValuesEach; ++h) {
              const u64 upto = low + n[h];
              if (k <= low) {
                n[h] = 0;
              } else if (k <= upto && n[h]) {
                n[h] = static_cast<uint32_t>(k - low);  // the last of them to be kept
                tell(value_at(o0 + h), n[h], o0 + h != kSide);
              }
              low = upto;
            }
          }
          if (by_p) {
            u64 c = 0;
#pragma unroll
            for (int h = 0; h < kValuesEach; ++h) c += here(h);
            const u64 all = scan(c, low, by_k ? nullptr : &second);
            if (!by_k) one_all = second;
            const u64 need = need_of(top_p, all);
            // (Where top_k cuts next to zero, what it leaves there is not known.)
            const bool known = sh.border[2];
#pragma unroll
            for (int h = 0; h < kValuesEach; ++h) {
              const u64 x = here(h);
              if (known && low < need && need <= low + x)
                tell(value_at(o0 + h),
                     o0 + h == kSide ? 0 : static_cast<uint32_t>((need - low + w[h] - 1) / w[h]),
                     o0 + h != kSide);
              low += x;
            }
          }
          cluster_sync_cta();
          if (sh.border[2]) {
            // Kept: what is above the border's value, and the first `count` of it
            // (without a border: every entry that has a weight).
            const float at = __uint_as_float(sh.border[0]);
            const u64 count = sh.border[1];
            u64 equal = 0, lower;
            u64 mine = row.part_of([&](float l) { return l > at && wt.place(l) < kNowhere; },
                                   [&](float l) -> u64 {
                                     const double x = wt.weight(l);
                                     return x >= wt.least ? fixed44(x) : 0;
                                   },
                                   at, &equal);
            // How many of the border's value a warp keeps.
            u64 eq_low;
            row.gather(equal, eq_low);
            u64 eq_at = eq_low;
            for (int i = 0; i < row.warp; ++i) eq_at += sh.warp_sum[i];
            const u64 w_at = count ? kept_weight(at) : 0;
            mine += (eq_at >= count ? 0 : min(equal, count - eq_at)) * w_at;
            if (row.lane == 0) {
              sh.equal_before[row.warp] = eq_at;
              sh.equal[row.warp] = static_cast<uint32_t>(equal);
            }
            const u64 kept = row.gather(mine, lower);
            // Within a warp's entries: those above, and of the border's value as
            // many as `count` leaves after the warps before.
            token = row.find_from(
                share_of(kept), lower,
                [&](int owner, int from, int to) {
                  const u64 n0 = sh.equal_before[owner], n1 = n0 + sh.equal[owner];
                  I = n0 >= count   ? 0
                      : n1 <= count ? 0xffffffffu
                                    : row.nth_equal(at, count - n0, from, to) + 1;
                },
                [&](float l, int i) -> u64 {
                  return l > at || (l == at && static_cast<uint32_t>(i) < I) ? kept_weight(l) : 0;
                });
            done = true;
          } else {
            for (int i = tid; i < kBins; i += kSampleThreads) row.hist[i] = 0;
            __syncthreads();
          }
        }
      }
      if (!done && (by_k || by_p)) {
        // The histogram, and where the nucleus is cut from the whole row, its
        // weight; prob's sum on the way.
        u64 s = 0;
        float terms = 0.f;
        const bool with_terms = p.prob && !one_all;
        for (int i = row.lo + 4 * row.lane; i < row.hi; i += 128) {
          float v[4];
          row.load4(i, v);
          bool t[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float at = wt.place(v[j]);
            t[j] = at < kNowhere;
            if (t[j]) atomicAdd(row.hist + wt.bin(at), 1u);
            if (with_terms) terms += row.term(v[j], m);
          }
          if (!by_k && (t[0] || t[1] || t[2] || t[3])) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const u64 w = fixed44(wt.weight(v[j]));
              s += t[j] ? w : 0;
            }
          }
        }
        u64 lower;
        u64 second = with_terms ? row.terms_total(terms) : 0;
        // (The barrier within completes the histograms.)
        const u64 all = row.gather(row.warp_total(s), lower, with_terms ? &second : nullptr);
        if (with_terms) one_all = second;
        u64 need = by_k ? static_cast<u64>(top_k) : need_of(top_p, all);
        // What the histograms say of the border: the first bin that is not before it
        // for certain and the last that is not behind it for certain, and how many
        // entries come before these two's ends. Bin i holds weights within a factor
        // `more` of 2^-(x0 + i step); entries of weight sure_w, sure_n of them, come
        // before the first bin; total_w: what all entries weigh, the histogram's
        // among them (0: not known). The first CTA joins the histograms and tells
        // the others: every CTA reading all of them cost 20 us at 32 rows of 8 CTAs.
        struct Bins {
          int lo, hi;
          uint32_t n_lo, n_hi;
        };
        auto locate = [&](double sure_w, uint32_t sure_n, double total_w, float x0, float step,
                          double more) -> Bins {
          if (row.rank == 0) {
            // Bins kBinsEach tid and on of the whole row, and what is before them.
            uint32_t own[kBinsEach];
#pragma unroll
            for (int h = 0; h < kBinsEach; ++h) own[h] = 0;
            if (tid < kBins / kBinsEach) {
#pragma unroll 4
              for (uint32_t r = 0; r < row.n_ranks; ++r) {
                uint32_t a[4];
                asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                             : "r"(map_to_rank(row.smem_addr(row.hist), r) + 4 * kBinsEach * tid)
                             : "memory");
#pragma unroll
                for (int h = 0; h < kBinsEach; ++h) own[h] += a[h];
              }
            }
            if (tid == 0) {
              sh.bin_lo = kBins;
              sh.bin_hi = 0;
              sh.n_lo = sure_n;
              sh.n_hi = sure_n;
            }
            double q = 0.0, own_q[kBinsEach];
            uint32_t n = 0;
#pragma unroll
            for (int h = 0; h < kBinsEach; ++h) {
              own_q[h] = static_cast<double>(exp2f(
                             -fmaf(static_cast<float>(kBinsEach * tid + h), step, x0))) *
                         own[h];
              q += own_q[h];
              n += own[h];
            }
            double before_q = q;
            uint32_t before_n = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double tq = __shfl_up_sync(0xffffffffu, before_q, o);
              const uint32_t tn = __shfl_up_sync(0xffffffffu, before_n, o);
              if (row.lane >= o) {
                before_q += tq;
                before_n += tn;
              }
            }
            if (row.lane == 31) {
              sh.warp_d[row.warp] = before_q;
              sh.warp_u[row.warp] = before_n;
            }
            __syncthreads();
            before_q -= q;
            before_n += sure_n - n;
            double base_q = 0.0;
#pragma unroll
            for (int w = 0; w < kSampleWarps; ++w) {
              if (w < row.warp) {
                before_q += sh.warp_d[w];
                before_n += sh.warp_u[w];
              }
              base_q += sh.warp_d[w];
            }
            const double need_w = static_cast<double>(need) * 0x1p-44, less = 1.0 / more;
#pragma unroll
            for (int h = 0; h < kBinsEach; ++h) {
              const uint32_t bin = kBinsEach * tid + h;
              const uint32_t upto_n = before_n + own[h];
              const double upto_q = before_q + own_q[h];
              if (own[h]) {
                bool sure, behind;
                if (by_k) {
                  sure = upto_n <= need;
                  behind = before_n >= need;
                } else {
                  double most = sure_w + upto_q * more, fewest = sure_w + before_q * less;
                  if (total_w > 0.0) {
                    most = fmin(most, total_w - (base_q - upto_q) * less);
                    fewest = fmax(fewest, total_w - (base_q - before_q) * more);
                  }
                  sure = most < need_w * (1 - 1e-9);
                  behind = fewest > need_w * (1 + 1e-9);
                }
                if (!sure) atomicMin(&sh.bin_lo, bin);
                if (!behind) {
                  atomicMax(&sh.bin_hi, bin);
                  atomicMax(&sh.n_hi, upto_n);
                }
                if (sure) atomicMax(&sh.n_lo, upto_n);
              }
              before_n = upto_n;
              before_q = upto_q;
            }
            __syncthreads();
            if (tid < 4 * row.n_ranks) {
              const uint32_t* from = tid & 2 ? (tid & 1 ? &sh.n_hi : &sh.n_lo)
                                             : (tid & 1 ? &sh.bin_hi : &sh.bin_lo);
              st_cluster_u32(map_to_rank(row.smem_addr(&sh.told[tid & 3]), tid >> 2), *from);
            }
          }
          cluster_sync_cta();
          return Bins{static_cast<int>(sh.told[0]), static_cast<int>(sh.told[1]), sh.told[2],
                      sh.told[3]};
        };
        const Bins bins = locate(0.0, 0, static_cast<double>(all) * 0x1p-44, 0.f,
                                 1.f / kBinsPerOctave, 1.0111);  // 2^(1/64), and roundings
        const int b_lo = bins.lo, b_hi = bins.hi;
        uint32_t n_lo = bins.n_lo, n_hi = bins.n_hi;
        // A list of every entry up to the last bin that may be kept, or of the
        // doubtful ones, found with a finer histogram of their bins where they are
        // too many; sums of whole rows otherwise.
        const bool whole = n_hi <= kList;
        bool doubt = !whole && !(by_k && by_p) && b_lo <= b_hi;
        const bool thin = by_p && wt.least > 0.0;  // min_p thins out a wide nucleus
        u64 sure_all = 0, mine = 0;
        float fine_c = 0.f, fine_0 = 0.f;  // place in the finer one
        float fine_lo = -INFINITY, fine_hi = INFINITY;
        auto fine = [&](float l) { return fmaf(l - m, -fine_c, fine_0); };
        auto kept_for_sure = [&](float l) -> u64 {
          const double w = wt.weight(l);
          return by_k && w < wt.least ? 0 : fixed44(w);  // the nucleus is cut first
        };
        if (doubt) {  // what is before the border for certain
          const float below = 8388608.f + static_cast<float>(b_lo);  // whole numbers, exact
          mine = row.part_of([&](float l) { return wt.place(l) < below; }, kept_for_sure);
          sure_all = row.gather(mine, lower);
          if (n_hi - n_lo > kList && (b_hi - b_lo + 1) * 2 >= kBins) {
            doubt = false;
          } else if (n_hi - n_lo > kList) {
            int R = 2;  // bins of one: as many as there are room for
            while ((b_hi - b_lo + 1) * 2 * R < kBins) R *= 2;
            fine_c = wt.bin_c * static_cast<float>(R);
            fine_0 = 8388608.f - static_cast<float>(b_lo * R - R / 2);
            const float to = 8388608.f + static_cast<float>(b_hi);
            for (int i = tid; i < kBins; i += kSampleThreads) row.hist[i] = 0;
            __syncthreads();
            for (int i = row.lo + 4 * row.lane; i < row.hi; i += 128) {
              float v[4];
              row.load4(i, v);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float at = wt.place(v[j]);
                if (at >= below && at <= to)
                  atomicAdd(row.hist + min(wt.bin(fmaxf(fine(v[j]), 8388608.f)),
                                           static_cast<uint32_t>(kBins - 1)), 1u);
              }
            }
            cluster_sync_cta();
            const float step = 1.f / (kBinsPerOctave * static_cast<float>(R));
            // (Weights of a nucleus' sure entries are whole here: by_k has no need of them.)
            const Bins f = locate(by_k ? 0.0 : static_cast<double>(sure_all) * 0x1p-44, n_lo, 0.0,
                                  static_cast<float>(b_lo * R - R / 2) * step, step,
                                  (1.0 + 0.35 * step) * (1.0 + 1e-5));
            n_lo = f.n_lo;
            n_hi = f.n_hi;
            fine_lo = 8388608.f + static_cast<float>(f.lo);
            fine_hi = f.hi == kBins - 1 ? INFINITY : 8388608.f + static_cast<float>(f.hi);
            doubt = f.lo <= f.hi && n_hi - n_lo <= kList;
            if (doubt) {
              mine += row.part_of(
                  [&](float l) {
                    const float at = wt.place(l);
                    return at >= below && at <= to && fmaxf(fine(l), 8388608.f) < fine_lo;
                  },
                  kept_for_sure);
              sure_all = row.gather(mine, lower);
            }
          }
        }
        if (whole || doubt) {
          const float from = 8388608.f + static_cast<float>(whole ? 0 : b_lo);
          const float to = 8388608.f + static_cast<float>(b_hi);
          const int n = row.collect([&](float l) {
            const float at = wt.place(l);
            if (!(at >= from && at <= to)) return false;
            const float x = fmaxf(fine(l), 8388608.f);
            return x >= fine_lo && x <= fine_hi;
          });
          settle(n, whole, whole ? 0 : n_lo, need, sure_all);
          cluster_sync_cta();
          if (whole) {
            token = static_cast<int>(sh.answer);
          } else {
            K = sh.border[0];
            I = sh.border[1];
            if (!thin) {
              mine += ld_cluster_u64(map_to_rank(
                  row.smem_addr(&sh.range_sum[row.rank * kSampleWarps + row.warp]), 0));
              const u64 kept = row.gather(mine, lower);
              token = row.find(
                  [&](float l, int i) -> u64 { return before(l, i) ? kept_weight(l) : 0; },
                  share_of(kept), lower);
            }
          }
          done = whole || !thin;
        } else if (b_lo > b_hi && !by_p) {
          // No bin is in doubt: the first top_k entries end with a bin, the last
          // before b_lo, or (b_lo is behind all bins) no more than those have a
          // weight.
          if (b_lo < kBins) end = 8388608.f + static_cast<float>(b_lo);
        } else {
          if (by_k) {
            uint32_t key = 0;  // the largest key that top_k entries reach
            for (int b = 31; b >= 0; --b) {
              const uint32_t t = key | (1u << b);
              if (row.total([&](float l, int) -> u64 { return key_of(l) >= t; }) >= need) key = t;
            }
            const u64 above = row.total([&](float l, int) -> u64 { return key_of(l) > key; });
            I = static_cast<uint32_t>(row.find([&](float l, int) -> u64 { return key_of(l) == key; },
                                               [&](u64) -> u64 { return need - above - 1; }));
            K = key;
          }
          if (by_p) {
            auto q = [&](float l, int i) -> u64 { return before(l, i) ? wt.fixed(l) : 0; };
            if (by_k) need = need_of(top_p, row.total(q));
            uint32_t key = 0;  // the largest key whose entries and those above weigh `need`
            for (int b = 31; b >= 0; --b) {
              const uint32_t t = key | (1u << b);
              if (row.total([&](float l, int i) -> u64 { return key_of(l) >= t ? q(l, i) : 0; }) >=
                  need)
                key = t;
            }
            const u64 above =
                row.total([&](float l, int i) -> u64 { return key_of(l) > key ? q(l, i) : 0; });
            const int last =
                row.find([&](float l, int i) -> u64 { return key_of(l) == key ? q(l, i) : 0; },
                         [&](u64) -> u64 { return need - above - 1; });
            K = key;
            I = static_cast<uint32_t>(last);
          }
        }
      }
      if (!done) {
        if (by_k || by_p)
          token = row.find(
              [&](float l, int i) -> u64 { return before(l, i) ? kept_weight(l) : 0; }, share_of);
        else {
          auto q = [&](float l, int) -> u64 { return kept_weight(l); };
          u64 terms = 0, lower;
          const u64 mine = row.part(q, m, p.prob ? &terms : nullptr);
          const u64 all = row.gather(mine, lower, p.prob ? &terms : nullptr);
          one_all = terms;
          token = row.find(q, share_of(all), lower);
        }
      }
    }
  }
  if (p.prob) {
    if (m != -INFINITY) {
      if (!one_all) {
        u64 terms, before;
        row.part([](float, int) -> u64 { return 0; }, m, &terms);
        one_all = row.gather(terms, before);
      }
      const int i = token - row.first;
      if (i >= 0 && i < len && tid == 0) {
        const float l = sizeof(T) == 4 ? reinterpret_cast<const float*>(seg)[i]
                                       : __uint_as_float(static_cast<uint32_t>(seg[i]) << 16);
        p.prob[cand] = static_cast<float>(
            (l == m ? 1.0 : static_cast<double>(expf(l - m))) / (static_cast<double>(one_all) * 0x1p-40));
      }
    } else if (tid == 0 && row.rank == 0) {
      p.prob[cand] = 0.f;
    }
  }
  if (tid == 0 && row.rank == 0) p.token[cand] = token;
  // No CTA leaves while another reads its shared memory (those reads are over).
  __syncwarp();
  cluster_arrive_relaxed();
  cluster_wait();
}

}  // namespace ca
