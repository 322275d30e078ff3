// kv8.cuh -- the 8-bit inter-step cache: quantising K/V rows as they are
// written and reading them back.
//
// K and V are held as e4m3 values with one fp32 scale for each block of T
// consecutive positions and kv head; the value held is e4m3 * scale. The
// store writes only powers of two: 2^k with the smallest k in [-64, 120] for
// which amax <= 448 * 2^k. Dividing by it is exact, so a value is rounded
// once (to e4m3, nearest even); a held row keeps its bits until its block's
// scale grows, and then loses nothing but what falls below e4m3's smallest
// step; and e4m3 * 2^k has at most 4 significant bits, so reading back as
// bf16 is exact. It replaces StepCache::store and ::gather
// (src/model/cache.rs:62-81) for a cache of half the bytes.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>

#include "sm100.cuh"

namespace ca {

constexpr int kKv8MinExp = -64, kKv8MaxExp = 120;
constexpr int kErrInvalidRow = -1;

struct Kv8View {
  uint8_t* k;        // [batch, n_total, Hkv, hd]; position stride row_stride
  uint8_t* v;
  float* k_scale;    // [batch, n_blocks, Hkv]
  float* v_scale;
  int batch, n_total, Hkv, hd;
  int T;             // positions per scale: 16, 32, 64 or 128
  int n_blocks;      // ceil(n_total / T)
  long long row_stride;
};

struct Kv8StoreParams {
  Kv8View c;
  const __nv_bfloat16* k;  // [rows, Hkv, hd]
  const __nv_bfloat16* v;
  const int* pos;          // [rows], ascending within a sequence
  const int* cu_active;    // [batch + 1] or null (na rows per sequence)
  const int* kv_len;       // [batch] or null
  int na;
  long long rows;
  int rows_per_job;
  int* err;
};

// These kernels are launched so that they may start while the kernel before
// them in the stream ends (programmatic dependent launch): until
// dependency_wait returns, which is when that kernel is complete and its
// writes are visible, they touch nothing in memory but their arguments. Each
// lets its own successor come up right away in the same manner. What the
// kernel before may have written is read with plain loads: read-only ones
// (__ldg, ld.global.nc) are defined only for data that does not change from
// the start of the kernel that reads it, and that start is before the wait.
__device__ __forceinline__ void dependency_wait() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

// Two fp32 to two e4m3 (round to nearest even, saturating, NaN kept): lo in
// the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The four e4m3 values of a word as f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) {
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(h));
  return r;
}

__device__ __forceinline__ void e4m3x4_to_f32(uint32_t w, float (&x)[4]) {
  uint32_t a, b;
  e4m3x4_to_f16(w, a, b);
  const float2 p = f16x2_to_f32(a), q = f16x2_to_f32(b);
  x[0] = p.x;
  x[1] = p.y;
  x[2] = q.x;
  x[3] = q.y;
}

// The smallest k in [lo, hi] with amax <= 448 * 2^k. 448 = 1.75 * 2^8, so
// amax = m * 2^e (1 <= m < 2) needs e - 8, or e - 7 where m > 1.75; read off
// the fp32 bits, so it is exact.
__device__ __forceinline__ int e4m3_exp(float amax, int lo, int hi) {
  if (!(amax > 0.f)) return lo;
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127;
  const int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(k, lo), hi);
}

__device__ __forceinline__ float exp2_int(int k) {  // 2^k, -126 <= k <= 127
  return __int_as_float((k + 127) << 23);
}

// Magnitudes of two bf16 into a running pair of maxima (NaN has no part).
__device__ __forceinline__ void amax_bf16x2(uint32_t& m, uint32_t w) {
  asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w & 0x7fff7fffu));
}

// The larger of such a pair, infinities as the largest finite value.
__device__ __forceinline__ float amax_of(uint32_t m) {
  const float x = fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  return fminf(x, __uint_as_float(0x7f7f0000u));
}

// Sixteen bf16 times inv as e4m3.
__device__ __forceinline__ uint4 quantise16(const uint4 (&raw)[2], float inv) {
  uint32_t o[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const uint4& v = raw[y >> 1];
    const uint32_t a = (y & 1) ? v.z : v.x, c = (y & 1) ? v.w : v.y;
    o[y] = cvt_e4m3x2(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv) |
           (cvt_e4m3x2(__uint_as_float(c << 16) * inv, __uint_as_float(c & 0xffff0000u) * inv)
            << 16);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// W warps write the rows of one (block, kv head) of K or of V: the largest
// magnitude of its new rows, the scale, the rounded rows, and, if the scale
// grew, the rows that stay. A job is rows_per_job consecutive entries of the
// active list, for one head of K or V; it takes on the blocks whose first
// active row lies among them and follows each into the next job's entries,
// so every block has exactly one writer (where a sequence's positions do not
// ascend, which is reported, a block may have two: its contents are then
// unspecified). A lane has U 16-value units (two 16-byte loads) in flight;
// where W x 32 x U units are all of the block's rows, they stay in registers
// between the maximum and the rounding.
//
// Bound by latency on a step's few rows: one warp and one unit a lane, whose
// code is short (4 rows of 4 heads x 128: 4.3 us; four units a lane took 1.8
// us more, most of it instruction fetch; 16 x 32 scattered rows of 8 x 128:
// 6.6 us). Passes over many rows: four warps, 8 units; a block after the
// other, each found through its entries, which is well short of HBM's rate (4
// x 7000 of 8192 positions, 8 x 256: 104 us, 3.3 TB/s; 8 x 3000 of 4096, 8 x
// 128, blocks of 32: 105 us, 1.4 TB/s).
template <int W, int U>
__global__ void __launch_bounds__(W == 1 ? 256 : 32 * W) kv8_store_kernel(const Kv8StoreParams p) {
  constexpr int kJobs = W == 1 ? 8 : 1;  // jobs of a CTA at a time
  dependency_wait();
  __shared__ uint32_t s_max[W];
  const int lane = threadIdx.x & 31;
  const int jt = W == 1 ? lane : threadIdx.x;  // thread of the job
  const long long first = static_cast<long long>(blockIdx.x) * kJobs + (W == 1 ? threadIdx.x >> 5 : 0);
  const int heads2 = 2 * p.c.Hkv;
  const long long jobs = (p.rows + p.rows_per_job - 1) / p.rows_per_job * heads2;
  const int T = p.c.T, hd = p.c.hd, upr = hd / 16;  // 16-value units of a row
  const unsigned magic = ((1u << 20) + upr - 1) / upr;  // u / upr for u < 2^12
  for (long long job = first; job < jobs; job += static_cast<long long>(gridDim.x) * kJobs) {
    const int hh = static_cast<int>(job % heads2);
    const bool is_v = hh >= p.c.Hkv;
    const int h = is_v ? hh - p.c.Hkv : hh;
    const __nv_bfloat16* src = is_v ? p.v : p.k;
    uint8_t* dst = is_v ? p.c.v : p.c.k;
    float* scales = is_v ? p.c.v_scale : p.c.k_scale;
    const long long job0 = job / heads2 * p.rows_per_job;
    const long long job1 = min(job0 + p.rows_per_job, p.rows);
    // Each lane looks at one entry (a job has at most 32): its sequence, where
    // that one's entries end, and whether it is its block's first.
    const long long mine = job0 + lane;
    int my_b = 0, my_pos = -1;
    long long my_end = 0;
    bool leads = false;
    if (mine < job1) {
      long long s0;
      if (p.cu_active) {
        int lo = 0, hi = p.c.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.cu_active[mid] <= mine) lo = mid;
          else hi = mid - 1;
        }
        my_b = lo;
        s0 = p.cu_active[lo];
        my_end = min(static_cast<long long>(p.cu_active[lo + 1]), p.rows);
      } else {
        my_b = static_cast<int>(mine / p.na);
        s0 = static_cast<long long>(my_b) * p.na;
        my_end = s0 + p.na;
      }
      my_pos = p.pos[mine];
      const int before = mine > s0 ? p.pos[mine - 1] : -1;
      if (my_pos < 0 || my_pos >= p.c.n_total || my_pos <= before || mine >= my_end) {
        if (p.err) atomicExch(p.err, kErrInvalidRow);
      } else {
        leads = before < 0 || before / T != my_pos / T;
      }
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, leads); todo; todo &= todo - 1u) {
      const int who = __ffs(todo) - 1;
      const long long i = job0 + who;
      const int b = __shfl_sync(0xffffffffu, my_b, who);
      const int blk = __shfl_sync(0xffffffffu, my_pos, who) / T;
      const long long s1 = __shfl_sync(0xffffffffu, my_end, who);
      // The block's entries are i .. i + n - 1 (at most T, ascending), and
      // its active positions the bits of act.
      uint32_t act[4] = {0u, 0u, 0u, 0u};
      int n = 0;
      int last = -1;
      bool more = true;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (more && c * 32 < T) {
          const long long j = i + c * 32 + lane;
          const int q = j < s1 ? p.pos[j] : -1;
          int prev = __shfl_up_sync(0xffffffffu, q, 1);
          if (lane == 0) prev = last;
          last = __shfl_sync(0xffffffffu, q, 31);
          const bool in = q >= 0 && q < p.c.n_total && q / T == blk && q > prev;
          const uint32_t ball = __ballot_sync(0xffffffffu, in);
          const int got = ball == 0xffffffffu ? 32 : __ffs(~ball) - 1;  // the run from the first
          n += got;
          more = got == 32;
          const int bit = q - blk * T;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            act[w] |= __reduce_or_sync(
                0xffffffffu, lane < got && (bit >> 5) == w ? 1u << (bit & 31) : 0u);
        }
      }
      const int in_block = min(T, p.c.n_total - blk * T);
      const int held = p.kv_len ? min(max(p.kv_len[b] - blk * T, 0), in_block) : in_block;
      bool stays = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int bits = min(max(held - 32 * w, 0), 32);
        const uint32_t want = bits == 32 ? 0xffffffffu : (1u << bits) - 1u;
        stays |= (want & ~act[w]) != 0u;
      }
      // The old scale is on its way while the rows are read.
      float* sp = scales + (static_cast<long long>(b) * p.c.n_blocks + blk) * p.c.Hkv + h;
      const float was = *sp;
      // Largest magnitude of the new rows. An infinity counts as the largest
      // finite value, a NaN not at all.
      const int units = n * upr;
      uint4 raw[U][2];
      auto row_of = [&](int u) -> int { return static_cast<int>((u * magic) >> 20); };
      auto read = [&](int u0) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int u = u0 + 32 * W * k + jt;
          raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
          if (u < units) {
            const int r = row_of(u), e = (u - r * upr) * 16;
            const uint4* from =
                reinterpret_cast<const uint4*>(src + ((i + r) * p.c.Hkv + h) * hd + e);
            raw[k][0] = from[0];
            raw[k][1] = from[1];
          }
        }
      };
      uint32_t pair = 0u;
      for (int u0 = 0; u0 < units; u0 += 32 * W * U) {
        read(u0);
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            amax_bf16x2(pair, raw[k][x].x);
            amax_bf16x2(pair, raw[k][x].y);
            amax_bf16x2(pair, raw[k][x].z);
            amax_bf16x2(pair, raw[k][x].w);
          }
      }
      uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax_of(pair)));
      if constexpr (W > 1) {
        __syncthreads();  // the last block's maxima were read
        if (lane == 0) s_max[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) top = max(top, s_max[w]);
      }
      const float need = exp2_int(e4m3_exp(__uint_as_float(top), kKv8MinExp, kKv8MaxExp));
      const bool keep = stays && was > 0.f;
      const float now = keep ? fmaxf(was, need) : need;
      __syncwarp();
      if (jt == 0) *sp = now;
      const float inv = __fdiv_rn(1.f, now);
      uint8_t* base = dst + (static_cast<long long>(b) * p.c.n_total) * p.c.row_stride +
                      static_cast<long long>(h) * hd;
      for (int u0 = 0; u0 < units; u0 += 32 * W * U) {
        if (units > 32 * W * U) read(u0);
        int to[U];  // positions, before the first store
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int u = u0 + 32 * W * k + jt;
          to[k] = u < units ? p.pos[i + row_of(u)] : 0;
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int u = u0 + 32 * W * k + jt;
          if (u < units) {
            const int r = row_of(u), e = (u - r * upr) * 16;
            *reinterpret_cast<uint4*>(base + to[k] * p.c.row_stride + e) = quantise16(raw[k], inv);
          }
        }
      }
      if (keep && now > was) {
        const float ratio = __fdiv_rn(was, now);
        for (int u = jt; u < in_block * upr; u += 32 * W) {
          const int r = row_of(u), e = (u - r * upr) * 16;
          if ((act[r >> 5] >> (r & 31)) & 1u) continue;
          uint4* at = reinterpret_cast<uint4*>(base + (static_cast<long long>(blk) * T + r) *
                                                          p.c.row_stride + e);
          const uint4 old = *at;
          uint32_t w4[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            float x[4];
            e4m3x4_to_f32(w4[y], x);
            w4[y] = cvt_e4m3x2(x[0] * ratio, x[1] * ratio) |
                    (cvt_e4m3x2(x[2] * ratio, x[3] * ratio) << 16);
          }
          *at = make_uint4(w4[0], w4[1], w4[2], w4[3]);
        }
      }
    }
  }
}

// Every position of every sequence at once (as many active rows as
// positions: in order, they can only be 0, 1, 2, ...): a block is its T rows,
// there is nothing to look up and nothing that stays. Four warps take a block
// of a kv head of K or V, 8 units a thread in flight. A block whose entries
// are not those positions is left as it was and reported. Bound by HBM: 2
// bytes read and 1 written for each value, 4 x 8192 x 8 x 256 in 62.4 us,
// 6.4 TB/s.
__global__ void __launch_bounds__(128) kv8_store_all_kernel(const Kv8StoreParams p) {
  constexpr int U = 8;
  __shared__ uint32_t s_max[4];
  dependency_wait();
  const int lane = threadIdx.x & 31;
  const int T = p.c.T, hd = p.c.hd, upr = hd / 16, heads2 = 2 * p.c.Hkv;
  const unsigned magic = ((1u << 20) + upr - 1) / upr;
  const unsigned hh = blockIdx.x % heads2;
  const int blk = blockIdx.x / heads2, b = blockIdx.y;
  const bool is_v = hh >= static_cast<unsigned>(p.c.Hkv);
  const int h = is_v ? hh - p.c.Hkv : hh;
  const int pos0 = blk * T, n = min(T, p.c.n_total - pos0);
  const long long row0 = static_cast<long long>(b) * p.c.n_total + pos0;
  const __nv_bfloat16* src = (is_v ? p.v : p.k) + (row0 * p.c.Hkv + h) * hd;
  const int src_stride = p.c.Hkv * hd;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + row0 * p.c.row_stride + static_cast<long long>(h) * hd;
  const int units = n * upr;
  uint4 raw[U][2];
  auto read = [&](int u0) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const unsigned u = u0 + 128 * k + threadIdx.x;
      raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
      if (u < static_cast<unsigned>(units)) {
        const unsigned r = (u * magic) >> 20;
        const uint4* from = reinterpret_cast<const uint4*>(
            src + static_cast<long long>(r) * src_stride + (u - r * upr) * 16);
        raw[k][0] = from[0];
        raw[k][1] = from[1];
      }
    }
  };
  uint32_t pair = 0u;
  for (int u0 = 0; u0 < units; u0 += 128 * U) {
    read(u0);
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        amax_bf16x2(pair, raw[k][x].x);
        amax_bf16x2(pair, raw[k][x].y);
        amax_bf16x2(pair, raw[k][x].z);
        amax_bf16x2(pair, raw[k][x].w);
      }
  }
  const bool bad = static_cast<int>(threadIdx.x) < n &&
                   p.pos[row0 + threadIdx.x] != pos0 + static_cast<int>(threadIdx.x);
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax_of(pair)));
  if (lane == 0) s_max[threadIdx.x >> 5] = top;
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, kErrInvalidRow);
    return;
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) top = max(top, s_max[w]);
  const int ex = e4m3_exp(__uint_as_float(top), kKv8MinExp, kKv8MaxExp);
  const float inv = exp2_int(-ex);
  if (threadIdx.x == 0)
    (is_v ? p.c.v_scale : p.c.k_scale)[(static_cast<long long>(b) * p.c.n_blocks + blk) * p.c.Hkv +
                                       h] = exp2_int(ex);
  for (int u0 = 0; u0 < units; u0 += 128 * U) {
    if (units > 128 * U) read(u0);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const unsigned u = u0 + 128 * k + threadIdx.x;
      if (u < static_cast<unsigned>(units)) {
        const unsigned r = (u * magic) >> 20;
        *reinterpret_cast<uint4*>(dst + r * p.c.row_stride + (u - r * upr) * 16) =
            quantise16(raw[k], inv);
      }
    }
  }
}

struct Kv8LoadParams {
  Kv8View c;
  void* k_out;     // [rows, Hkv, hd] bf16 or fp32, or null
  void* v_out;
  int out_f32;
  const int* pos;  // [batch, n_pos] or null (positions 0 .. n_pos - 1)
  int n_pos;
  int* err;
};

// Eight 32-bit words to a 32-byte aligned address in one store.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Rows of the cache as bf16 or fp32. A thread has 16 values of a row (one
// 16-byte load, one 32-byte store in bf16) and keeps its column from row to
// row, so that indices cost it next to nothing; U rows are in flight. Bound
// by HBM: 1 byte read and 2 (4) written for each value; 8 x 4096 x 16 x 128 in
// bf16 in 68.9 us, 5.8 TB/s.
template <int U>
__global__ void __launch_bounds__(256) kv8_load_kernel(const Kv8LoadParams p) {
  dependency_wait();
  const int upr = p.c.Hkv * p.c.hd / 16;  // 16-value units of a row
  const uint8_t* src = blockIdx.y ? p.c.v : p.c.k;
  const float* scales = blockIdx.y ? p.c.v_scale : p.c.k_scale;
  void* dst = blockIdx.y ? p.v_out : p.k_out;
  if (!dst) return;
  const int b = blockIdx.z;
  const int shift = 31 - __clz(p.c.T);
  const int rows = upr < 256 ? 256 / upr : 1;  // rows a CTA has at a time
  const int mine = upr < 256 ? static_cast<int>(threadIdx.x) / upr : 0;
  if (mine >= rows) return;
  const int* pos = p.pos ? p.pos + static_cast<long long>(b) * p.n_pos : nullptr;
  const bool v8 = (reinterpret_cast<uintptr_t>(dst) & 31u) == 0;
  const int step = rows;  // a CTA's U x rows rows lie side by side
  for (int un = upr < 256 ? static_cast<int>(threadIdx.x) - mine * upr : threadIdx.x; un < upr;
       un += 256) {
    const uint8_t* from = src + static_cast<long long>(b) * p.c.n_total * p.c.row_stride + un * 16;
    const float* sc = scales + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + un * 16 / p.c.hd;
    const long long out0 = static_cast<long long>(b) * p.n_pos * upr + un;
    for (long long at = static_cast<long long>(blockIdx.x) * U * rows + mine; at < p.n_pos;
         at += static_cast<long long>(gridDim.x) * U * rows) {
      const int i0 = static_cast<int>(at);
      int q[U];  // positions; -1: no row
      bool bad = false;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * step;
        const bool row = i < p.n_pos && i >= i0;
        q[k] = row ? (pos ? pos[i] : i) : -1;
        const bool held = q[k] >= 0 && q[k] < p.c.n_total;
        bad |= row && !held;
        q[k] = held ? q[k] : -1;
      }
      uint4 raw[U];
      float s[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (q[k] >= 0) {
          raw[k] = *reinterpret_cast<const uint4*>(from + q[k] * p.c.row_stride);
          s[k] = sc[(q[k] >> shift) * p.c.Hkv];
        }
      }
      if (bad && p.err) atomicExch(p.err, kErrInvalidRow);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (q[k] < 0) continue;
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        float x[16];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float v[4];
          e4m3x4_to_f32(w[y], v);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * y + j] = v[j] * s[k];
        }
        const long long o = (out0 + static_cast<long long>(i0 + k * step) * upr) * 16;
        if (p.out_f32) {
          float4* d = reinterpret_cast<float4*>(static_cast<float*>(dst) + o);
#pragma unroll
          for (int y = 0; y < 4; ++y)
            d[y] = make_float4(x[4 * y], x[4 * y + 1], x[4 * y + 2], x[4 * y + 3]);
        } else {
          uint32_t h[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) h[y] = pack_bf16(x[2 * y], x[2 * y + 1]);
          __nv_bfloat16* d = static_cast<__nv_bfloat16*>(dst) + o;
          if (v8) {
            st_global_v8(d, h);
          } else {
            reinterpret_cast<uint4*>(d)[0] = make_uint4(h[0], h[1], h[2], h[3]);
            reinterpret_cast<uint4*>(d)[1] = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
      }
    }
  }
}

}  // namespace ca
