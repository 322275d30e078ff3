// skinny.cuh -- act . W^T for few rows of act, alone or gated, on tcgen05.
//
//   out[t, r] = sa[t] sw[r] sum_c act[t, c] W[r, c] (+ bias[r]) (+ residual[t, r])
//   out[t, r] = f(sa[t] sg[r] act . Wg[r]) * (sa[t] su[r] act . Wu[r])
//
// The weights are the M operand: a CTA takes 128 of their rows (for the gated
// form of both matrices) and the tokens are the N columns, 16 to 64 of them,
// so one token costs the tensor core no more than 16. What bounds it is the
// weights' way from HBM: each is read once. A stage holds 128 bytes of each
// row; the ring of stages (about 100 KB, so that two CTAs share an SM) keeps
// the loads in flight. Where 128 rows a CTA would leave SMs idle, the S CTAs
// of a cluster split the columns between them. Each sends its part of a token
// to the shared memory of the CTA that finishes it, which adds the parts in
// the order of their ranks: no workspace, no atomics, the same bits every time.
//
// CHUNK > 0 (fp32 outputs of more columns than the largest split takes): as in
// pair.cuh an accumulator takes CHUNK pieces of 128 bytes at most, which the
// storing warps add up in registers while the next one fills.
//
// Lane = weight row, TMEM column = token, so that a warp's 32 threads store 32
// neighbours of an output row.
#pragma once

#include <climits>
#include <cstdint>
#include <cuda_bf16.h>

#include "cluster.cuh"
#include "sm100.cuh"

namespace ca {

constexpr int kKindBf16 = 0, kKindE4m3 = 1;

struct LinearParams {
  const float* act_scale;   // [n] or null
  const float* w_scale;     // [rows] or null
  const float* up_scale;    // gated: [rows] or null
  const float* bias;        // [rows] or null
  const void* residual;     // out's type, or null
  void* out;
  long long out_stride, res_stride;
  long long n, rows;
  int kblocks;              // 128-byte pieces of a row
  int out_f32;
  int act;                  // CA_ACT_*
  int r_tiles, t_tiles;     // pair.cuh: its tiles
  int* err;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* tmap, uint32_t bar,
                                            int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

// D[tmem] (+)= A[smem] x B[smem]^T, both K-major.
template <int KIND>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (KIND == kKindBf16) {
    umma_ss(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Instruction descriptor: e4m3 (formats 0) or bf16 operands, fp32 D.
__host__ __device__ constexpr uint32_t linear_idesc(int kind, int M, int N) {
  return kind == kKindBf16 ? umma_idesc_bf16(M, N, 0, 0)
                           : (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) |
                                 (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// The gate's activation, in fp32: g / (1 + e^-g), and with y = sqrt(2/pi) (g +
// 0.044715 g^3), 0.5 g (1 + tanh y) = g / (1 + e^-2y). Exponentials that run to
// infinity give 0. 2^(x log2 e) of a rounded product is off by 2 + 1.16 |x| units
// of 2^-23 (1e-5 at -80), which a bf16 output does not show (2e-3). For fp32 ones
// (`exact`) what the product lost, and the constant, come back as a factor: 2
// units, one for the factor and 2 for the quotient. (expf and a division took
// 2048 gated tokens 4096 -> 12288 in e4m3 from 160 to 256 us.)
__device__ __forceinline__ float activate(float g, int act, bool exact) {
  constexpr float kLog2E = 1.44269502f, kLog2ERest = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float x =
      act == 0 ? -g : -2.f * (0.7978845608028654f * (g + 0.044715f * g * g * g));
  float e = ex2_approx(x * kLog2E);
  if (exact) {
    const float c = fminf(fmaxf(x, -200.f), 200.f);  // (beyond, e is 0 or infinite)
    const float lost = fmaf(c, kLog2ERest, fmaf(c, kLog2E, -(c * kLog2E)));
    e *= fmaf(lost, kLn2, 1.f);
  }
  return __fdividef(g, 1.f + e);
}

// A sum times its two scales, a token's and a row's, the smaller one first: it is
// out of range in between only where the result is (rows quantised at 2^100 and
// more times weights of 2^-10 are finite). No operand's scale from ca_rms_norm
// takes a sum below the normal numbers.
__device__ __forceinline__ float scaled(float a, float s, float w) {
  const bool first = fabsf(s) < fabsf(w);
  return a * (first ? s : w) * (first ? w : s);
}

// How many of the N tokens from t on have an element r of their own.
template <int N>
__device__ __forceinline__ int tokens_in(const LinearParams& p, long long t, bool ok) {
  return ok ? static_cast<int>(max(0ll, min(static_cast<long long>(N), p.n - t))) : 0;
}

// The residual's element r of the first m of N tokens from t on. Loads without
// conditions (tokens behind the m-th read the m-th's), so that all N are on
// their way before the first is waited for.
template <int N>
__device__ __forceinline__ void load_residual(const LinearParams& p, float (&x)[N], long long t,
                                              long long r, int m) {
  if (m <= 0) return;
  if (p.out_f32) {
    const float* s = static_cast<const float*>(p.residual) + t * p.res_stride + r;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = s[min(j, m - 1) * p.res_stride];
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(p.residual) + t * p.res_stride + r;
    uint16_t raw[N];
#pragma unroll
    for (int j = 0; j < N; ++j) raw[j] = s[min(j, m - 1) * p.res_stride];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __uint_as_float(static_cast<uint32_t>(raw[j]) << 16);
  }
}

// Element r of the first m of N tokens from t on, rounded once.
template <int N>
__device__ __forceinline__ void store_tokens(const LinearParams& p, const float (&v)[N],
                                             long long t, long long r, int m) {
  if (p.out_f32) {
    float* o = static_cast<float*>(p.out) + t * p.out_stride + r;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < m) o[j * p.out_stride] = v[j];
  } else {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + t * p.out_stride + r;
    if (m == N) {
#pragma unroll
      for (int j = 0; j < N; ++j) o[j * p.out_stride] = __float2bfloat16_rn(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < m) o[j * p.out_stride] = __float2bfloat16_rn(v[j]);
    }
  }
}

// The scales of tokens t .. t + 31, one a lane.
__device__ __forceinline__ float act_scale_of(const LinearParams& p, long long t) {
  return p.act_scale && t < p.n ? p.act_scale[t] : 1.f;
}

template <int KIND_, int G_, int NT_, int CHUNK_ = 0>
struct SkinnyCfg {
  static constexpr int CHUNK = CHUNK_;
  static constexpr int KIND = KIND_;  // operands
  static constexpr int G = G_;        // weight matrices
  static constexpr int NT = NT_;      // tokens of a CTA
  static constexpr int kStage = G * 16384 + NT * 128;
  static constexpr int kParts = G * NT * 512;  // of a sum, from every rank
  // Few tokens' parts have memory of their own, so that they can be sent while
  // another CTA still multiplies; more lie over the ring.
  static constexpr bool kApart = kParts <= 16384;
  static constexpr int kStages = (104 * 1024 - (kApart ? kParts : 0)) / kStage;
  static constexpr int kRing = kStages * kStage;
  static_assert(kApart || kRing >= kParts, "the parts of a sum are laid over the ring");
  static constexpr int kThreads = 192;
  static constexpr int kBufs = CHUNK > 0 ? 2 : 1;  // accumulators
  static constexpr int kBars = 2 * kStages + 2 * kBufs;
  static constexpr int kSmem = 1024 + kRing + (kApart ? kParts : 0) + 8 * kBars + 16;
  static constexpr int kBuf = G * NT;  // TMEM columns of an accumulator
  static constexpr int kTmemCols = kBufs * kBuf < 32 ? 32 : kBufs * kBuf;
  static_assert(kTmemCols <= 256, "two CTAs share an SM");
  static constexpr int kElems = KIND == kKindBf16 ? 64 : 128;  // of 128 bytes
};

// CHUNK: two CTAs an SM (168 registers, with 84 bytes of spills at 64 tokens of
// two matrices, which would take 175: gated, 64 tokens 18944 -> 4096 in bf16 43
// us, one CTA an SM 91).
template <class C>
__global__ void __launch_bounds__(C::kThreads, C::CHUNK > 0 ? 2 : 0)
    skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_u,
                  const __grid_constant__ CUtensorMap tm_x, const LinearParams p) {
  extern __shared__ uint8_t raw_smem[];
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  const uint32_t parts = C::kApart ? base + C::kRing : base;
  const uint32_t bars = base + C::kRing + (C::kApart ? C::kParts : 0);
  const uint32_t slot = bars + 8 * C::kBars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (C::kStages + s); };
  auto acc_full = [&](int b) { return bars + 8 * (2 * C::kStages + b); };
  auto acc_empty = [&](int b) { return bars + 8 * (2 * C::kStages + C::kBufs + b); };
  const uint32_t S = cluster_size(), rank = cluster_rank();
  const int r0 = static_cast<int>(blockIdx.x / S) * 128;
  const int t0 = static_cast<int>(blockIdx.y) * C::NT;
  const int kb0 = static_cast<int>(static_cast<long long>(p.kblocks) * rank / S);
  const int kb1 = static_cast<int>(static_cast<long long>(p.kblocks) * (rank + 1) / S);

  bool dead = false;
  int filled = 0;  // stages, by the loading thread
  auto fill = [&](int i) {
    const int s = i % C::kStages, x = (kb0 + i) * C::kElems;
    const uint32_t dst = base + s * C::kStage;
    mbar_arrive_expect_tx(full(s), C::kStage);
    tma_load_2d(dst, &tm_w, full(s), x, r0);
    if constexpr (C::G == 2) tma_load_2d(dst + 16384, &tm_u, full(s), x, r0);
    tma_load_2d(dst + C::G * 16384, &tm_x, full(s), x, t0);
  };
  if (tid == 0) {
    tma_prefetch_desc(&tm_w);
    if constexpr (C::G == 2) tma_prefetch_desc(&tm_u);
    tma_prefetch_desc(&tm_x);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < C::kBufs; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  cluster_arrive_relaxed();  // (waited for before anything is written to another CTA)
  // TMEM is taken only once the kernel before is complete, and the next one
  // let in only then: neither can hold columns that the other waits for. The
  // first loads need no TMEM.
  wait_prior_kernel();
  if (tid == 0)
    for (; filled < min(C::kStages, kb1 - kb0); ++filled) fill(filled);
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_kernel();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  if (warp == 0) {
    if (lane == 0) {
      for (; filled < kb1 - kb0; ++filled) {
        if (!mbar_wait(empty(filled % C::kStages), ((filled / C::kStages) - 1) & 1, dead, p.err))
          break;
        fill(filled);
      }
      // After an expired wait the copies in flight still have to land.
      if (dead) {
        bool late = false;
        for (int j = max(0, filled - C::kStages); j < filled; ++j)
          mbar_wait(full(j % C::kStages), (j / C::kStages) & 1, late, p.err);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = linear_idesc(C::KIND, 128, C::NT);
      constexpr int kChunk = C::CHUNK > 0 ? C::CHUNK : INT_MAX;
      int i = 0, n = 0, in = 0;  // pieces taken; accumulators filled; pieces in this one
      uint32_t acc = tmem;
      for (int kb = kb0; kb < kb1; ++kb, ++i, ++in) {
        if (in == kChunk) {
          umma_commit(acc_full(n++ & 1));
          in = 0;
          if (n >= 2 && !mbar_wait(acc_empty(n & 1), ((n >> 1) - 1) & 1, dead, p.err)) break;
          tc_fence_after();
          acc = tmem + (n & 1) * C::kBuf;
        }
        const int s = i % C::kStages;
        if (!mbar_wait(full(s), (i / C::kStages) & 1, dead, p.err)) break;
        tc_fence_after();
        const uint32_t at = base + s * C::kStage;
        const uint64_t dw = umma_desc_sw128(at, 16, 1024);
        const uint64_t dx = umma_desc_sw128(at + C::G * 16384, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          mma_ss<C::KIND>(acc, dw + 2 * kk, dx + 2 * kk, idesc, in | kk);
          if constexpr (C::G == 2)
            mma_ss<C::KIND>(acc + C::NT, dw + 1024 + 2 * kk, dx + 2 * kk, idesc, in | kk);
        }
        umma_commit(empty(s));
      }
      umma_commit(acc_full(n & 1));
    }
    __syncwarp();
  }

  // Warps 2 to 5: lanes 32 (warp % 4) .. + 31 of TMEM, a weight row each.
  const int f = (warp & 3) * 32 + lane;
  const long long r = r0 + f;
  float w0 = 1.f, w1 = 1.f, bias = 0.f;
  auto combine = [&](float a, float b, float sa) {
    const float s = scaled(a, sa, w0);
    return C::G == 2 ? activate(s, p.act, p.out_f32) * scaled(b, sa, w1) : s + bias;
  };
  const int live = static_cast<int>(min(static_cast<long long>(C::NT), p.n - t0));  // tokens
  const int each = C::NT / static_cast<int>(S);  // tokens that a rank finishes, from `first` on
  const int shift = 31 - __clz(each);            // (a power of two)
  const int first = each * static_cast<int>(rank), mine = max(0, min(each, live - first));
  const bool on = warp >= 2 && r < p.rows;
  // Residuals of its first tokens are asked for before the wait: a row's
  // latency each time was most of what 64 tokens took (4 us of 15 without
  // splits, 11 of 19 with two).
  constexpr int kGroup = C::NT < 32 ? C::NT : 32;
  float x[kGroup];
  if (C::G == 1 && on && p.residual) load_residual(p, x, t0 + first, r, mine);
  const uint32_t col = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  float v0[C::CHUNK > 0 ? C::NT : 1], v1[C::CHUNK > 0 && C::G == 2 ? C::NT : 1];  // CHUNK's sums
  if (warp >= 2) {
    if (r < p.rows) {
      if (p.w_scale) w0 = p.w_scale[r];
      if (C::G == 2 && p.up_scale) w1 = p.up_scale[r];
      if (C::G == 1 && p.bias) bias = p.bias[r];
    }
    if constexpr (C::CHUNK == 0) {
      mbar_wait(acc_full(0), 0, dead, p.err);
      __syncwarp();
      tc_fence_after();
    } else {
#pragma unroll
      for (int j = 0; j < C::NT; ++j) {
        v0[j] = 0.f;
        if constexpr (C::G == 2) v1[j] = 0.f;
      }
      for (int n = 0; n * C::CHUNK < kb1 - kb0; ++n) {
        mbar_wait(acc_full(n & 1), (n >> 1) & 1, dead, p.err);
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int j0 = 0; j0 < C::NT; j0 += 16) {
          uint32_t d0[16], d1[16];
          tmem_ld16(col + (n & 1) * C::kBuf + j0, d0);
          if constexpr (C::G == 2) tmem_ld16(col + (n & 1) * C::kBuf + C::NT + j0, d1);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            v0[j0 + j] += __uint_as_float(d0[j]);
            if constexpr (C::G == 2) v1[j0 + j] += __uint_as_float(d1[j]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(n & 1));
      }
    }
  }
  __syncwarp();
  cluster_wait();                               // every CTA of the cluster has started
  if (S > 1 && !C::kApart) cluster_sync_all();  // every ring is free
  if (warp >= 2) {
#pragma unroll
    for (int j0 = 0; j0 < C::NT; j0 += 16) {
      if (j0 >= live) break;
      uint32_t d0[16], d1[16];
      if constexpr (C::CHUNK == 0) {
        tmem_ld16(col + j0, d0);
        if constexpr (C::G == 2) tmem_ld16(col + C::NT + j0, d1);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          d0[j] = __float_as_uint(v0[j0 + j]);
          if constexpr (C::G == 2) d1[j] = __float_as_uint(v1[j0 + j]);
        }
      }
      const float sa = act_scale_of(p, t0 + j0 + (lane & 15));
      if constexpr (C::CHUNK == 0) tmem_wait_ld();
      if (S == 1) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = combine(__uint_as_float(d0[j]), C::G == 2 ? __uint_as_float(d1[j]) : 0.f,
                         __shfl_sync(0xffffffffu, sa, j));
          if (C::G == 1 && p.residual) v[j] += x[j0 % kGroup + j];
        }
        store_tokens(p, v, t0 + j0, r, tokens_in<16>(p, t0 + j0, r < p.rows));
        // (out may be the residual: the next ones are not asked for earlier.)
        if (C::G == 1 && p.residual && on && (j0 + 16) % kGroup == 0 && j0 + 16 < C::NT)
          load_residual(p, x, t0 + j0 + 16, r, live - j0 - 16);
      } else {
        // Token j goes to rank j / each, place (this rank, j % each).
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j0 + j < live) {
            const int to = (j0 + j) >> shift, k = (j0 + j) & (each - 1);
            const uint32_t at = map_to_rank(
                parts + ((static_cast<int>(rank) * each + k) * C::G * 128 + f) * 4, to);
            st_cluster_f32(at, __uint_as_float(d0[j]));
            if constexpr (C::G == 2) st_cluster_f32(at + 512, __uint_as_float(d1[j]));
          }
        }
      }
    }
    tc_fence_before();
  }
  if (S > 1) {
    __syncwarp();
    cluster_sync_all();
    if (on) {
#pragma unroll
      for (int j0 = 0; j0 < (C::NT < 32 ? C::NT : 32); j0 += 4) {  // two ranks: 32 tokens each
        if (j0 >= mine) break;
        const int k = min(mine - j0, 4);
        float d[2][4] = {};
        for (int q = 0; q < static_cast<int>(S); ++q) {
          const uint32_t at = parts + ((q * each + j0) * C::G * 128 + f) * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int g = 0; g < C::G; ++g) {
              float t = 0.f;
              if (j < k)
                asm volatile("ld.shared.f32 %0, [%1];"
                             : "=f"(t) : "r"(at + (j * C::G + g) * 512) : "memory");
              d[g][j] += t;
            }
          }
        }
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float sa = j < k && p.act_scale ? p.act_scale[t0 + first + j0 + j] : 1.f;
          v[j] = combine(d[0][j], d[1][j], sa);
          if (C::G == 1 && p.residual) v[j] += x[j0 + j];
        }
        store_tokens(p, v, t0 + first + j0, r, k);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

}  // namespace ca
