// attn_kv8_tile.cuh -- attention of many query rows over the 8-bit cache on
// the fifth-generation tensor cores.
//
// One CTA takes 128 query rows (token, head-of-the-group pairs, token-major)
// of one (sequence, kv head) and one stretch of its key tiles. Mathematics
// and the treatment of the scales are those of attn_kv8_rows.cuh:
//   t = a (q . k8) + L,   p = 2^(t - m),   out = sum p v8 / sum p 2^-L.
//
// S = Q K^T runs on K as it is held (kind::f8f6f4, e4m3 x e4m3, fp32
// accumulators): each row of Q is scaled by a power of two into e4m3's range
// and split into two e4m3 terms, q = hi + lo, whose products land in the same
// accumulator. Two terms of 4 significant bits hold bf16's 8 exactly, down to
// 2^-18 of the row's largest value. The two e4m3 products cost the tensor
// core what one bf16 product would, and K needs no conversion. P V cannot do
// the same: a weight's range (2^-31 .. 1 counts in a long row) does not fit
// two e4m3 terms, so P is f16 (11 bits, in TMEM over S) and V is turned into
// f16 in shared memory by four warps of its own, which keep out of the
// softmax warps' issue slots.
//
// Warp roles (one CTA per SM):
//   warp 0       K tiles, TMA into a ring (lane 0)
//   warp 1       TMEM, tcgen05.mma issue (lane 0)
//   warp 2       V tiles, TMA into a ring (lane 0)
//   warps 4-11   softmax
//   warps 12-15  V tile -> f16
// head_dim <= 128: tiles of 128 keys; two groups of four softmax warps take
// alternate tiles, a row a thread, each group with an S and an O of its own,
// merged at the end; P takes S's place (two O's leave no TMEM for both), and
// P V of a tile's first 64 keys starts while the others are exponentiated.
// head_dim 256: tiles of 64 keys, one group of eight warps, two to a row
// (they exchange row maxima through shared memory and a barrier of their
// own), one O; P has columns of its own, so S runs two tiles ahead.
//
// Bound, measured on B200: 2 sequences x 4096 x 4096, 16 heads of 128: 320 us,
// 860 TFLOP/s in runs of half a second (296 us, 929 TFLOP/s in runs of
// milliseconds, at a higher clock; tensor pipe busy 44%): the chain S -> TMEM
// load -> maximum -> exponentials -> TMEM store -> P V of a group, about 4100
// clocks for 128 keys, two groups in turn; P V and S are 1072 of them. 16 x 32
// queries over 4128 positions, 32/8 heads: 54 us (51 in short runs). head_dim
// 256, window 512, soft-cap, 2048 rows: 76 us, about 2900 clocks a 64-key
// tile. Small tiles lose to their fixed part, exponentials on the FMA pipe to
// their issue slots.
#pragma once

#include <cfloat>

#include "attn_kv8_rows.cuh"

namespace ca {

// CAPPED: the soft-cap's arithmetic (a kernel of its own: the softmax loop is
// long, and instruction fetch is some of its time).
template <int HDP_, int CH_, bool CAPPED_>
struct TileCfg {
  static constexpr int HDP = HDP_;                       // 64, 128 or 256
  static constexpr bool CAPPED = CAPPED_;
  static constexpr int CH = CH_;                         // warps that share 32 rows of a tile
  static constexpr int TG = HDP <= 128 ? 2 : 1;          // tile groups, each with its own O
  static constexpr int BN = TG == 2 ? 128 : 64;          // keys of a tile
  // P has TMEM columns of its own (one group), or takes S's place (two: their
  // two O's leave no room).
  static constexpr bool PSEP = TG == 1;
  // P V of a tile's first half starts while the second is exponentiated.
  static constexpr bool HALVES = TG == 2 && CH == 1;
  static constexpr int SC = BN / CH;                     // keys of a softmax thread's part
  static constexpr int kSoftWarps = 4 * TG * CH;
  static constexpr int kSoftThreads = 32 * kSoftWarps;
  static constexpr int kThreads = 256 + kSoftThreads;
  static constexpr int kConvWarp0 = 4 + kSoftWarps;
  // Stages of K and V as held (V in f16 has two).
  static constexpr int STK = 3, STV = 2;
  static constexpr int kChunks = (HDP + 127) / 128;      // 128-byte columns of an e4m3 tile
  static constexpr int kSteps = HDP / 32;                // k-steps of S
  static constexpr int kQTerm = kChunks * 128 * 128;     // one term of Q
  static constexpr int kTile8 = kChunks * BN * 128;      // K or V as held
  static constexpr int kVAtoms = HDP / 64;               // 64-column atoms of V in f16
  static constexpr int kTile16 = kVAtoms * BN * 128;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + 2 * kQTerm;
  static constexpr int kOffV8 = kOffK + STK * kTile8;
  static constexpr int kOffV = kOffV8 + STV * kTile8;
  static constexpr int kOffBar = kOffV + 2 * kTile16;
  static constexpr int kBarK = 0;               // [STK] K landed
  static constexpr int kBarKE = kBarK + STK;    // [STK] K free
  static constexpr int kBarV8 = kBarKE + STK;   // [STV] V landed
  static constexpr int kBarV8E = kBarV8 + STV;  // [STV] V free
  static constexpr int kBarS = kBarV8E + STV;   // [2] S of an (even, odd) tile
  static constexpr int kBarSE = kBarS + 2;      // [2] read
  static constexpr int kBarP = kBarSE + 2;      // [2] P (its first half) written and V in f16
  static constexpr int kBarP2 = kBarP + 2;      // [2] P's second half
  static constexpr int kBarO = kBarP2 + 2;      // [2] P V done
  static constexpr int kBarF = kBarO + 2;       // every MMA done
  static constexpr int kNumBars = kBarF + 1;
  static constexpr int kOffQs = kOffBar + (kNumBars * 8 + 15) / 16 * 16;  // float [128]
  static constexpr int kOffXch = kOffQs + 128 * 4;       // float [TG CH][2][128]
  static constexpr int kOffSc = kOffXch + TG * CH * 2 * 128 * 4;  // float [warp][2][3][NC]
  static constexpr int NC = SC / 16;                     // 16-key pieces of a part
  static constexpr int kOffRow = kOffSc + kSoftWarps * 2 * 3 * NC * 4;  // int64 [128]
  static constexpr int kOffMisc = kOffRow + 128 * 8;
  static constexpr int kSmem = kOffMisc + 64;
  // TMEM: S of two tiles, P, O.
  static constexpr int kPCol = PSEP ? 2 * BN : 0;        // P of an (even, odd) tile
  static constexpr int kPStep = PSEP ? 8 : 16;           // columns of 16 keys
  static constexpr int kOCol = PSEP ? 3 * BN : 2 * BN;
  // Registers (CH 1, two groups: 512 threads launched with 128 each): two
  // warpgroups with whole rows of 128 keys at 200, the other two at 56, are
  // those 4 x 128. (192 and 64: 3% slower; 208 and 48: no different.)
  static constexpr int kSoftRegs = 200, kOtherRegs = 56;
  static constexpr bool REGS = SC == 128;
  static constexpr int kRegsAsked =
      kSoftThreads * kSoftRegs + (kThreads - kSoftThreads) * kOtherRegs;
  static constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(BN >> 3) << 17) |
                                      (128u >> 4 << 24);  // e4m3 x e4m3, fp32
  static constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) |
                                      (static_cast<uint32_t>(HDP >> 3) << 17) |
                                      (128u >> 4 << 24);  // f16 x f16 (MN-major), fp32
  static_assert(kOCol + TG * HDP <= 512, "TMEM");
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static constexpr int kRings = STK * kTile8 + STV * kTile8;
  static_assert(kSoftWarps * 4096 <= kRings, "output staging");
  static constexpr int kMaxSplits = kRings / 512;  // a join's weights: float [splits][128]
  static_assert(kMaxSplits >= 148, "weights of a join");
};

// D[tmem] (+)= A[smem] x B[smem]^T, kind::f8f6f4 (e4m3 in, fp32 accumulate).
__device__ __forceinline__ void umma_ss_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
    attn_kv8_tile_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const Kv8AttnParams p) {
  constexpr int BN = C::BN, HDP = C::HDP, SC = C::SC;
  constexpr int TG = C::TG, CH = C::CH;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicExch(p.err ? p.err : &g_device_error, kErrLayout);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int hd = p.c.hd;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  dependency_wait();
  const int q_beg = p.cu_q ? p.cu_q[b] : b * p.sq;
  const int q_len = p.cu_q ? p.cu_q[b + 1] - q_beg : p.sq;
  const long long n_rows = static_cast<long long>(q_len) * p.G;
  const long long row0 = static_cast<long long>(tile) * 128;
  if (row0 >= n_rows) return;
  const int rows = static_cast<int>(min(128ll, n_rows - row0));
  const int len = p.kv_len ? min(max(p.kv_len[b], 0), p.c.n_total) : p.c.n_total;
  const int prefix = p.seq_prefix ? p.seq_prefix[b] : p.causal_prefix;

  const uint32_t sQ = smem_u32(smem + C::kOffQ);
  const uint32_t sK = smem_u32(smem + C::kOffK);
  const uint32_t sV8 = smem_u32(smem + C::kOffV8);
  const uint32_t sV = smem_u32(smem + C::kOffV);
  const uint32_t bar0 = smem_u32(smem + C::kOffBar);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * i; };
  float* sQs = reinterpret_cast<float*>(smem + C::kOffQs);
  int* misc = reinterpret_cast<int*>(smem + C::kOffMisc);  // [0] TMEM, [1..4] key ranges, [5] join

  const bool masked = p.window != kNoWindow || prefix >= 0;
  auto interval = [&](int r, int& lo, int& hi) {
    lo = 0;
    hi = len;
    if (!masked) return;
    const int tok = static_cast<int>((row0 + r) / p.G);
    const int pos = p.q_pos ? p.q_pos[q_beg + tok] : len - q_len + tok;
    kv8_interval(pos, len, p.window, prefix, lo, hi);
  };
  const int tok0 = b * p.c.n_total;  // the sequence's first row of the tensor maps

  // Warps 0, 2 and 3 find the keys: the hull of what the rows see, what
  // every row sees, and this CTA's tiles kt0 .. kt0 + n - 1. The producers
  // set up their own barriers and ask for their first tiles at once, while
  // warps 4-11 split Q.
  int k_lo = 0, k_hi = 0, f_lo = 0, f_hi = 0, kt0 = 0, n = 0;
  auto find_keys = [&]() {
    k_lo = 0;
    k_hi = f_hi = len;
    f_lo = 0;
    if (masked) {
      k_lo = f_hi = INT_MAX;
      k_hi = 0;
      for (int r = lane; r < rows; r += 32) {
        int lo, hi;
        interval(r, lo, hi);
        if (lo < hi) {
          k_lo = min(k_lo, lo);
          k_hi = max(k_hi, hi);
        }
        f_lo = max(f_lo, lo);
        f_hi = min(f_hi, hi);
      }
      k_lo = __reduce_min_sync(0xffffffffu, k_lo);
      k_hi = __reduce_max_sync(0xffffffffu, k_hi);
      f_lo = __reduce_max_sync(0xffffffffu, f_lo);
      f_hi = __reduce_min_sync(0xffffffffu, f_hi);
    }
    if (k_lo < k_hi) {
      const int first = k_lo / BN, all = (k_hi + BN - 1) / BN - first;
      const int per = (all + p.splits - 1) / p.splits;
      kt0 = first + min(all, split * per);
      n = first + min(all, (split + 1) * per) - kt0;
    }
  };
  auto load_tile = [&](const CUtensorMap* tm, uint32_t base, int full, int u, int s) {
    mbar_arrive_expect_tx(bar(full + s), C::kTile8);
#pragma unroll
    for (int c = 0; c < C::kChunks; ++c)
      tma_load_3d(base + s * C::kTile8 + c * BN * 128, tm, bar(full + s), c * 128, kvh,
                  tok0 + (kt0 + u) * BN);
  };
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < C::STK; ++s) {
        mbar_init(bar(C::kBarK + s), 1);
        mbar_init(bar(C::kBarKE + s), 1);
      }
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    find_keys();
    if (lane == 0 && n > 0) load_tile(&tm_k, sK, C::kBarK, 0, 0);
  } else if (warp == 2) {
    if (lane == 0) {
      for (int s = 0; s < C::STV; ++s) {
        mbar_init(bar(C::kBarV8 + s), 1);
        mbar_init(bar(C::kBarV8E + s), 4);
      }
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    find_keys();
    if (lane == 0 && n > 0) load_tile(&tm_v, sV8, C::kBarV8, 0, 0);
  } else if (warp == 3) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(bar(C::kBarS + s), 1);
        mbar_init(bar(C::kBarSE + s), 4 * CH);
        mbar_init(bar(C::kBarP + s), 4 * CH + 4);
        mbar_init(bar(C::kBarP2 + s), 4 * CH);
        mbar_init(bar(C::kBarO + s), 1);
      }
      mbar_init(bar(C::kBarF), 1);
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    find_keys();
    if (lane == 0) {
      misc[1] = k_lo;
      misc[2] = k_hi;
      misc[3] = f_lo;
      misc[4] = f_hi;
      misc[6] = kt0;
      misc[7] = n;
    }
  } else if (warp == 1) {
    tmem_alloc(smem_u32(misc), 512);
    tmem_relinquish();
  } else if (warp < 12) {
    // Q into its two terms: a lane takes 16 values, HDP / 16 lanes a row.
    constexpr int LPR = HDP / 16, RPW = 32 / LPR, NP = 128 / (8 * RPW);
    constexpr int NB = NP < 8 ? NP : 8;  // rows a lane has in flight
    const int un = lane % LPR, e = un * 16;
#pragma unroll 1
    for (int p0 = 0; p0 < NP; p0 += NB) {
      uint4 raw[NB][2];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int qr = ((p0 + i) * 8 + warp - 4) * RPW + lane / LPR;
        raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
        if (qr < rows && e < hd) {
          const unsigned rr = static_cast<unsigned>(row0 + qr);  // < 2^31 (checked on the host)
          const unsigned tok = rr / static_cast<unsigned>(p.G);
          const uint4* src = reinterpret_cast<const uint4*>(
              p.q + (q_beg + static_cast<long long>(tok)) * p.q_row_stride +
              (kvh * p.G + static_cast<int>(rr - tok * p.G)) * static_cast<long long>(hd) + e);
          raw[i][0] = src[0];
          raw[i][1] = src[1];
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int qr = ((p0 + i) * 8 + warp - 4) * RPW + lane / LPR;
        const uint32_t w8[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                                raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          amax = fmax3(amax, fabsf(__uint_as_float(w8[k] << 16)),
                       fabsf(__uint_as_float(w8[k] & 0xffff0000u)));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1)
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int ex = e4m3_exp(fminf(amax, __uint_as_float(0x7f7f0000u)), -120, 120);
        // A negative scale turns Q's sign, so that the scores' factor is not.
        const float inv = p.scale < 0.f ? -exp2_int(-ex) : exp2_int(-ex);
        // A row with an infinity has scores that are none: NaN comes out.
        if (un == 0) sQs[qr] = amax == INFINITY ? INFINITY : exp2_int(ex);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x[4] = {__uint_as_float(w8[2 * k] << 16) * inv,
                              __uint_as_float(w8[2 * k] & 0xffff0000u) * inv,
                              __uint_as_float(w8[2 * k + 1] << 16) * inv,
                              __uint_as_float(w8[2 * k + 1] & 0xffff0000u) * inv};
          split_e4m3(x, hi[k], lo[k]);
        }
        const uint32_t at = sQ + (un >> 3) * 128 * 128 + qr * 128 + (((un & 7) ^ (qr & 7)) << 4);
        st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
        st_shared_v4(at + C::kQTerm, lo[0], lo[1], lo[2], lo[3]);
      }
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(misc[0]);
  k_lo = misc[1];
  k_hi = misc[2];
  f_lo = misc[3];
  f_hi = misc[4];
  kt0 = misc[6];
  n = misc[7];
  bool dead = false;

  if (warp < 4) {
    if constexpr (C::REGS) reg_dec<C::kOtherRegs>();
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------- producers
      if (lane == 0) {
        const bool is_k = warp == 0;
        const int full = is_k ? C::kBarK : C::kBarV8;
        const int empty = is_k ? C::kBarKE : C::kBarV8E;
        const int NS = is_k ? C::STK : C::STV;
        // The first tiles were asked for before Q; the rest of the rings only
        // now, so as not to stand in Q's way.
        int u = 1;
        for (; u < n; ++u) {
          const int s = u % NS;
          if (u >= NS && !mbar_wait(bar(empty + s), ((u / NS) - 1) & 1, dead, p.err)) break;
          load_tile(is_k ? &tm_k : &tm_v, is_k ? sK : sV8, full, u, s);
        }
        // Leave no copy in flight: those of the last tiles asked for.
        const int end = n > 0 ? u : 0;
        bool d2 = false;
        for (int w = max(0, end - NS); w < end; ++w)
          mbar_wait(bar(full + w % NS), (w / NS) & 1, d2, p.err);
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------- MMA issue
      // One thread: an issuing thread is held while its MMAs run, and two (S
      // from one, P V from another) interleave them, so that both of a pair
      // end late: a 2 x 4096 canvas took 5% longer that way. A descriptor's
      // address field counts 16-byte units: offsets add.
      const uint64_t dq = umma_desc_sw128(sQ, 16, 1024), dk0 = umma_desc_sw128(sK, 16, 1024);
      const uint64_t dv0 = umma_desc_sw128(sV, BN * 128, 1024);
      auto issue_s = [&](int j) -> bool {
        const int s = j % C::STK, x = j & 1;
        if (!mbar_wait(bar(C::kBarK + s), (j / C::STK) & 1, dead, p.err)) return false;
        // The buffer is free once S[j - 2] was read (or, with P in its place,
        // once P V[j - 2] is done).
        if (j >= 2 &&
            !mbar_wait(bar((C::PSEP ? C::kBarSE : C::kBarO) + x), ((j >> 1) - 1) & 1, dead, p.err))
          return false;
        tc_fence_after();
        const uint64_t dk = dk0 + s * (C::kTile8 >> 4);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int kk = 0; kk < C::kSteps; ++kk)
            umma_ss_f8(tmem + x * BN,
                       dq + ((term * C::kQTerm + (kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4),
                       dk + (((kk >> 2) * BN * 128 + (kk & 3) * 32) >> 4), C::kIdescS,
                       term + kk > 0 ? 1u : 0u);
        umma_commit(bar(C::kBarS + x));
        return true;
      };
      auto issue_pv = [&](int j) -> bool {
        const int x = j & 1;
        if (!mbar_wait(bar(C::kBarP + x), (j >> 1) & 1, dead, p.err)) return false;
        tc_fence_after();
        const uint64_t dv = dv0 + x * (C::kTile16 >> 4);
        const uint32_t pcol = tmem + C::kPCol + x * (BN / 16 * C::kPStep);
        const uint32_t dst = tmem + C::kOCol + (TG == 2 ? x * HDP : 0);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {
          if (C::HALVES && kk == BN / 32) {
            if (!mbar_wait(bar(C::kBarP2 + x), (j >> 1) & 1, dead, p.err)) return false;
            tc_fence_after();
          }
          umma_ts(dst, pcol + kk * C::kPStep, dv + ((kk * 2048) >> 4), C::kIdescO,
                  j >= TG || kk > 0 ? 1u : 0u);
        }
        umma_commit(bar(C::kBarO + x));
        return true;
      };
      bool ok = n > 0 && issue_s(0) && (n < 2 || issue_s(1));
      for (int j = 0; ok && j < n; ++j) {
        if (C::PSEP) ok = (j + 2 >= n || issue_s(j + 2)) && issue_pv(j);
        else ok = issue_pv(j) && (j + 2 >= n || issue_s(j + 2));
      }
      // Every MMA issued is done before the role ends.
      umma_commit(bar(C::kBarF));
      bool d2 = false;
      mbar_wait(bar(C::kBarF), 0, d2, p.err);
    }
  } else if (warp >= C::kConvWarp0) {
    // ------------------------------------------------------------ V to f16
    if constexpr (C::REGS) reg_dec<C::kOtherRegs>();
    const int cw = warp - C::kConvWarp0;
    constexpr int UPR = HDP == 64 ? 4 : 8;  // units of a row within a 128-byte column
    constexpr int RPW = 32 / UPR;           // rows a warp covers at once
    static_assert((4 * RPW) % 8 == 0, "one swizzle a lane");
    const int u = lane % UPR, r0 = cw * RPW + lane / UPR;
    const bool swap = UPR == 8 && u >= 4;
    const uint32_t from = r0 * 128 + ((u ^ (r0 & 7)) << 4);
    const uint32_t to0 = (u >> 2) * BN * 128 + r0 * 128 + (((2 * (u & 3)) ^ (r0 & 7)) << 4);
    const uint32_t to1 = (u >> 2) * BN * 128 + r0 * 128 + (((2 * (u & 3) + 1) ^ (r0 & 7)) << 4);
    for (int j = 0; j < n; ++j) {
      const int s8 = j % C::STV, s = j & 1;
      mbar_wait(bar(C::kBarV8 + s8), (j / C::STV) & 1, dead, p.err);
      if (j >= 2) mbar_wait(bar(C::kBarO + s), ((j >> 1) - 1) & 1, dead, p.err);
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      const uint32_t src = sV8 + s8 * C::kTile8, dst = sV + s * C::kTile16;
      const int key0 = (kt0 + j) * BN;
      // A row's 16-byte unit u (16 values) becomes two units of its atom.
      // Eight lanes take a row's units; those of the upper half write their
      // second unit first, so that each store of eight lanes covers all banks.
      // A lane's rows are 4 RPW apart, so its swizzle is the same in all.
      auto turn = [&](auto edge_c) {
        constexpr bool EDGE = decltype(edge_c)::value;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
#pragma unroll
          for (int i = 0; i < BN / (4 * RPW); ++i) {
            uint32_t w[4], o[8];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(src + from + c * BN * 128 + i * 4 * RPW * 128));
            if (EDGE) {
              // Keys that no row sees are zeros: what lies there is not data.
              const int key = key0 + r0 + i * 4 * RPW;
              if (key < k_lo || key >= k_hi) w[0] = w[1] = w[2] = w[3] = 0u;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) e4m3x4_to_f16(w[k], o[2 * k], o[2 * k + 1]);
            const uint32_t at = dst + c * 2 * BN * 128 + i * 4 * RPW * 128;
            if (swap) {
              st_shared_v4(at + to1, o[4], o[5], o[6], o[7]);
              st_shared_v4(at + to0, o[0], o[1], o[2], o[3]);
            } else {
              st_shared_v4(at + to0, o[0], o[1], o[2], o[3]);
              st_shared_v4(at + to1, o[4], o[5], o[6], o[7]);
            }
          }
        }
      };
      if (key0 < k_lo || key0 + BN > k_hi) turn(std::true_type{});
      else turn(std::false_type{});
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(C::kBarP + s));
        mbar_arrive(bar(C::kBarV8E + s8));
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    if constexpr (C::REGS) reg_inc<C::kSoftRegs>();
    const int wg = (warp - 4) >> 2;       // warpgroup: tile group, part of the row
    const int grp = wg / CH, part = wg % CH;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const int st = tid - 128;  // softmax thread
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const int row_bar = 2 + grp * 4 + wq;  // the warps that share these rows
    float* xch = reinterpret_cast<float*>(smem + C::kOffXch);

    // Where a row goes in the output.
    long long* row_at = reinterpret_cast<long long*>(smem + C::kOffRow);
    if (wg == 0 && r < rows) {
      const unsigned rr = static_cast<unsigned>(row0 + r), tok = rr / static_cast<unsigned>(p.G);
      row_at[r] = (q_beg + static_cast<long long>(tok)) * p.out_row_stride +
                  (kvh * p.G + static_cast<int>(rr - tok * p.G)) * static_cast<long long>(hd);
    }
    int lo = 0, hi = INT_MAX;  // rows past the end see everything: they slow nothing down
    if (r < rows) interval(r, lo, hi);
    const float qs = sQs[r];
    constexpr bool capped = C::CAPPED;
    // Score factor without the block's K scale: log2 units, or for the
    // soft-cap the argument of tanh.
    const float row_c =
        qs * fabsf(capped ? p.scale / p.softcap : p.scale_log2);
    const float cap_l2 = p.softcap * 1.4426950408889634f;
    const int shift = 31 - __clz(p.c.T);
    const float* ksc = p.c.k_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
    const float* vsc = p.c.v_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
    // Lane c < SC / 16 takes the scales of this part's keys 16 c .. 16 c + 15,
    // loaded a tile ahead; they reach the other lanes through shared memory.
    constexpr int NC = C::NC;
    float nk = 0.f, nv = 1.f;
    auto scales = [&](int j) {
      if (j < n) {
        const int key = (kt0 + j) * BN + part * SC + (lane % NC) * 16;
        const long long at = static_cast<long long>(min(key >> shift, p.c.n_blocks - 1)) * p.c.Hkv;
        nk = ksc[at];
        nv = vsc[at];
      }
    };
    float* my_sc = reinterpret_cast<float*>(smem + C::kOffSc) + (warp - 4) * 6 * NC;
    float m = -INFINITY, l = 0.f;
    int used = 0;
    // Nothing but padding in this warp's 32 rows: their P stays as it is.
    const bool idle = wq * 32 >= rows;
    scales(grp);
    for (int j = grp; j < n; j += TG) {
      const int x2 = j & 1, use = j >> 1;
      if (__builtin_expect(idle, 0)) {
        mbar_wait(bar(C::kBarS + x2), use & 1, dead, p.err);
        if (C::PSEP) {
          if (lane == 0) mbar_arrive(bar(C::kBarSE + x2));
          // As below: P[j] counts only once P[j - 2] was read.
          if (j >= 2) mbar_wait(bar(C::kBarO + x2), (use - 1) & 1, dead, p.err);
        }
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        if (lane == 0) {
          mbar_arrive(bar(C::kBarP + x2));
          if (C::HALVES) mbar_arrive(bar(C::kBarP2 + x2));
        }
        continue;
      }
      float* tab = my_sc + (used & 1) * 3 * NC;  // [k scale, L, 2^-L][NC]
      if (lane < NC) {
        const float L = kv8_log2(nv);
        tab[lane] = nk;
        tab[NC + lane] = L;
        tab[2 * NC + lane] = ex2_approx(-L);
      }
      scales(j + TG);
      __syncwarp();
      mbar_wait(bar(C::kBarS + x2), use & 1, dead, p.err);
      dead = __any_sync(0xffffffffu, dead);
      if (st == grp * 128 * CH) mbar_arrive(bar(C::kBarKE + j % C::STK));  // K[j] was read
      if (CH == 1 && dead) break;
      // (The warps of a row end together, so that none waits for another.)
      tc_fence_after();
      const uint32_t s_addr = tmem + lane_off + x2 * BN + part * SC;
      const int key0 = (kt0 + j) * BN + part * SC;
      const bool full = key0 >= f_lo && key0 + SC <= f_hi;
      // Column i of the part is visible iff (unsigned)(i - v0) < v1.
      const int v0 = lo - key0;
      const uint32_t v1 = static_cast<uint32_t>(hi) - static_cast<uint32_t>(lo);
      float sr[SC];
      if constexpr (SC >= 32) {
#pragma unroll
        for (int cb = 0; cb < SC / 32; ++cb)
          tmem_ld32(s_addr + cb * 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[cb * 32]));
      } else {
        tmem_ld16(s_addr, *reinterpret_cast<uint32_t(*)[16]>(&sr[0]));
      }
      float a16[NC], L16[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        a16[c] = row_c * tab[c];
        L16[c] = tab[NC + c];
      }
      tmem_wait_ld();
      if constexpr (C::PSEP) {
        tc_fence_before();
        if (lane == 0) mbar_arrive(bar(C::kBarSE + x2));
      }
      if (__builtin_expect(!full, 0)) {
#pragma unroll
        for (int i = 0; i < SC; ++i)
          sr[i] = static_cast<uint32_t>(i - v0) < v1 ? sr[i] : -INFINITY;
        // A masked score has to stay -inf times its piece's factor. That one
        // is no number above zero where nothing was written (scale 0, or
        // whatever the allocation held), where scale is 0, or where it
        // underflowed (a row of zeros over a block of zeros): the smallest
        // normal number stands in, which adds nothing to a visible score.
#pragma unroll
        for (int c = 0; c < NC; ++c) a16[c] = fmaxf(a16[c], FLT_MIN);
      }
      float cmax = -INFINITY;
      float m16[NC];  // each piece's largest score
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float* x = &sr[c * 16];
        float m0 = fmax3(x[0], x[1], x[2]), m1 = fmax3(x[3], x[4], x[5]);
        m0 = fmax3(m0, x[6], x[7]);
        m1 = fmax3(m1, x[8], x[9]);
        m0 = fmax3(m0, x[10], x[11]);
        m1 = fmax3(m1, x[12], x[13]);
        m0 = fmax3(m0, x[14], x[15]);
        m16[c] = fmaxf(m0, m1);
      }
      bool poly = false;
      if constexpr (capped) {
        // Whether every argument of tanh is in the polynomial's range: the
        // largest magnitude (masked scores, -inf, count as 0).
        float umax = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float* x = &sr[c * 16];
          float u0 = 0.f, u1 = 0.f;
          if (full) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              u0 = fmax3(u0, fabsf(x[i]), fabsf(x[i + 1]));
              u1 = fmax3(u1, fabsf(x[i + 2]), fabsf(x[i + 3]));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) u0 = fmaxf(u0, x[i] == -INFINITY ? 0.f : fabsf(x[i]));
          }
          umax = fmaxf(umax, fmaxf(u0, u1) * a16[c]);
        }
        poly = __all_sync(0xffffffffu, umax <= kTanhPolyMax);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float u = m16[c] * a16[c];
          const float t = poly ? tanh_poly(u) : kv8_tanh(u);
          cmax = fmaxf(cmax, m16[c] == -INFINITY ? m16[c] : fmaf(cap_l2, t, L16[c]));
        }
      } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) cmax = fmaxf(cmax, fmaf(m16[c], a16[c], L16[c]));
      }
      if constexpr (CH > 1) {
        // The other parts' maxima (and whether a warp gave up: a NaN, which a
        // maximum never is).
        xch[(wg * 2 + (used & 1)) * 128 + r] = dead ? __int_as_float(0x7fc00000) : cmax;
        named_bar_sync(row_bar, 32 * CH);
#pragma unroll
        for (int k = 1; k < CH; ++k) {
          const int o = grp * CH + (part + k) % CH;
          const float other = xch[(o * 2 + (used & 1)) * 128 + r];
          dead |= other != other;
          cmax = fmaxf(cmax, other);
        }
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
      }
      const bool resc = cmax > m + kKv8Lazy;
      float corr = 1.f;
      if (resc) {
        corr = ex2_approx(m - cmax);
        m = cmax;
      }
      const float mu = m == -INFINITY ? 0.f : m - kKv8Shift;
      // P of tile j - 2 must have been read before P[j] takes its place. (P in
      // S's place: S[j] waited for that, and this group's O is at rest.)
      if (C::PSEP && j >= 2) {
        mbar_wait(bar(C::kBarO + x2), (use - 1) & 1, dead, p.err);
        dead = __any_sync(0xffffffffu, dead);
        tc_fence_after();
      }
      const uint32_t p_addr =
          tmem + lane_off + C::kPCol + x2 * (BN / 16 * C::kPStep) + part * (SC / 16 * C::kPStep);
      // O follows a moved maximum before any of this tile's P V.
      if (__builtin_expect(j >= TG && __any_sync(0xffffffffu, resc), 0)) {
        if (TG == 1) {  // the previous P V may still add to O
          mbar_wait(bar(C::kBarO + (x2 ^ 1)), ((j - 1) >> 1) & 1, dead, p.err);
          dead = __any_sync(0xffffffffu, dead);
          tc_fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < HDP / CH / 32; ++c) {
          uint32_t o[32];
          const uint32_t ta = tmem + lane_off + C::kOCol + grp * HDP + part * (HDP / CH) + c * 32;
          tmem_ld32(ta, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = f2u(u2f(o[i]) * corr);
          tmem_st32(ta, o);
        }
      }
      float sum = 0.f;
      auto pass2 = [&](auto cap_c, auto full_c) {
        constexpr int CAP = decltype(cap_c)::value;  // 0 none, 1 tanh, 2 its polynomial
        constexpr bool FULL = decltype(full_c)::value;
        // Two pieces of 16 keys at a time, operation by operation: the chain
        // of one element is long, so many are kept in flight.
        constexpr int PP = NC < 2 ? 1 : 2;
#pragma unroll
        for (int c0 = 0; c0 < NC; c0 += PP) {
          if (C::HALVES && c0 == NC / 2) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::kBarP + x2));
          }
          float2 y[PP][8];
#pragma unroll
          for (int h = 0; h < PP; ++h) {
            const int c = c0 + h;
            const float off = L16[c] - mu;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float x0 = sr[c * 16 + 2 * q], x1 = sr[c * 16 + 2 * q + 1];
              if constexpr (CAP == 0) {
                y[h][q] = __ffma2_rn(make_float2(x0, x1), make_float2(a16[c], a16[c]),
                                     make_float2(off, off));
              } else if constexpr (CAP == 1) {
                y[h][q].x = x0 == -INFINITY ? x0 : fmaf(cap_l2, kv8_tanh(x0 * a16[c]), off);
                y[h][q].y = x1 == -INFINITY ? x1 : fmaf(cap_l2, kv8_tanh(x1 * a16[c]), off);
              } else {
                const float2 t = tanh_poly2(__fmul2_rn(make_float2(x0, x1),
                                                       make_float2(a16[c], a16[c])));
                y[h][q] = __ffma2_rn(make_float2(cap_l2, cap_l2), t, make_float2(off, off));
                if (!FULL) {
                  y[h][q].x = x0 == -INFINITY ? x0 : y[h][q].x;
                  y[h][q].y = x1 == -INFINITY ? x1 : y[h][q].y;
                }
              }
            }
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int h = 0; h < PP; ++h) {
              y[h][q].x = ex2_approx(y[h][q].x);
              y[h][q].y = ex2_approx(y[h][q].y);
            }
#pragma unroll
          for (int h = 0; h < PP; ++h) {
            uint32_t w[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) w[q] = pack_f16(y[h][q].x, y[h][q].y);
            tmem_st8(p_addr + (c0 + h) * C::kPStep, w);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1)
#pragma unroll
              for (int q = 0; q < o; ++q) y[h][q] = __fadd2_rn(y[h][q], y[h][q + o]);
            sum = fmaf(y[h][0].x + y[h][0].y, tab[2 * NC + c0 + h], sum);
          }
        }
      };
      if constexpr (!capped) {
        pass2(std::integral_constant<int, 0>{}, std::true_type{});
      } else {
        if (!poly) pass2(std::integral_constant<int, 1>{}, std::true_type{});
        else if (full) pass2(std::integral_constant<int, 2>{}, std::true_type{});
        else pass2(std::integral_constant<int, 2>{}, std::false_type{});
      }
      l = fmaf(l, corr, sum);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar((C::HALVES ? C::kBarP2 : C::kBarP) + x2));
      ++used;
    }

    // ------------------------------------------------------------ epilogue
    if (n > 0 && !dead) {
      mbar_wait(bar(C::kBarF), 0, dead, p.err);
      dead = __any_sync(0xffffffffu, dead);
      tc_fence_after();
    }
    // Maxima and sums of all parts: [warpgroup][l, m][128]. The parts of a
    // group have one maximum.
    named_bar_sync(1, C::kSoftThreads);
    xch[wg * 256 + r] = l;
    xch[wg * 256 + 128 + r] = m;
    named_bar_sync(1, C::kSoftThreads);
    auto group_sum = [&](int k) -> float {
      float y = 0.f;
#pragma unroll
      for (int h = 0; h < CH; ++h) y += xch[(k * CH + h) * 256 + r];
      return y;
    };
    float s_me = 1.f, s_ot = 0.f, mt = m, lt = group_sum(grp);
    if constexpr (TG == 2) {
      const float l_ot = group_sum(grp ^ 1);
      const float m_ot = xch[((grp ^ 1) * CH) * 256 + 128 + r];
      mt = fmaxf(m, m_ot);
      const float ref = mt == -INFINITY ? 0.f : mt;
      s_me = ex2_approx(m - ref);
      s_ot = ex2_approx(m_ot - ref);
      lt = grp == 0 ? fmaf(lt, s_me, l_ot * s_ot) : fmaf(l_ot, s_ot, lt * s_me);
    }
    const int n_me = TG == 2 ? (grp == 0 ? (n + 1) / 2 : n / 2) : n;
    const int n_ot = n - n_me;
    const bool final_out = p.splits == 1;
    const float inv = final_out ? __fdiv_rn(1.f, lt) : 1.f;
    const long long cell = (static_cast<long long>(b) * p.c.Hkv + kvh) * p.tiles + tile;
    // Each warp puts 32 columns of its 32 rows into shared memory (the K ring
    // is idle), 16-byte units turned by the row, and writes them out row by
    // row, so that global stores are whole 64- or 128-byte pieces.
    const bool f32 = !final_out || p.out_f32;
    const uint32_t stage = sK + (warp - 4) * 4096;
    constexpr int WC = HDP / (CH * TG);  // columns a warp writes
    constexpr int PC = WC < 32 ? WC : 32;  // ... at a time
#pragma unroll 1
    for (int c = 0; c < WC / PC; ++c) {
      const int col0 = wg * WC + c * PC;
      uint32_t o[32];
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
      if (n_me > 0 && !dead) {
        tmem_ld32(tmem + lane_off + C::kOCol + grp * HDP + col0, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = u2f(o[i]) * s_me;
      }
      if (TG == 2 && n_ot > 0 && !dead) {
        tmem_ld32(tmem + lane_off + C::kOCol + (grp ^ 1) * HDP + col0, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = fmaf(u2f(o[i]), s_ot, v[i]);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = dead ? __int_as_float(0x7fc00000) : v[i] * inv;
      // Units of 16 bytes: 4 fp32 or 8 bf16.
      const int units = f32 ? PC / 4 : PC / 8, sh = 31 - __clz(units);
      const uint32_t my_row = stage + lane * (units * 16);
#pragma unroll
      for (int u = 0; u < PC / 4; ++u) {
        if (f32) {
          st_shared_v4(my_row + ((u ^ (lane & (PC / 4 - 1))) << 4), f2u(v[4 * u]),
                       f2u(v[4 * u + 1]), f2u(v[4 * u + 2]), f2u(v[4 * u + 3]));
        } else if (u < PC / 8) {
          st_shared_v4(my_row + ((u ^ (lane & (PC / 8 - 1))) << 4), pack_bf16(v[8 * u], v[8 * u + 1]),
                       pack_bf16(v[8 * u + 2], v[8 * u + 3]), pack_bf16(v[8 * u + 4], v[8 * u + 5]),
                       pack_bf16(v[8 * u + 6], v[8 * u + 7]));
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int i = lane; i < 32 * units; i += 32) {
        const int wr = i >> sh, u = i & (units - 1);
        const int gr = wq * 32 + wr, col = col0 + u * (f32 ? 4 : 8);
        if (gr < rows && col < hd) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(stage + wr * (units * 16) + ((u ^ (wr & (units - 1))) << 4)));
          char* d = !final_out
                        ? reinterpret_cast<char*>(
                              p.part_o + ((cell * p.splits + split) * 128 + gr) * hd + col)
                        : static_cast<char*>(p.out) + (row_at[gr] + col) * (f32 ? 4 : 2);
          *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
    }
    if (!final_out) {
      float* pml = p.part_ml + (cell * p.splits + split) * 256;
      if (wg == 0 && r < rows) {
        pml[r] = mt;
        pml[128 + r] = lt;
      }
      __threadfence();
      named_bar_sync(1, C::kSoftThreads);
      if (st == 0) {
        const int done = atomicAdd(p.tickets + cell, 1);
        misc[5] = done == p.splits - 1;
        if (misc[5]) p.tickets[cell] = 0;  // as the next call finds it
      }
      named_bar_sync(1, C::kSoftThreads);
      if (misc[5]) {
        __threadfence();
        pml = p.part_ml + cell * p.splits * 256;
        const float* po = p.part_o + cell * p.splits * 128 * static_cast<long long>(hd);
        // Each split's weight in each row, divided by the row's sum, first (in
        // the idle rings); then the sums, eight loads of a thread in flight.
        float* jw = reinterpret_cast<float*>(smem + C::kOffK);
        for (int jr = st; jr < rows; jr += C::kSoftThreads) {
          float mj = -INFINITY, lj = 0.f;
#pragma unroll 8
          for (int k = 0; k < p.splits; ++k) mj = fmaxf(mj, __ldcg(pml + k * 256 + jr));
#pragma unroll 8
          for (int k = 0; k < p.splits; ++k) {
            const float w = mj == -INFINITY ? 0.f : ex2_approx(__ldcg(pml + k * 256 + jr) - mj);
            lj = fmaf(__ldcg(pml + k * 256 + 128 + jr), w, lj);
            jw[k * 128 + jr] = w;
          }
          // A row that sees nothing: 0 / 0.
          const float ij = mj == -INFINITY ? __int_as_float(0x7fc00000) : __fdiv_rn(1.f, lj);
          for (int k = 0; k < p.splits; ++k) jw[k * 128 + jr] *= ij;
        }
        named_bar_sync(1, C::kSoftThreads);
        const int upr = hd / 4, total = rows * upr;
        constexpr int U = 4;
#pragma unroll 1
        for (int i0 = st; i0 < total; i0 += U * C::kSoftThreads) {
          float4 acc[U];
#pragma unroll
          for (int u = 0; u < U; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
          for (int k = 0; k < p.splits; ++k) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int i = min(i0 + u * C::kSoftThreads, total - 1);
              const float w = jw[k * 128 + i / upr];
              // Rows lie hd apart: element i of the tile is float4 i of the split's.
              const float4 x = __ldcg(reinterpret_cast<const float4*>(
                  po + static_cast<long long>(k) * 128 * hd) + i);
              acc[u].x = fmaf(x.x, w, acc[u].x);
              acc[u].y = fmaf(x.y, w, acc[u].y);
              acc[u].z = fmaf(x.z, w, acc[u].z);
              acc[u].w = fmaf(x.w, w, acc[u].w);
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = i0 + u * C::kSoftThreads;
            if (i < total) {
              const int jr = i / upr;
              const long long d = row_at[jr] + (i - jr * upr) * 4;
              if (p.out_f32)
                *reinterpret_cast<float4*>(static_cast<float*>(p.out) + d) = acc[u];
              else
                *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + d) =
                    make_uint2(pack_bf16(acc[u].x, acc[u].y), pack_bf16(acc[u].z, acc[u].w));
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ca
