// pair.cuh -- act . W^T for many rows of act, alone or gated: two SMs on one
// tile (tcgen05 with cta_group::2), persistent.
//
// Formulas as in skinny.cuh. The two CTAs of a cluster take 256 weight rows by
// NT tokens: each holds 128 rows of the weights and half the tokens in its
// shared memory and, in its TMEM, its 128 rows of the product, so that an
// operand byte fetched from L2 serves twice the multiplications that it would
// in one CTA. Accumulators are double buffered in TMEM: while the tensor cores
// work on a tile, eight warps of each CTA scale, activate, round and store the
// one before.
//
// Gated: of a CTA's 128 rows 64 are of Wgate and 64 of Wup, the same ones. A
// row's gate and up are then 64 lanes apart, in two warps that pass each other
// half their tokens through shared memory (16 tokens at a time: eight stores,
// a barrier of the two, eight loads) and finish the other half each. Both
// matrices as operands of their own would leave room for 128 tokens a tile
// with two buffers, and at 128 the operands' way out of shared memory is the
// bound (8192 tokens, 4096 -> 12288 in e4m3: 1031 us); turns of 16 rows, which
// a shuffle could bring together, need nine loads a stage (887 us).
//
// CHUNK > 0: the tensor core adds to an accumulator for CHUNK pieces of 128
// bytes at most, then the storing warps add it up in registers. It truncates
// as it accumulates: without it fp32 results of bf16 operands of 4112 columns
// were 9e-6 off in 2-norm, those of e4m3 ones over 18944 columns 9e-6 where all
// products have one sign (5e-7 over 4096 columns, and with it). It is for fp32
// outputs alone; a bf16 one rounds by 2e-3. (512 gated tokens 4096 -> 12288 in
// bf16: one rounding in 220 falls to the other side of that of exact sums, 2e-4
// in 2-norm; results are as far from the exact ones, 1.6567e-3.) 8192 tokens
// 12288 -> 4096 in e4m3 to fp32: 320 us without it, 342 with it (128 sums a
// thread, 848 bytes of spills), 530 to 580 in tiles of 128 tokens.
//
// Warps: 0 loads (TMA, both CTAs, completing on the even CTA's barriers), 1
// issues (the even CTA alone), 2-9 store, half the tokens of 32 lanes each.
// Lane = weight row, column = token: a warp's threads store 32 neighbours of an
// output row.
#pragma once

#include <cstdint>

#include "skinny.cuh"

namespace ca {

// A load into this CTA's shared memory that completes on `bar`, which may be a
// barrier of the pair's other CTA.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t bar,
                                                 int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

template <int KIND>
__device__ __forceinline__ void mma_ss_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  if constexpr (KIND == kKindBf16) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Arrives on `bar` of both CTAs when every MMA issued so far is done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

template <int KIND_, int G_, int NT_, int CHUNK_ = 0>
struct PairCfg {
  static constexpr int CHUNK = CHUNK_;
  static constexpr int KIND = KIND_;
  static constexpr int G = G_;
  static constexpr int NT = NT_;  // tokens of a tile
  static constexpr int kStage = 16384 + NT / 2 * 128;
  static constexpr int kStages = 208 * 1024 / kStage < 8 ? 208 * 1024 / kStage : 8;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kThreads = 320;
  static constexpr int kBars = 2 * kStages + 4;
  static constexpr int kHalf = NT / 2;  // tokens of a storing warp
  static constexpr int kScales = 8 * kHalf * 4;
  static constexpr int kSwap = G == 2 ? 16384 : 0;  // 8 warps x 2 buffers x 8 tokens x 32 lanes
  static constexpr int kSmem = 1024 + kRing + kScales + kSwap + 8 * kBars + 16;
  static constexpr int kBuf = NT;  // TMEM columns of a buffer
  static constexpr int kRows = 256 / G;  // output rows of a tile
  static constexpr int kTmemCols = 2 * kBuf;
  static constexpr int kElems = KIND == kKindBf16 ? 64 : 128;
  static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM");
};

constexpr int kPairGroup = 8;  // row tiles side by side in the order of the tiles

// Tile i of r_tiles x t_tiles: row tiles in groups, tokens in a group's turn,
// so that the tiles in work at a time share what they read in both operands.
__device__ __forceinline__ void pair_tile(const LinearParams& p, int i, int& rt, int& tt) {
  const int g = i / (kPairGroup * p.t_tiles);
  const int first = g * kPairGroup, size = min(kPairGroup, p.r_tiles - first);
  const int j = i - first * p.t_tiles;
  rt = first + j % size;
  tt = j / size;
}

// A row's scale w as factors of a sum before and after the token's scale, one of
// them 1: below 1 it goes first, to the same end as in `scaled`, whose choice for
// each element took 512 tokens 4096 -> 4096 from 15.5 to 16.4 us here. Without a
// token's scale: all of it after.
struct RowScale {
  float before, after;
  __device__ __forceinline__ RowScale(float w, bool alone)
      : before(!alone && fabsf(w) < 1.f ? w : 1.f), after(!alone && fabsf(w) < 1.f ? 1.f : w) {}
};

template <class C>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(C::kThreads)
    pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_u,
                const __grid_constant__ CUtensorMap tm_x, const LinearParams p) {
  extern __shared__ uint8_t raw_smem[];
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  const uint32_t scales = base + C::kRing, swap = scales + C::kScales;
  const uint32_t bars = swap + C::kSwap, slot = bars + 8 * C::kBars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto full = [&](int s) { return bars + 8 * s; };                      // of the even CTA
  auto empty = [&](int s) { return bars + 8 * (C::kStages + s); };      // each CTA's
  auto acc_full = [&](int b) { return bars + 8 * (2 * C::kStages + b); };
  auto acc_empty = [&](int b) { return bars + 8 * (2 * C::kStages + 2 + b); };  // of the even CTA
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int tiles = p.r_tiles * p.t_tiles;

  bool dead = false;
  // The loading thread's place: stages filled, and the piece of the tile.
  int filled = 0, tile = pair, kb = 0, r0 = 0, t0 = 0;
  auto fill = [&]() {
    if (kb == 0) {
      int rt, tt;
      pair_tile(p, tile, rt, tt);
      r0 = rt * C::kRows + static_cast<int>(rank) * (C::kRows / 2);
      t0 = tt * C::NT + static_cast<int>(rank) * (C::NT / 2);
    }
    const int s = filled % C::kStages;
    if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * C::kStage);
    const uint32_t dst = base + s * C::kStage, bar = map_to_rank(full(s), 0);
    tma_load_2d_pair(dst, &tm_w, bar, kb * C::kElems, r0);
    if constexpr (C::G == 2) tma_load_2d_pair(dst + 8192, &tm_u, bar, kb * C::kElems, r0);
    tma_load_2d_pair(dst + 16384, &tm_x, bar, kb * C::kElems, t0);
    ++filled;
    if (++kb == p.kblocks) {
      kb = 0;
      tile += n_pairs;
    }
  };
  if (tid == 0) {
    tma_prefetch_desc(&tm_w);
    if constexpr (C::G == 2) tma_prefetch_desc(&tm_u);
    tma_prefetch_desc(&tm_x);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 16);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  cluster_arrive_relaxed();  // (the barriers' initialisation has a fence of its own)
  cluster_wait();            // the barriers of both are set
  wait_prior_kernel();  // before TMEM is taken, as in skinny.cuh
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(C::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_relaxed();
  if (tid == 0)
    while (filled < C::kStages && tile < tiles) fill();  // the first loads need no TMEM
  __syncwarp();
  cluster_wait();  // both CTAs have theirs
  tc_fence_after();
  let_next_kernel();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  if (warp == 0) {
    if (lane == 0) {
      while (tile < tiles) {
        if (!mbar_wait(empty(filled % C::kStages), ((filled / C::kStages) - 1) & 1, dead, p.err))
          break;
        fill();
      }
      // After an expired wait the copies in flight still have to land; the
      // even CTA's barriers count those of both.
      if (dead && rank == 0) {
        bool late = false;
        for (int j = max(0, filled - C::kStages); j < filled; ++j)
          mbar_wait(full(j % C::kStages), (j / C::kStages) & 1, late, p.err);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = linear_idesc(C::KIND, 256, C::NT);
      int i = 0, n = 0;  // stages taken, accumulators filled
      for (int tile = pair; tile < tiles && !dead; tile += n_pairs, ++n) {
        uint32_t acc = 0;
        int first = 0;
        for (int kb = 0; kb < p.kblocks; ++kb, ++i) {
          if (kb == 0 || (C::CHUNK > 0 && kb % (C::CHUNK > 0 ? C::CHUNK : 1) == 0)) {
            if (kb > 0) umma_commit_pair(acc_full(n++ & 1));
            if (n >= 2 && !mbar_wait(acc_empty(n & 1), ((n >> 1) - 1) & 1, dead, p.err)) break;
            tc_fence_after();
            acc = tmem + (n & 1) * C::kBuf;
            first = kb;
          }
          const int s = i % C::kStages;
          if (!mbar_wait(full(s), (i / C::kStages) & 1, dead, p.err)) break;
          tc_fence_after();
          const uint32_t at = base + s * C::kStage;
          const uint64_t dw = umma_desc_sw128(at, 16, 1024);
          const uint64_t dx = umma_desc_sw128(at + 16384, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss_pair<C::KIND>(acc, dw + 2 * kk, dx + 2 * kk, idesc, (kb - first) | kk);
          umma_commit_pair(empty(s));
        }
        umma_commit_pair(acc_full(n & 1));
      }
    }
  } else {
    int n = 0;
    const int half0 = (warp - 2) / 4 * C::kHalf;  // this warp's first token of a tile
    // Gated: the warp that holds the other matrix's rows, its barrier.
    const bool up = C::G == 2 && (warp & 2);
    const int swap_bar = 1 + (warp & 1) + (warp - 2) / 4 * 2;
    int turn = 0;
    const uint32_t sa_at = scales + (warp - 2) * C::kHalf * 4;
    auto take = [&]() {  // the next accumulator
      mbar_wait(acc_full(n & 1), (n >> 1) & 1, dead, p.err);
      __syncwarp();
      tc_fence_after();
      return tmem + (n & 1) * C::kBuf + half0 + (static_cast<uint32_t>(warp & 3) << 21);
    };
    auto give = [&]() {  // it may be written again
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_rank(acc_empty(n & 1), 0));
      ++n;
    };
    // An expired wait (`dead`: later ones return at once) ends no warp early:
    // warps that pass each other their parts stay in step.
    for (int tile = pair; tile < tiles; tile += n_pairs) {
      int rt, tt;
      pair_tile(p, tile, rt, tt);
      // The output row of this lane; gated: of lanes l and l + 64 of TMEM.
      const int q = (C::G == 2 ? warp & 1 : warp & 3) * 32 + lane;
      const long long r = static_cast<long long>(rt) * C::kRows + rank * (C::kRows / 2) + q;
      const long long t0 = static_cast<long long>(tt) * C::NT + half0;
      const bool ok = r < p.rows;
      RowScale w0(1.f, true), w1(1.f, true);
      float bias = 0.f;
      if (ok) {
        if (p.w_scale) w0 = RowScale(p.w_scale[r], !p.act_scale);
        if (C::G == 2 && p.up_scale) w1 = RowScale(p.up_scale[r], !p.act_scale);
        if (C::G == 1 && p.bias) bias = p.bias[r];
      }
      if (p.act_scale) {
        __syncwarp();  // the last tile's are read
        for (int j = lane; j < C::kHalf; j += 32)
          st_shared_f32(sa_at + 4 * j, t0 + j < p.n ? p.act_scale[t0 + j] : 1.f);
        __syncwarp();
      }
      const float before = up ? w1.before : w0.before;  // of the rows that this warp holds
      // Residuals of the 32 tokens to come; the first ones are asked for before
      // the tile is there.
      float next[2][16];
      auto ask = [&](int j0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          load_residual(p, next[h], t0 + j0 + 16 * h, r, tokens_in<16>(p, t0 + j0 + 16 * h, ok));
      };
      if (C::G == 1 && p.residual) ask(0);
      // Sixteen tokens from t0 + j0 on, `h`: the second of 32.
      auto finish = [&](float (&d)[16], int j0, int h) {
        if (p.act_scale) {
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            float s[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(s[0]), "=f"(s[1]), "=f"(s[2]), "=f"(s[3])
                         : "r"(sa_at + 4 * (j0 + j)));
#pragma unroll
            for (int k = 0; k < 4; ++k) d[j + k] = d[j + k] * before * s[k];
          }
        }
        if constexpr (C::G == 2) {
          // Gate warps finish the first eight tokens, up warps the others.
          const uint32_t mine = swap + (warp - 2) * 2048 + (turn & 1) * 1024 + lane * 4;
          const uint32_t theirs = swap + ((warp - 2) ^ 2) * 2048 + (turn & 1) * 1024 + lane * 4;
          ++turn;
#pragma unroll
          for (int j = 0; j < 8; ++j) st_shared_f32(mine + j * 128, up ? d[j] : d[8 + j]);
          named_bar_sync(swap_bar, 64);
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float other;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(theirs + j * 128) : "memory");
            const float g = up ? other : d[j], u = up ? d[8 + j] : other;
            v[j] = activate(g * w0.after, p.act, p.out_f32) * (u * w1.after);
          }
          const long long t = t0 + j0 + (up ? 8 : 0);
          store_tokens(p, v, t, r, tokens_in<8>(p, t, ok));
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) d[j] = fmaf(d[j], w0.after, bias);
          if (p.residual) {
#pragma unroll
            for (int j = 0; j < 16; ++j) d[j] += next[h][j];
            if (h == 1 && j0 + 16 < C::kHalf) ask(j0 + 16);
          }
          store_tokens(p, d, t0 + j0, r, tokens_in<16>(p, t0 + j0, ok));
        }
      };
      if constexpr (C::CHUNK > 0) {
        float v[C::kHalf / 16][16];
#pragma unroll
        for (int j = 0; j < C::kHalf; ++j) v[j / 16][j % 16] = 0.f;
        for (int kb = 0; kb < p.kblocks; kb += C::CHUNK) {
          const uint32_t col = take();
#pragma unroll
          for (int j0 = 0; j0 < C::kHalf; j0 += 16) {
            uint32_t d[16];
            tmem_ld16(col + j0, d);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j0 / 16][j] += __uint_as_float(d[j]);
          }
          give();
        }
#pragma unroll
        for (int j0 = 0; j0 < C::kHalf; j0 += 16) finish(v[j0 / 16], j0, j0 / 16 & 1);
      } else {
        const uint32_t col = take();
#pragma unroll 1
        for (int j0 = 0; j0 < C::kHalf; j0 += 32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t d[16];
            tmem_ld16(col + j0 + 16 * h, d);
            tmem_wait_ld();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(d[j]);
            finish(v, j0 + 16 * h, h);
          }
        }
        give();
      }
    }
  }
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmemCols));
  }
  __syncwarp();
  cluster_arrive_relaxed();
  cluster_wait();
}

}  // namespace ca
