// attn_kv8_rows.cuh -- attention of a few query rows over the 8-bit cache.
//
// One CTA takes 8 or 16 query rows (token, head-of-the-group pairs, token-
// major) of one (sequence, kv head) and one stretch of its keys. Its warps
// walk that stretch in chunks of 16 keys, each on its own: a ring of K and V
// chunks filled by TMA, a softmax state, no barrier with the others until
// their sums meet at the end.
//
// Mathematics. A cached value is e4m3 * scale, one scale for each block of
// keys. With a = scale_k(block) * scale * log2 e and L = log2 scale_v(block),
//   t = a (q . k8) + L,   p = 2^(t - m),
//   O = sum p v8,         l = sum p 2^-L,     out = O / l
// with m a running bound of t: the V scale rides in the exponent, so P V
// runs on the held values, and only l has to take it out again. P is f16 at
// up to 2^15 (2^7 for t = m, and m is only moved when t passes it by 8), so
// weights down to 2^-31 of the largest count; sums and maxima are fp32.
//
// Both products are computed transposed, keys (or head dims) as the 16 rows
// of an mma and query rows as its 8 columns: the few query rows of a step
// then fill it, where as the 16-row operand they would leave most of it idle.
//   S^T = K Q^T   K as it is held (e4m3), Q in two e4m3 terms, q = hi + lo,
//                 each row scaled by a power of two into e4m3's range: bf16's
//                 8 bits exactly, down to 2^-18 of the row's largest value
//   O^T = V^T P^T V as f16 (exact), P^T by an 8 x 8 transpose of P
// The order of the head dims inside a product is free, so every lane reads
// whole 16-byte pieces of a row.
//
// Bound by HBM: 2 hd bytes a key. One token over 131072 positions of 8 kv
// heads x 128: 53 us, 5.1 TB/s, of which about 8 us are start and join (the
// 16-row form of both products, with K and V turned in registers, took 90);
// 1001 positions of 4 kv heads: 9.4 us, all latency. Long caches are split
// over CTAs; the last CTA of a row tile to finish joins their partial sums in
// order, so results do not depend on which that was.
#pragma once

#include <climits>
#include <cstdint>
#include <cuda_bf16.h>

#include "attn_fwd.cuh"
#include "kv8.cuh"

namespace ca {

struct Kv8AttnParams {
  Kv8View c;
  const __nv_bfloat16* q;  // [rows, H, hd]; token stride q_row_stride
  void* out;
  int out_f32;
  long long q_row_stride, out_row_stride;
  int sq;              // uniform batch (cu_q == null)
  const int* cu_q;
  const int* q_pos;    // per global query row; null: the last rows held
  const int* kv_len;   // [batch] or null (n_total)
  const int* seq_prefix;
  int causal_prefix;
  int window;
  int H, G;
  float scale, scale_log2, softcap;
  int splits;
  // A cell is a row tile of a (sequence, kv head), of nr = 8, 16 or 128 rows.
  float* part_o;       // [cell][split][nr][hd]
  float* part_ml;      // [cell][split][2][nr]
  int* tickets;        // [cell], zero between calls
  int tiles;           // row tiles of a (sequence, kv head)
  int* err;
};

// Keys a query row sees: [lo, hi) of the sequence's len held positions.
// visible() (src/model/attention.rs:35-57) on keys at positions 0 .. len - 1
// of one sequence is an interval.
__device__ __forceinline__ void kv8_interval(int pos, int len, int window, int prefix, int& lo,
                                             int& hi) {
  lo = 0;
  hi = len;
  if (window != kNoWindow) {
    const long long a = static_cast<long long>(pos) - window + 1;
    const long long z = static_cast<long long>(pos) + window;
    lo = static_cast<int>(a > 0 ? min(a, static_cast<long long>(len)) : 0);
    hi = static_cast<int>(z < len ? max(z, 0ll) : len);
  }
  if (prefix >= 0 && pos < prefix) hi = min(hi, max(pos, -1) + 1);
  if (hi < lo) hi = lo;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// D (+)= A B, 16 x 8 x 16, f16 in, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D (+)= A B, 16 x 8 x 32, e4m3 in, fp32 accumulate.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of 16-bit values held two a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Four scaled values into their two e4m3 terms.
__device__ __forceinline__ void split_e4m3(const float (&x)[4], uint32_t& hi, uint32_t& lo) {
  hi = cvt_e4m3x2(x[0], x[1]) | (cvt_e4m3x2(x[2], x[3]) << 16);
  float back[4];
  e4m3x4_to_f32(hi, back);
  lo = cvt_e4m3x2(x[0] - back[0], x[1] - back[1]) |
       (cvt_e4m3x2(x[2] - back[2], x[3] - back[3]) << 16);
}

// tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1), good to 2e-7 (the soft-cap's logits
// to 1e-5 of a unit); the infinities come out as 1 and -1.
__device__ __forceinline__ float kv8_tanh(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2_approx(x * 2.8853900817779268f) + 1.f));
  return fmaf(-2.f, r, 1.f);
}

constexpr float kKv8Shift = 7.f;  // P's f16 exponent for t = m
constexpr float kKv8Lazy = 8.f;   // how far t may pass m before m moves

// log2 of a V scale, kept where 2^L and 2^-L are both finite.
__device__ __forceinline__ float kv8_log2(float s) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return fminf(fmaxf(y, -100.f), 120.f);
}

// HDP: head_dim padded to 64, 128, 256 or 512. NR: query rows of a CTA, 8 or
// 16 (head_dim <= 128). At head_dim 512 two warps share a stretch of keys,
// each with half of the output columns and all of S.
template <int HDP_, int NR_>
struct RowsCfg {
  static constexpr int HDP = HDP_, NR = NR_;
  static constexpr int VS = HDP == 512 ? 2 : 1;
  static constexpr int kWarps = HDP == 512 ? 8 : HDP == 256 || NR == 16 ? 12 : 16;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kGroups = kWarps / VS;           // key-walking groups
  static constexpr int ST = HDP <= 128 ? (NR == 8 ? 3 : 4) : 2;  // chunks of a warp's ring
  static constexpr int KC = (HDP + 127) / 128;          // 128-byte columns of K
  static constexpr int VC = (KC + VS - 1) / VS;         // ... and of a warp's part of V
  static constexpr int kCol = 16 * 128;                 // bytes of such a column of a chunk
  static constexpr int kStage = (KC + VC) * kCol;
  static constexpr int kWarpBytes = ST * kStage;        // later the warp's partial O
  static constexpr int kOffBar = kWarps * kWarpBytes;
  static constexpr int kOffML = kOffBar + (kWarps * ST * 8 + 15) / 16 * 16;
  static constexpr int kOffMisc = kOffML + (kGroups * 3 + 1) * NR * 4;
  static constexpr int kSmem = kOffMisc + 16;
  static constexpr int OC = HDP / VS;                   // output columns of a warp
  static constexpr int LC = HDP == 64 ? 8 : 16;         // columns a lane has of each 128
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(NR * OC * 4 <= kWarpBytes, "a warp's sums fit its ring");
};

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
    attn_kv8_rows_kernel(const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const Kv8AttnParams p) {
  constexpr int HDP = C::HDP, NR = C::NR, ST = C::ST;
  constexpr int NT = NR / 8;             // 8-row tiles
  constexpr int KU = HDP / 64;           // 16-byte pieces of a K row per lane
  constexpr int VB = C::OC / (8 * C::LC);  // 128-byte columns (one half-filled at 64) of V
  constexpr int MT = VB * C::LC / 2;     // 16-dim tiles of O^T
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicExch(p.err ? p.err : &g_device_error, kErrLayout);
    return;
  }
  float* sml = reinterpret_cast<float*>(smem + C::kOffML);
  int* smisc = reinterpret_cast<int*>(smem + C::kOffMisc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int grp = warp / C::VS, vs = warp % C::VS;
  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int hd = p.c.hd;

  // What needs nothing but the arguments comes first.
  const uint32_t ring = smem_u32(smem + warp * C::kWarpBytes);
  const uint32_t bar0 = smem_u32(smem + C::kOffBar) + warp * ST * 8;
  if (lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int s = 0; s < ST; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  dependency_wait();

  const int q_beg = p.cu_q ? p.cu_q[b] : b * p.sq;
  const int q_len = p.cu_q ? p.cu_q[b + 1] - q_beg : p.sq;
  const long long n_rows = static_cast<long long>(q_len) * p.G;
  const long long row0 = static_cast<long long>(tile) * NR;
  if (row0 >= n_rows) return;
  const int rows = static_cast<int>(min(static_cast<long long>(NR), n_rows - row0));
  const unsigned G = static_cast<unsigned>(p.G);

  // Q's way from HBM is as long as that of kv_len: both at once.
  uint4 raw[NT][KU][2];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int r = 8 * x + g;
    const unsigned rr = static_cast<unsigned>(row0 + r), tok = rr / G;
    const __nv_bfloat16* src = p.q + (q_beg + static_cast<long long>(tok)) * p.q_row_stride +
                               (kvh * p.G + static_cast<int>(rr - tok * G)) *
                                   static_cast<long long>(hd);
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const int e = (t + 4 * i) * 16;
      raw[x][i][0] = raw[x][i][1] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && e < hd) {
        raw[x][i][0] = reinterpret_cast<const uint4*>(src + e)[0];
        raw[x][i][1] = reinterpret_cast<const uint4*>(src + e)[1];
      }
    }
  }
  const int len = p.kv_len ? min(max(p.kv_len[b], 0), p.c.n_total) : p.c.n_total;
  const int prefix = p.seq_prefix ? p.seq_prefix[b] : p.causal_prefix;

  // Lane (g, t) has query rows 2 t and 2 t + 1 of each 8: what they see, the
  // hull of what any row sees, and what every row sees.
  int lo[NT][2], hi[NT][2];
  int k_lo = 0, k_hi = len, f_lo = 0, f_hi = len;
#pragma unroll
  for (int x = 0; x < NT; ++x) lo[x][0] = lo[x][1] = 0, hi[x][0] = hi[x][1] = len;
  if (p.window != kNoWindow || prefix >= 0) {
    k_lo = f_hi = INT_MAX;
    k_hi = f_lo = 0;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int r = 8 * x + 2 * t + y;
        if (r < rows) {
          const int tok = static_cast<int>(static_cast<unsigned>(row0 + r) / G);
          const int pos = p.q_pos ? p.q_pos[q_beg + tok] : len - q_len + tok;
          kv8_interval(pos, len, p.window, prefix, lo[x][y], hi[x][y]);
          // A row that sees nothing does not widen the hull.
          if (lo[x][y] < hi[x][y]) {
            k_lo = min(k_lo, lo[x][y]);
            k_hi = max(k_hi, hi[x][y]);
          }
          f_lo = max(f_lo, lo[x][y]);
          f_hi = min(f_hi, hi[x][y]);
        }
      }
    k_lo = __reduce_min_sync(0xffffffffu, k_lo);
    k_hi = __reduce_max_sync(0xffffffffu, k_hi);
    f_lo = __reduce_max_sync(0xffffffffu, f_lo);
    f_hi = __reduce_min_sync(0xffffffffu, f_hi);
  }
  // This group's chunks: c_beg + grp, + kGroups, ...
  int c_beg = 0, c_end = 0;
  if (k_lo < k_hi) {
    const int first = k_lo >> 4, n = ((k_hi + 15) >> 4) - first;
    const int per = (n + p.splits - 1) / p.splits;
    c_beg = first + min(n, split * per);
    c_end = first + min(n, (split + 1) * per);
  }
  const int c0 = c_beg + grp;

  const int tok0 = b * p.c.n_total;
  auto fetch = [&](int ch, int s) {  // lane 0
    const uint32_t dst = ring + s * C::kStage, bar = bar0 + 8 * s;
    mbar_arrive_expect_tx(bar, C::kStage);
#pragma unroll
    for (int c = 0; c < C::KC; ++c)
      tma_load_3d(dst + c * C::kCol, &tm_k, bar, c * 128, kvh, tok0 + ch * 16);
#pragma unroll
    for (int c = 0; c < C::VC; ++c)
      tma_load_3d(dst + (C::KC + c) * C::kCol, &tm_v, bar, (vs * C::VC + c) * 128, kvh,
                  tok0 + ch * 16);
  };
  if (lane == 0) {
    for (int s = 0; s < ST; ++s)
      if (c0 + s * C::kGroups < c_end) fetch(c0 + s * C::kGroups, s);
  }
  __syncwarp();

  const float* ksc = p.c.k_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
  const float* vsc = p.c.v_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
  const int shift = 31 - __clz(p.c.T);
  float nk = 0.f, nv = 1.f;  // the next chunk's scales
  auto scales = [&](int ch) {
    if (ch < c_end) {
      const long long blk = static_cast<long long>((ch * 16) >> shift) * p.c.Hkv;
      nk = ksc[blk];
      nv = vsc[blk];
    }
  };
  scales(c0);

  // Q as the products' B operand: lane (g, t) has of row g the head dims
  // (t + 4 i) 16 .. + 15, two steps of 32 for each i.
  uint32_t qf[NT][2][KU][4];
  float qs[NT][2];  // the scale of rows 2 t, 2 t + 1
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < KU; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w4[4] = {raw[x][i][h].x, raw[x][i][h].y, raw[x][i][h].z, raw[x][i][h].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          amax = fmax3(amax, fabsf(__uint_as_float(w4[k] << 16)),
                       fabsf(__uint_as_float(w4[k] & 0xffff0000u)));
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int ex = e4m3_exp(fminf(amax, __uint_as_float(0x7f7f0000u)), -120, 120);
    const float inv = exp2_int(-ex);
#pragma unroll
    for (int i = 0; i < KU; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w4[4] = {raw[x][i][h].x, raw[x][i][h].y, raw[x][i][h].z, raw[x][i][h].w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float v[4] = {__uint_as_float(w4[2 * k] << 16) * inv,
                              __uint_as_float(w4[2 * k] & 0xffff0000u) * inv,
                              __uint_as_float(w4[2 * k + 1] << 16) * inv,
                              __uint_as_float(w4[2 * k + 1] & 0xffff0000u) * inv};
          split_e4m3(v, qf[x][0][i][2 * h + k], qf[x][1][i][2 * h + k]);
        }
      }
    // A row with an infinity has scores that are none: NaN comes out.
    const float mine = amax == INFINITY ? INFINITY : exp2_int(ex);
#pragma unroll
    for (int y = 0; y < 2; ++y) qs[x][y] = __shfl_sync(0xffffffffu, mine, (2 * t + y) * 4);
  }

  float o[NT][MT][4];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int y = 0; y < 4; ++y) o[x][j][y] = 0.f;
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x) m[x][0] = m[x][1] = -INFINITY, l[x][0] = l[x][1] = 0.f;
  const bool capped = p.softcap != 0.f;
  const float score = capped ? p.scale / p.softcap : p.scale_log2;
  const float cap_l2 = p.softcap * 1.4426950408889634f;
  bool dead = false;

  int it = 0;
  for (int ch = c0; ch < c_end; ch += C::kGroups, ++it) {
    const int s = it % ST;
    const float ks = nk, L = kv8_log2(nv);
    scales(ch + C::kGroups);
    mbar_wait(bar0 + 8 * s, (it / ST) & 1, dead, p.err);
    if (__builtin_expect(__any_sync(0xffffffffu, dead), 0)) {
      // A wait ran out: leave no copy of this warp's in flight (the ring is
      // about to hold its sums, and shared memory ends with the CTA), and
      // make its rows NaN.
      if (lane == 0) {
        bool d2 = false;
        for (int k = 0; k < ST && ch + k * C::kGroups < c_end; ++k)
          mbar_wait(bar0 + 8 * ((it + k) % ST), ((it + k) / ST) & 1, d2, p.err);
      }
      __syncwarp();
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          m[x][y] = 0.f;  // a maximum, so that the joins take the sum in
          l[x][y] = __int_as_float(0x7fc00000);
        }
      break;
    }
    const uint32_t kb = ring + s * C::kStage, vb = kb + C::KC * C::kCol;
    // S^T: keys g and g + 8 of the chunk as rows, query rows as columns.
    float st[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) st[x][y] = 0.f;
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const int u = t + 4 * (i & 1);
      uint32_t a[4], c[4];
      const uint32_t at = kb + (i >> 1) * C::kCol + g * 128 + ((u ^ g) << 4);
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at));
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(at + 8 * 128));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int term = 0; term < 2; ++term)
            mma_e4m3(st[x], a[2 * h], c[2 * h], a[2 * h + 1], c[2 * h + 1],
                     qf[x][term][i][2 * h], qf[x][term][i][2 * h + 1]);
    }
    // V: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, LC columns of each 128.
    uint32_t vw[4][VB][C::LC / 4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = 2 * t + (k & 1) + 8 * (k >> 1);
#pragma unroll
      for (int c = 0; c < VB; ++c) {
        if constexpr (C::LC == 8) {
          asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                       : "=r"(vw[k][c][0]), "=r"(vw[k][c][1])
                       : "r"(vb + key * 128 + (((g >> 1) ^ (key & 7)) << 4) + (g & 1) * 8));
        } else {
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(vw[k][c][0]), "=r"(vw[k][c][1]), "=r"(vw[k][c][2]),
                         "=r"(vw[k][c][3])
                       : "r"(vb + c * C::kCol + key * 128 + ((g ^ (key & 7)) << 4)));
        }
      }
    }
    const int key0 = ch * 16;
    const bool full = key0 >= f_lo && key0 + 16 <= f_hi;
    if (!full) {
      // Keys that no row sees are zeros: what lies there is not data.
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = key0 + 2 * t + (k & 1) + 8 * (k >> 1);
        if (key < k_lo || key >= k_hi) {
#pragma unroll
          for (int c = 0; c < VB; ++c)
#pragma unroll
            for (int w = 0; w < C::LC / 4; ++w) vw[k][c][w] = 0u;
        }
      }
    }
    // Every lane has read the stage: the next chunk may take its place.
    __syncwarp();
    if (lane == 0 && ch + ST * C::kGroups < c_end) fetch(ch + ST * C::kGroups, s);

    // Logits in log2 units, plus the V scale's log2.
    bool raise = false;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const float a[2] = {qs[x][0] * ks * score, qs[x][1] * ks * score};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        float v = st[x][y] * a[y & 1];
        v = capped ? fmaf(cap_l2, kv8_tanh(v), L) : v + L;
        if (!full) {
          const int key = key0 + g + 8 * (y >> 1);
          v = key >= lo[x][y & 1] && key < hi[x][y & 1] ? v : -INFINITY;
        }
        st[x][y] = v;
      }
      raise |= fmaxf(st[x][0], st[x][2]) > m[x][0] + kKv8Lazy ||
               fmaxf(st[x][1], st[x][3]) > m[x][1] + kKv8Lazy;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float mx = fmaxf(st[x][y], st[x][2 + y]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          if (mx > m[x][y] + kKv8Lazy) {
            const float corr = ex2_approx(m[x][y] - mx);
            m[x][y] = mx;
            l[x][y] *= corr;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[x][j][y] *= corr;
              o[x][j][2 + y] *= corr;
            }
          }
        }
    }
    const float unscale = ex2_approx(-L);
    uint32_t pb[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const float mu0 = m[x][0] == -INFINITY ? 0.f : m[x][0] - kKv8Shift;
      const float mu1 = m[x][1] == -INFINITY ? 0.f : m[x][1] - kKv8Shift;
      const float p0 = ex2_approx(st[x][0] - mu0), p1 = ex2_approx(st[x][1] - mu1);
      const float p2 = ex2_approx(st[x][2] - mu0), p3 = ex2_approx(st[x][3] - mu1);
      l[x][0] = fmaf(p0 + p2, unscale, l[x][0]);
      l[x][1] = fmaf(p1 + p3, unscale, l[x][1]);
      pb[x][0] = transpose8(pack_f16(p0, p1));
      pb[x][1] = transpose8(pack_f16(p2, p3));
    }
    // O^T: tile j of column c has dims LC g + 2 j (rows 0-7) and + 1 (8-15).
#pragma unroll
    for (int c = 0; c < VB; ++c)
#pragma unroll
      for (int w = 0; w < C::LC / 4; ++w) {
        uint32_t lo2[4], hi2[4];  // tiles 2 w and 2 w + 1
        e4m3x4_to_f16(__byte_perm(vw[0][c][w], vw[1][c][w], 0x5140), lo2[0], lo2[1]);
        e4m3x4_to_f16(__byte_perm(vw[2][c][w], vw[3][c][w], 0x5140), lo2[2], lo2[3]);
        e4m3x4_to_f16(__byte_perm(vw[0][c][w], vw[1][c][w], 0x7362), hi2[0], hi2[1]);
        e4m3x4_to_f16(__byte_perm(vw[2][c][w], vw[3][c][w], 0x7362), hi2[2], hi2[3]);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const int j = c * C::LC / 2 + 2 * w;
          mma_f16(o[x][j], lo2, pb[x][0], pb[x][1]);
          mma_f16(o[x][j + 1], hi2, pb[x][0], pb[x][1]);
        }
      }
  }

  // The warps' sums meet in shared memory, each in its own ring.
  float* so = reinterpret_cast<float*>(smem);
  constexpr int kSo = C::kWarpBytes / 4;
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = 8 * x + 2 * t + y;
      float sum = l[x][y];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0 && vs == 0) {
        sml[(grp * 2 + 0) * NR + r] = m[x][y];
        sml[(grp * 2 + 1) * NR + r] = sum;
      }
      if (r < rows) {
        float* d = so + warp * kSo + r * C::OC + g * C::LC;
#pragma unroll
        for (int c = 0; c < VB; ++c)
#pragma unroll
          for (int j = 0; j < C::LC / 2; j += 2)
            *reinterpret_cast<float4*>(d + c * 128 + 2 * j) =
                make_float4(o[x][c * C::LC / 2 + j][y], o[x][c * C::LC / 2 + j][2 + y],
                            o[x][c * C::LC / 2 + j + 1][y], o[x][c * C::LC / 2 + j + 1][2 + y]);
      }
    }
  __syncthreads();
  // Each group's weight for each row, its sum times that, and the row's
  // maximum.
  float* row_m = sml + C::kGroups * 2 * NR;
  float* sw = row_m + NR;
  for (int i = threadIdx.x; i < NR * C::kGroups; i += C::kThreads) {
    const int r = i % NR, k = i / NR;
    float mt = -INFINITY;
#pragma unroll
    for (int x = 0; x < C::kGroups; ++x) mt = fmaxf(mt, sml[x * 2 * NR + r]);
    const float w = mt == -INFINITY ? 0.f : ex2_approx(sml[k * 2 * NR + r] - mt);
    const float part = sml[(k * 2 + 1) * NR + r] * w;
    if (k == 0) row_m[r] = mt;
    sml[(k * 2 + 1) * NR + r] = mt == -INFINITY ? 0.f : part;
    sw[i] = w;
  }
  __syncthreads();
  const long long cell = (static_cast<long long>(b) * p.c.Hkv + kvh) * p.tiles + tile;
  auto row_base = [&](int r) -> long long {
    const unsigned rr = static_cast<unsigned>(row0 + r), tok = rr / G;
    return (q_beg + static_cast<long long>(tok)) * p.out_row_stride +
           (kvh * p.G + static_cast<int>(rr - tok * G)) * static_cast<long long>(hd);
  };
  auto write_out = [&](int r, int e, float4 v, float inv) {
    const long long at = row_base(r) + e;
    if (p.out_f32)
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) =
          make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    else
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
          make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
  };
  auto fma4 = [](float4& a, const float4& x, float w) {
    a.x = fmaf(x.x, w, a.x);
    a.y = fmaf(x.y, w, a.y);
    a.z = fmaf(x.z, w, a.z);
    a.w = fmaf(x.w, w, a.w);
  };
  float* po = p.part_o + (cell * p.splits + split) * NR * hd;
  float* pml = p.part_ml + (cell * p.splits + split) * 2 * NR;
  for (int i = threadIdx.x; i < rows * (HDP / 4); i += C::kThreads) {
    const int r = i / (HDP / 4), e = i % (HDP / 4) * 4;
    if (e >= hd) continue;
    float lt = 0.f;
    float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < C::kGroups; ++k) {
      const float w = sw[k * NR + r];
      lt += sml[(k * 2 + 1) * NR + r];
      // A group without a chunk left nothing: its sums are zeros.
      fma4(ot, *reinterpret_cast<const float4*>(so + (k * C::VS + e / C::OC) * kSo + r * C::OC +
                                                e % C::OC), w);
    }
    if (p.splits == 1) {
      write_out(r, e, ot, __fdiv_rn(1.f, lt));
    } else {
      *reinterpret_cast<float4*>(po + r * hd + e) = ot;
      if (e == 0) {
        pml[r] = row_m[r];
        pml[NR + r] = lt;
      }
    }
  }
  if (p.splits == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int done = atomicAdd(p.tickets + cell, 1);
    smisc[0] = done == p.splits - 1;
    if (smisc[0]) p.tickets[cell] = 0;  // as the next call finds it
  }
  __syncthreads();
  if (!smisc[0]) return;
  __threadfence();
  // The last CTA joins the splits: weights first, as above, then the sums.
  po = p.part_o + cell * p.splits * NR * hd;
  pml = p.part_ml + cell * p.splits * 2 * NR;
  float* jm = so;                      // [splits][2][NR], then the weights
  float* jw = so + p.splits * 2 * NR;  // [splits][NR]
  for (int i = threadIdx.x; i < p.splits * 2 * NR; i += C::kThreads) jm[i] = __ldcg(pml + i);
  __syncthreads();
  for (int i = threadIdx.x; i < p.splits * NR; i += C::kThreads) {
    const int r = i % NR, k = i / NR;
    float mt = -INFINITY;
    for (int x = 0; x < p.splits; ++x) mt = fmaxf(mt, jm[x * 2 * NR + r]);
    jw[i] = mt == -INFINITY ? 0.f : ex2_approx(jm[k * 2 * NR + r] - mt);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (HDP / 4); i += C::kThreads) {
    const int r = i / (HDP / 4), e = i % (HDP / 4) * 4;
    if (e >= hd) continue;
    float lt = 0.f;
    float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < p.splits; ++k) {
      const float w = jw[k * NR + r];
      lt = fmaf(jm[(k * 2 + 1) * NR + r], w, lt);
      fma4(ot, __ldcg(reinterpret_cast<const float4*>(
                   po + (static_cast<long long>(k) * NR + r) * hd + e)), w);
    }
    write_out(r, e, ot, __fdiv_rn(1.f, lt));
  }
}

}  // namespace ca
