// attn_kv8_rows.cuh -- attention of a few query rows over the 8-bit cache.
//
// One CTA takes 16 query rows (token, head-of-the-group pairs, token-major)
// of one (sequence, kv head) and one stretch of its keys. Each warp walks
// chunks of 16 keys of that stretch on its own, K and V going from HBM
// straight to registers in the layout the tensor core wants: the order of
// the head dims inside Q K^T, and of the output columns inside P V, is free,
// so every lane loads whole 16-byte pieces of a row and turns them into f16
// (exact for e4m3) without a shuffle or shared memory.
//
// Mathematics. A cached value is e4m3 * scale, one scale for each block of
// keys. With a = scale_k(block) * scale * log2 e and L = log2 scale_v(block),
//   t = a (q . k8) + L,   p = 2^(t - m),
//   O = sum p v8,         l = sum p 2^-L,     out = O / l
// with m a running bound of t: the V scale rides in the exponent, so P V
// runs on the held values, and only l has to take it out again. A row of Q
// is scaled by a power of two into [1, 2) before it is rounded to f16, which
// keeps bf16's 8 bits down to 2^-24 of the row's largest value. P is f16 at
// up to 2^15 (2^7 for t = m, and m is only moved when t passes it by 8), so
// weights down to 2^-31 of the largest count; sums and maxima are fp32.
//
// Bound by HBM: 2 hd bytes a key. Long caches are split over CTAs; the last
// CTA of a row tile to finish joins their partial sums in order, so results
// do not depend on which that was.
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
  float* part_o;       // [tile][split][16][hd]
  float* part_ml;      // [tile][split][2][16]
  int* tickets;        // [tile], zero between calls
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

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr float kKv8Shift = 7.f;  // P's f16 exponent for t = m
constexpr float kKv8Lazy = 8.f;   // how far t may pass m before m moves

// log2 of a V scale, kept where 2^L and 2^-L are both finite.
__device__ __forceinline__ float kv8_log2(float s) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return fminf(fmaxf(y, -100.f), 120.f);
}

// HDP: head_dim padded to 64, 128, 256 or 512. VS warps share a stretch of
// keys, each with 128 of the output columns (and all of Q K^T).
template <int HDP>
struct RowsCfg {
  static constexpr int VS = HDP <= 128 ? 1 : HDP / 128;
  static constexpr int kWarps = 8;
  static constexpr int kGroups = kWarps / VS;           // key-walking groups
  static constexpr int VC = HDP / VS;                   // output columns of a warp (64 or 128)
  static constexpr int KU = HDP / 64;                   // 16-byte pieces of a K row per lane
  static constexpr int kQBytes = 16 * HDP * 2;          // f16 fragments of the 16 rows
  static constexpr int kOBytes = kGroups * 16 * HDP * 4;
  static constexpr int kOffML = kQBytes + kOBytes;
  static constexpr int kSmem = kOffML + kGroups * 2 * 16 * 4 + 64;
  // Chunks in registers: one being used and, where they fit, one in flight.
  static constexpr int kBufs = HDP <= 256 ? 2 : 1;
};

template <int HDP>
__global__ void __launch_bounds__(256, 1) attn_kv8_rows_kernel(const Kv8AttnParams p) {
  using C = RowsCfg<HDP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint32_t* sq = reinterpret_cast<uint32_t*>(smem);
  float* so = reinterpret_cast<float*>(smem + C::kQBytes);
  float* sml = reinterpret_cast<float*>(smem + C::kOffML);
  int* smisc = reinterpret_cast<int*>(smem + C::kOffML + C::kGroups * 2 * 16 * 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int grp = warp / C::VS, vb = warp % C::VS;
  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int hd = p.c.hd;

  const int q_beg = p.cu_q ? p.cu_q[b] : b * p.sq;
  const int q_len = p.cu_q ? p.cu_q[b + 1] - q_beg : p.sq;
  const long long n_rows = static_cast<long long>(q_len) * p.G;
  const long long row0 = static_cast<long long>(tile) * 16;
  if (row0 >= n_rows) return;
  const int rows = static_cast<int>(min(16ll, n_rows - row0));
  const int len = p.kv_len ? min(max(p.kv_len[b], 0), p.c.n_total) : p.c.n_total;

  // Rows g and g + 8 of this lane: interval, and the tile's hull.
  int lo[2], hi[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = g + 8 * x;
    lo[x] = hi[x] = 0;
    if (r < rows) {
      const int tok = static_cast<int>((row0 + r) / p.G);
      const int pos = p.q_pos ? p.q_pos[q_beg + tok] : len - q_len + tok;
      kv8_interval(pos, len, p.window, p.seq_prefix ? p.seq_prefix[b] : p.causal_prefix, lo[x],
                   hi[x]);
    }
  }
  // Rows that see nothing do not widen the hull; rows past the end neither.
  const int any0 = lo[0] < hi[0], any1 = lo[1] < hi[1];
  int k_lo = min(any0 ? lo[0] : INT_MAX, any1 ? lo[1] : INT_MAX);
  int k_hi = max(any0 ? hi[0] : 0, any1 ? hi[1] : 0);
  const bool r0 = g < rows, r1 = g + 8 < rows;
  int f_lo = max(r0 ? lo[0] : 0, r1 ? lo[1] : 0);
  int f_hi = min(r0 ? hi[0] : INT_MAX, r1 ? hi[1] : INT_MAX);
  k_lo = __reduce_min_sync(0xffffffffu, k_lo);
  k_hi = __reduce_max_sync(0xffffffffu, k_hi);
  f_lo = __reduce_max_sync(0xffffffffu, f_lo);  // every row sees [f_lo, f_hi)
  f_hi = __reduce_min_sync(0xffffffffu, f_hi);
  // This CTA's chunks of 16 keys.
  int c_beg = 0, c_end = 0;
  if (k_lo < k_hi) {
    const int first = k_lo >> 4, n = ((k_hi + 15) >> 4) - first;
    const int per = (n + p.splits - 1) / p.splits;
    c_beg = first + min(n, split * per);
    c_end = first + min(n, (split + 1) * per);
  }

  // Q: each row scaled by a power of two, rounded to f16, in fragment order
  // [k-step][lane][4]: step 4 i + c of lane (g, t) takes head dims
  // (t + 4 i) 16 + 4 c .. + 3 of rows g and g + 8.
  float qs[2];
  {
    __shared__ int s_exp[16];
    for (int r = warp; r < 16; r += C::kWarps) {
      float amax = 0.f;
      const __nv_bfloat16* src = nullptr;
      if (r < rows) {
        const long long rr = row0 + r;
        src = p.q + (q_beg + rr / p.G) * p.q_row_stride + (kvh * p.G + rr % p.G) * hd;
        for (int e = lane * 4; e < hd; e += 128) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + e));
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(__uint_as_float(w.x << 16)),
                                         fabsf(__uint_as_float(w.x & 0xffff0000u))),
                                   fmaxf(fabsf(__uint_as_float(w.y << 16)),
                                         fabsf(__uint_as_float(w.y & 0xffff0000u)))));
        }
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
      const int ex = min(max(static_cast<int>(top >> 23) - 127, -100), 120);
      if (lane == 0) s_exp[r] = ex;
      const float inv = exp2_int(-ex);
      for (int e = lane * 4; e < HDP; e += 128) {
        uint32_t w0 = 0u, w1 = 0u;
        if (r < rows && e < hd) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + e));
          w0 = pack_f16(__uint_as_float(w.x << 16) * inv, __uint_as_float(w.x & 0xffff0000u) * inv);
          w1 = pack_f16(__uint_as_float(w.y << 16) * inv, __uint_as_float(w.y & 0xffff0000u) * inv);
        }
        const int piece = e >> 4, c = (e >> 2) & 3;
        const int step = (piece >> 2) * 4 + c, tt = piece & 3;
        uint32_t* d = sq + (step * 32 + (r & 7) * 4 + tt) * 4 + (r >> 3);
        d[0] = w0;
        d[2] = w1;
      }
    }
    __syncthreads();
    qs[0] = exp2_int(s_exp[g]);
    qs[1] = exp2_int(s_exp[g + 8]);
  }

  const uint8_t* kb = p.c.k + static_cast<long long>(b) * p.c.n_total * p.c.row_stride +
                      static_cast<long long>(kvh) * hd;
  const uint8_t* vbase = p.c.v + static_cast<long long>(b) * p.c.n_total * p.c.row_stride +
                         static_cast<long long>(kvh) * hd;
  const float* ksc = p.c.k_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
  const float* vsc = p.c.v_scale + static_cast<long long>(b) * p.c.n_blocks * p.c.Hkv + kvh;
  const int shift = 31 - __clz(p.c.T);

  constexpr int NT = C::VC / 8;  // 8-column tiles of O
  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[j][x] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float cap_l2 = p.softcap * 1.4426950408889634f;
  const float inv_cap = p.softcap != 0.f ? p.scale / p.softcap : 0.f;

  // K piece i of key n: 16 bytes at head dim (t + 4 i) 16. V: keys 2 t,
  // 2 t + 1, 2 t + 8, 2 t + 9 of the chunk, columns g 16 (g 8 at 64) on.
  uint4 kr[C::kBufs][2][C::KU];
  uint4 vr[C::kBufs][4];
  float sc[C::kBufs][2];
  auto load = [&](int ch, int buf) {
    const int key0 = ch * 16;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int key = key0 + 8 * n + g;
      const uint8_t* a = kb + static_cast<long long>(key) * p.c.row_stride;
#pragma unroll
      for (int i = 0; i < C::KU; ++i) {
        const int e = (t + 4 * i) * 16;
        kr[buf][n][i] = key < k_hi && e < hd ? __ldg(reinterpret_cast<const uint4*>(a + e))
                                            : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int key = key0 + 2 * t + (x & 1) + 8 * (x >> 1);
      const uint8_t* a = vbase + static_cast<long long>(key) * p.c.row_stride;
      if constexpr (C::VC == 64) {
        const int e = g * 8;
        const uint2 w = key >= k_lo && key < k_hi && e < hd ? __ldg(reinterpret_cast<const uint2*>(a + e))
                                            : make_uint2(0u, 0u);
        vr[buf][x] = make_uint4(w.x, w.y, 0u, 0u);
      } else {
        const int e = vb * 128 + g * 16;
        vr[buf][x] = key >= k_lo && key < k_hi && e < hd ? __ldg(reinterpret_cast<const uint4*>(a + e))
                                         : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    const long long blk = static_cast<long long>(key0 >> shift) * p.c.Hkv;
    sc[buf][0] = __ldg(ksc + blk);
    sc[buf][1] = __ldg(vsc + blk);
  };

  auto chunk = [&](int ch, int buf) {
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] = 0.f;
#pragma unroll
    for (int i = 0; i < C::KU; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 a = *reinterpret_cast<const uint4*>(sq + ((i * 4 + c) * 32 + lane) * 4);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint4& w4 = kr[buf][n][i];
          const uint32_t w = c == 0 ? w4.x : c == 1 ? w4.y : c == 2 ? w4.z : w4.w;
          uint32_t b0, b1;
          e4m3x4_to_f16(w, b0, b1);
          mma_f16(s[n], a.x, a.y, a.z, a.w, b0, b1);
        }
      }
    }
    // Logits in log2 units, plus the V scale's log2.
    const float L = kv8_log2(sc[buf][1]);
    const int key0 = ch * 16 + 2 * t;
    const bool full = ch * 16 >= f_lo && ch * 16 + 16 <= f_hi;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float raw = s[n][x] * (qs[x >> 1] * sc[buf][0]);
        float y;
        if (p.softcap != 0.f) y = fmaf(cap_l2, tanh_via_exp2(raw * inv_cap), L);
        else y = fmaf(raw, p.scale_log2, L);
        const int key = key0 + 8 * n + (x & 1);
        s[n][x] = full || (key >= lo[x >> 1] && key < hi[x >> 1]) ? y : -INFINITY;
      }
    float mx[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      mx[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
    if (__any_sync(0xffffffffu, mx[0] > m[0] + kKv8Lazy || mx[1] > m[1] + kKv8Lazy)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        if (mx[r] > m[r] + kKv8Lazy) {
          const float corr = ex2_approx(m[r] - mx[r]);
          m[r] = mx[r];
          l[r] *= corr;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            o[j][2 * r] *= corr;
            o[j][2 * r + 1] *= corr;
          }
        }
      }
    }
    const float mu0 = m[0] == -INFINITY ? 0.f : m[0] - kKv8Shift;
    const float mu1 = m[1] == -INFINITY ? 0.f : m[1] - kKv8Shift;
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n][0] = ex2_approx(s[n][0] - mu0);
      s[n][1] = ex2_approx(s[n][1] - mu0);
      s[n][2] = ex2_approx(s[n][2] - mu1);
      s[n][3] = ex2_approx(s[n][3] - mu1);
      sum0 += s[n][0] + s[n][1];
      sum1 += s[n][2] + s[n][3];
    }
    const float unscale = ex2_approx(-L);
    l[0] = fmaf(sum0, unscale, l[0]);
    l[1] = fmaf(sum1, unscale, l[1]);
    const uint32_t a0 = pack_f16(s[0][0], s[0][1]), a1 = pack_f16(s[0][2], s[0][3]);
    const uint32_t a2 = pack_f16(s[1][0], s[1][1]), a3 = pack_f16(s[1][2], s[1][3]);
#pragma unroll
    for (int w = 0; w < NT / 4; ++w) {
      auto word = [&](int x) -> uint32_t {
        const uint4& v4 = vr[buf][x];
        return w == 0 ? v4.x : w == 1 ? v4.y : w == 2 ? v4.z : v4.w;
      };
      const uint32_t p01 = word(0), q01 = word(1), p89 = word(2), q89 = word(3);
      uint32_t b0[4], b1[4];
      e4m3x4_to_f16(__byte_perm(p01, q01, 0x5140), b0[0], b0[1]);
      e4m3x4_to_f16(__byte_perm(p01, q01, 0x7362), b0[2], b0[3]);
      e4m3x4_to_f16(__byte_perm(p89, q89, 0x5140), b1[0], b1[1]);
      e4m3x4_to_f16(__byte_perm(p89, q89, 0x7362), b1[2], b1[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f16(o[4 * w + j], a0, a1, a2, a3, b0[j], b1[j]);
    }
  };

  if constexpr (C::kBufs == 2) {
    int ch = c_beg + grp;
    if (ch < c_end) load(ch, 0);
    while (ch < c_end) {
      const int nx = ch + C::kGroups;
      if (nx < c_end) load(nx, 1);
      chunk(ch, 0);
      if (nx >= c_end) break;
      const int nn = nx + C::kGroups;
      if (nn < c_end) load(nn, 0);
      chunk(nx, 1);
      ch = nn;
    }
  } else {
    for (int ch = c_beg + grp; ch < c_end; ch += C::kGroups) {
      load(ch, 0);
      chunk(ch, 0);
    }
  }

  // The groups' sums meet in shared memory. Lane (g, t) holds, of rows g and
  // g + 8, columns 2 t NT .. + 2 NT - 1 of its warp's VC: tile j's first
  // column is 2 t NT + j, its second NT further.
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t == 0 && vb == 0) {
      sml[(grp * 2 + 0) * 16 + g + 8 * r] = m[r];
      sml[(grp * 2 + 1) * 16 + g + 8 * r] = l[r];
    }
    float* d = so + (grp * 16 + g + 8 * r) * HDP + vb * C::VC + 2 * t * NT;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      d[j] = o[j][2 * r];
      d[NT + j] = o[j][2 * r + 1];
    }
  }
  __syncthreads();
  const long long cell = (static_cast<long long>(b) * p.c.Hkv + kvh) * p.tiles + tile;
  auto write_out = [&](int r, int e, float v) {
    const long long rr = row0 + r;
    const long long at = (q_beg + rr / p.G) * p.out_row_stride + (kvh * p.G + rr % p.G) * hd + e;
    if (p.out_f32) static_cast<float*>(p.out)[at] = v;
    else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  };
  float* po = p.part_o + (cell * p.splits + split) * 16 * hd;
  float* pml = p.part_ml + (cell * p.splits + split) * 32;
  for (int i = threadIdx.x; i < rows * hd; i += 256) {
    const int r = i / hd, e = i - r * hd;
    float mt = -INFINITY;
#pragma unroll
    for (int k = 0; k < C::kGroups; ++k) mt = fmaxf(mt, sml[k * 32 + r]);
    float lt = 0.f, ot = 0.f;
    if (mt != -INFINITY) {
#pragma unroll
      for (int k = 0; k < C::kGroups; ++k) {
        const float w = ex2_approx(sml[k * 32 + r] - mt);
        lt = fmaf(sml[k * 32 + 16 + r], w, lt);
        ot = fmaf(so[(k * 16 + r) * HDP + e], w, ot);
      }
    }
    if (p.splits == 1) {
      write_out(r, e, __fdiv_rn(ot, lt));
    } else {
      po[i] = ot;
      if (e == 0) {
        pml[r] = mt;
        pml[16 + r] = lt;
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
  po = p.part_o + cell * p.splits * 16 * hd;
  pml = p.part_ml + cell * p.splits * 32;
  for (int i = threadIdx.x; i < rows * hd; i += 256) {
    const int r = i / hd, e = i - r * hd;
    float mt = -INFINITY;
    for (int k = 0; k < p.splits; ++k) mt = fmaxf(mt, __ldcg(pml + k * 32 + r));
    float lt = 0.f, ot = 0.f;
    if (mt != -INFINITY) {
      for (int k = 0; k < p.splits; ++k) {
        const float w = ex2_approx(__ldcg(pml + k * 32 + r) - mt);
        lt = fmaf(__ldcg(pml + k * 32 + 16 + r), w, lt);
        ot = fmaf(__ldcg(po + static_cast<long long>(k) * 16 * hd + i), w, ot);
      }
    }
    write_out(r, e, __fdiv_rn(ot, lt));
  }
}

}  // namespace ca
