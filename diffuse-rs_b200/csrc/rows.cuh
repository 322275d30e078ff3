// rows.cuh -- the rows between a layer's products: residual addition, RMS
// norm, and output in bf16, fp32 or e4m3 with a scale for each row.
//
//   s = round(x + residual),  y = s w / sqrt(sum s^2 / cols + eps)
//   e4m3: scale = 2^k, the smallest k with amax |y| <= 448 2^k; y / scale is
//   exact in fp32, so each value is rounded once.
//
// A CTA takes a row at a time, the row in registers between the passes (sum of
// squares, largest magnitude, output), so HBM sees each input once and each
// output once. What a row waits for are its loads and two reductions over the
// CTA. rows_kernel, for rows that start on 16 bytes, therefore keeps the gain
// in registers, asks for the next row before it works on the one it has, and
// stays resident. Eight squares are added in fp32, the rest in 64 bits, as the
// reference adds all of them.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>

#include "e4m3.cuh"
#include "sm100.cuh"

namespace ca {

struct RowsParams {
  const void* x;
  const void* res;
  void* sum;
  const float* w;
  void* out;
  float* out_scale;
  long long x_stride, res_stride, sum_stride, out_stride;
  long long rows;
  int cols;
  int x_f32, res_f32, out_type;  // CA_TYPE_* of out
  int norm;
  float eps;
};

constexpr int kOutBf16 = 0, kOutF32 = 1, kOutE4m3 = 2;

// Eight elements i .. i + 7 of a row (16- or 32-byte loads).
__device__ __forceinline__ void load8(const void* row, int f32, long long i, float (&v)[8]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + i);
    const float4 a = p[0], b = p[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + i);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(u[k] << 16);
      v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                    pack_bf16(v[6], v[7]));
}

__device__ __forceinline__ void store8(void* row, int f32, long long i, const float (&v)[8]) {
  if (f32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + i);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(row) + i) = pack8(v);
  }
}

__device__ __forceinline__ float load1(const void* row, int f32, long long i) {
  return f32 ? static_cast<const float*>(row)[i]
             : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
}

__device__ __forceinline__ void store1(void* row, int f32, long long i, float v) {
  if (f32)
    static_cast<float*>(row)[i] = v;
  else
    static_cast<__nv_bfloat16*>(row)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ const void* row_at(const void* p, int f32, long long off) {
  return static_cast<const char*>(p) + (off << (f32 ? 2 : 1));
}
__device__ __forceinline__ void* row_at(void* p, int f32, long long off) {
  return static_cast<char*>(p) + (off << (f32 ? 2 : 1));
}

// Eight elements as they are loaded, and as fp32. They are read once: first to
// leave the caches (16384 x 4096 81.5 -> 76.5 us).
template <bool F32>
struct Raw8 {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* p, long long i) {
    if constexpr (F32) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
      a = __ldcs(q);
      b = __ldcs(q + 1);
    } else {
      a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i));
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (F32) {
        v[k] = __uint_as_float(x[k]);
        v[4 + k] = __uint_as_float(y[k]);
      } else {
        v[2 * k] = __uint_as_float(x[k] << 16);
        v[2 * k + 1] = __uint_as_float(x[k] & 0xffff0000u);
      }
    }
  }
};

// The largest over the CTA's `warps` warps; `red` holds a float for each.
__device__ __forceinline__ float cta_max_n(float v, float* red, int warps) {
  // (Of numbers that are not negative, whose bits have their order.)
  v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.f;
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

__device__ __forceinline__ double cta_sum_n(double v, double* red, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 1 / sqrt(x) for x >= 0: the approximation of fp32, and a Newton step in 64
// bits (1e-14 off), which takes a tenth of the instructions of a 64-bit root and
// division. Every thread of a row computes it.
__device__ __forceinline__ float inv_root(double x) {
  const float r0 = rsqrtf(static_cast<float>(x));
  if (!(r0 > 0.f && r0 < INFINITY)) return r0;
  const double r = r0;
  return static_cast<float>(r * fma(-0.5 * x * r, r, 1.5));
}

// C chunks of eight elements a thread; blockDim.x * C * 8 >= cols. At most 64
// registers (128 of five chunks), so that an SM holds 1024 threads; of three
// or five chunks the gain is read for each row (from L1). Forms of three and five
// chunks with a residual or fp32 rows spill 8 to 350 bytes. RES: 0 none, 1 bf16,
// 2 fp32.
template <bool XF32, int RES, int OUT, int C>
__global__ void __launch_bounds__(C >= 3 ? 512 : 1024, C == 3 ? 2 : 1)
    rows_kernel(const RowsParams p) {
  __shared__ double red_d[2][32];  // of a row and the next
  __shared__ float red[2][32];
  const int tid = threadIdx.x, cols = p.cols, warps = blockDim.x >> 5;
  int at[C];
  bool in[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    at[c] = (c * static_cast<int>(blockDim.x) + tid) * 8;
    in[c] = at[c] < cols;
  }
  dependency_wait();
  constexpr bool kHeld = C < 3;
  float g[kHeld ? C : 1][8];
#pragma unroll
  for (int c = 0; c < (kHeld ? C : 1); ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[c][j] = 1.f;
    if (kHeld && p.w && in[c]) load8(p.w, 1, at[c], g[c]);
  }
  Raw8<XF32> x[C];
  Raw8<RES == 2> res[C];
  auto fetch = [&](long long r) {
    const void* px = row_at(p.x, XF32, r * p.x_stride);
    const void* pr = RES ? row_at(p.res, RES == 2, r * p.res_stride) : nullptr;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (in[c]) {
        x[c].load(px, at[c]);
        if constexpr (RES != 0) res[c].load(pr, at[c]);
      }
    }
  };
  long long r = blockIdx.x;
  fetch(r);
  const double inv_cols = 1.0 / static_cast<double>(cols);
  for (int turn = 0; r < p.rows; r += gridDim.x, turn ^= 1) {
    float v[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x[c].get(v[c]);
      if constexpr (RES != 0) {
        float t[8];
        res[c].get(t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] += t[j];
        void* sum = row_at(p.sum, RES == 2, r * p.sum_stride);
        if constexpr (RES == 1) {
          const uint4 o = pack8(v[c]);
          if (in[c])
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(sum) + at[c]) = o;
          Raw8<false> back;
          back.a = o;
          back.get(v[c]);
        } else if (in[c]) {
          store8(sum, 1, at[c], v[c]);
        }
      }
      if (!in[c]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
      }
    }
    if (r + gridDim.x < p.rows) fetch(r + gridDim.x);
    float rs = 1.f;
    if (p.norm) {
      float s[C];
      double d = 0.0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        s[c] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[c] = fmaf(v[c][j], v[c][j], s[c]);
        d += static_cast<double>(s[c]);
      }
      const double ss = cta_sum_n(d, red_d[turn], warps);
      rs = inv_root(fma(ss, inv_cols, static_cast<double>(p.eps)));
    }
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!kHeld && p.w && in[c]) load8(p.w, 1, at[c], g[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[c][j] = v[c][j] * rs * g[kHeld ? c : 0][j];
        if (OUT == kOutE4m3) amax = fmaxf(amax, fabsf(v[c][j]));  // (NaN has no part)
      }
    }
    if constexpr (OUT != kOutE4m3) {
      void* out = row_at(p.out, OUT == kOutF32, r * p.out_stride);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (in[c]) store8(out, OUT == kOutF32, at[c], v[c]);
    } else {
      amax = cta_max_n(amax, red[turn], warps);
      if (amax == INFINITY) {  // infinities have no part in the scale, either
        amax = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (fabsf(v[c][j]) < INFINITY) amax = fmaxf(amax, fabsf(v[c][j]));
        __syncthreads();  // the infinity is read
        amax = cta_max_n(amax, red[turn], warps);
      }
      const int k = e4m3_exp(amax, kKv8MinExp, kKv8MaxExp);
      const float inv = exp2_int(-k);
      if (tid == 0) p.out_scale[r] = exp2_int(k);
      uint8_t* out = static_cast<uint8_t*>(p.out) + r * p.out_stride;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint32_t q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          q[h] = cvt_e4m3x2(v[c][4 * h] * inv, v[c][4 * h + 1] * inv) |
                 (cvt_e4m3x2(v[c][4 * h + 2] * inv, v[c][4 * h + 3] * inv) << 16);
        if (in[c]) *reinterpret_cast<uint2*>(out + at[c]) = make_uint2(q[0], q[1]);
      }
    }
  }
}

// The bits of N elements tid, tid + threads, ... of a row of `cols` that lie
// side by side across the threads; 0 behind its end. As fp32 they are these
// bits, of bf16 16 places up: a step of its own, so that what several tensors
// are asked for is on its way before the first is waited for.
template <int N>
__device__ __forceinline__ void load_strided(const void* row, int f32, int cols, uint32_t (&v)[N]) {
  const int tid = threadIdx.x, step = blockDim.x;
  if (f32) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      v[j] = tid + j * step < cols ? static_cast<const uint32_t*>(row)[tid + j * step] : 0;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      v[j] = tid + j * step < cols ? static_cast<const uint16_t*>(row)[tid + j * step] : 0;
  }
}
template <int N>
__device__ __forceinline__ void store_strided(void* row, int f32, int cols, const float (&v)[N]) {
  const int tid = threadIdx.x, step = blockDim.x;
  if (f32) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (tid + j * step < cols) static_cast<float*>(row)[tid + j * step] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (tid + j * step < cols)
        static_cast<__nv_bfloat16*>(row)[tid + j * step] = __float2bfloat16_rn(v[j]);
  }
}

// Rows of any alignment, element by element, N a thread (N * blockDim.x >=
// cols), otherwise as rows_kernel: held in registers between the passes, the
// gain among them. Several CTAs on an SM hide what a row waits for. (N = 20: 88
// bytes of spills.)
template <int N>
__global__ void __launch_bounds__(1024) rows_odd_kernel(const RowsParams p) {
  __shared__ double red_d[2][32];
  __shared__ float red[2][32];
  const int tid = threadIdx.x, step = blockDim.x, cols = p.cols, warps = blockDim.x >> 5;
  dependency_wait();
  uint32_t g[N];
#pragma unroll
  for (int j = 0; j < N; ++j) g[j] = __float_as_uint(1.f);
  if (p.w) load_strided(p.w, 1, cols, g);
  const double inv_cols = 1.0 / static_cast<double>(cols);
  const int x_up = p.x_f32 ? 0 : 16, res_up = p.res_f32 ? 0 : 16;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
    uint32_t x[N], t[N];
    load_strided(row_at(p.x, p.x_f32, r * p.x_stride), p.x_f32, cols, x);
    if (p.res) load_strided(row_at(p.res, p.res_f32, r * p.res_stride), p.res_f32, cols, t);
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __uint_as_float(x[j] << x_up);
    if (p.res) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        v[j] += __uint_as_float(t[j] << res_up);
        if (!p.res_f32) v[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
      }
      store_strided(row_at(p.sum, p.res_f32, r * p.sum_stride), p.res_f32, cols, v);
    }
    float rs = 1.f;
    if (p.norm) {
      double d = 0.0;
#pragma unroll
      for (int j0 = 0; j0 < N; j0 += 4) {
        float s = 0.f;
#pragma unroll
        for (int j = j0; j < (j0 + 4 < N ? j0 + 4 : N); ++j) s = fmaf(v[j], v[j], s);
        d += static_cast<double>(s);
      }
      rs = inv_root(fma(cta_sum_n(d, red_d[turn], warps), inv_cols, static_cast<double>(p.eps)));
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = v[j] * rs * __uint_as_float(g[j]);
      amax = fmaxf(amax, fabsf(v[j]));
    }
    if (p.out_type != kOutE4m3) {
      store_strided(row_at(p.out, p.out_type, r * p.out_stride), p.out_type, cols, v);
      continue;
    }
    amax = cta_max_n(amax, red[turn], warps);
    if (amax == INFINITY) {  // infinities have no part in the scale
      amax = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (fabsf(v[j]) < INFINITY) amax = fmaxf(amax, fabsf(v[j]));
      __syncthreads();  // the infinity is read
      amax = cta_max_n(amax, red[turn], warps);
    }
    const int k = e4m3_exp(amax, kKv8MinExp, kKv8MaxExp);
    const float inv = exp2_int(-k);
    if (tid == 0) p.out_scale[r] = exp2_int(k);
    uint8_t* out = static_cast<uint8_t*>(p.out) + r * p.out_stride;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (tid + j * step < cols)
        out[tid + j * step] = static_cast<uint8_t>(cvt_e4m3x2(v[j] * inv, 0.f));
  }
}

// Rows of more columns than registers hold, of any alignment: elements one by
// one, side by side across the threads. Each thread goes back to its
// own elements, which it finds in the sum (or in x) as it left them.
__global__ void __launch_bounds__(256) rows_any_kernel(const RowsParams p) {
  __shared__ double red_d[2][32];
  __shared__ float red[2][32];
  dependency_wait();
  const int tid = threadIdx.x, cols = p.cols;
  int turn = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
    const void* x = row_at(p.x, p.x_f32, r * p.x_stride);
    const void* res = p.res ? row_at(p.res, p.res_f32, r * p.res_stride) : nullptr;
    void* sum = p.res ? row_at(p.sum, p.res_f32, r * p.sum_stride) : nullptr;
    double ss = 0.0;
    if (p.res || p.norm) {
#pragma unroll 4
      for (int i = tid; i < cols; i += 256) {
        float v = load1(x, p.x_f32, i);
        if (p.res) {
          v += load1(res, p.res_f32, i);
          if (!p.res_f32) v = __bfloat162float(__float2bfloat16_rn(v));
          store1(sum, p.res_f32, i, v);
        }
        ss += static_cast<double>(v * v);
      }
    }
    const void* from = p.res ? sum : x;
    const int from_f32 = p.res ? p.res_f32 : p.x_f32;
    float rs = 1.f;
    if (p.norm) {
      ss = cta_sum_n(ss, red_d[turn], 8);
      rs = inv_root(ss / cols + static_cast<double>(p.eps));
    }
    auto value = [&](int i) {
      const float v = load1(from, from_f32, i) * rs;
      return p.w ? v * p.w[i] : v;
    };
    if (p.out_type != kOutE4m3) {
      void* out = row_at(p.out, p.out_type, r * p.out_stride);
#pragma unroll 4
      for (int i = tid; i < cols; i += 256) store1(out, p.out_type, i, value(i));
      continue;
    }
    float amax = 0.f;
#pragma unroll 4
    for (int i = tid; i < cols; i += 256) {
      const float m = fabsf(value(i));
      amax = fmaxf(amax, m < INFINITY ? m : 0.f);
    }
    amax = cta_max_n(amax, red[turn], 8);
    const int k = e4m3_exp(amax, kKv8MinExp, kKv8MaxExp);
    const float inv = exp2_int(-k);
    if (tid == 0) p.out_scale[r] = exp2_int(k);
    uint8_t* out = static_cast<uint8_t*>(p.out) + r * p.out_stride;
#pragma unroll 4
    for (int i = tid; i < cols; i += 256)
      out[i] = static_cast<uint8_t>(cvt_e4m3x2(value(i) * inv, 0.f));
  }
}

}  // namespace ca
