// rows.cuh -- the rows between a layer's products: residual addition, RMS
// norm, and output in bf16, fp32 or e4m3 with a scale for each row.
//
//   s = round(x + residual),  y = s w / sqrt(sum s^2 / cols + eps)
//   e4m3: scale = 2^k, the smallest k with amax |y| <= 448 2^k; y / scale is
//   exact in fp32, so each value is rounded once.
//
// One CTA per row, the row in registers between the passes (sum of squares,
// largest magnitude, output), so HBM sees each input once and each output
// once; the two reductions over the CTA are what a row waits for, and several
// CTAs per SM hide them. Sums in fp32: a thread adds at most 32 squares, the
// rest is a tree.
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

// A sum or a maximum over the CTA's NT threads; `red` holds NT / 32 floats
// that no other reduction uses.
template <int NT, bool MAX>
__device__ __forceinline__ float cta_reduce(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, t) : v + t;
  }
  if (NT == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  return v;
}

// Rows of at most NT * C * 8 columns, eight a chunk, C chunks a thread. VEC:
// every row of every tensor starts on 16 bytes and cols is a multiple of 8;
// otherwise elements are taken one by one, side by side across the threads.
template <int NT, int C, bool VEC>
__global__ void __launch_bounds__(NT) rows_kernel(const RowsParams p) {
  __shared__ float red[2][NT / 32];
  dependency_wait();
  const long long r = blockIdx.x;
  const int tid = threadIdx.x, cols = p.cols;
  const void* x = row_at(p.x, p.x_f32, r * p.x_stride);
  float v[C][8];
  auto elem = [&](int c, int j) { return VEC ? (c * NT + tid) * 8 + j : (c * 8 + j) * NT + tid; };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (VEC) {
      if (elem(c, 0) < cols) {
        load8(x, p.x_f32, elem(c, 0), v[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = elem(c, j) < cols ? load1(x, p.x_f32, elem(c, j)) : 0.f;
    }
  }
  if (p.res) {
    const void* res = row_at(p.res, p.res_f32, r * p.res_stride);
    void* sum = row_at(p.sum, p.res_f32, r * p.sum_stride);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float t[8];
      if (VEC) {
        if (elem(c, 0) < cols) {
          load8(res, p.res_f32, elem(c, 0), t);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[c][j] += t[j];
            if (!p.res_f32) v[c][j] = __bfloat162float(__float2bfloat16_rn(v[c][j]));
          }
          store8(sum, p.res_f32, elem(c, 0), v[c]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (elem(c, j) < cols) {
            v[c][j] += load1(res, p.res_f32, elem(c, j));
            if (!p.res_f32) v[c][j] = __bfloat162float(__float2bfloat16_rn(v[c][j]));
            store1(sum, p.res_f32, elem(c, j), v[c][j]);
          }
        }
      }
    }
  }
  float rs = 1.f;
  if (p.norm) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[c][j], v[c][j], ss);
    ss = cta_reduce<NT, false>(ss, red[0]);
    rs = 1.f / sqrtf(ss / static_cast<float>(cols) + p.eps);
  }
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float g[8];
    if (p.w) {
      if (VEC) {
        if (elem(c, 0) < cols) load8(p.w, 1, elem(c, 0), g);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = elem(c, j) < cols ? p.w[elem(c, j)] : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (p.norm) v[c][j] *= rs;
      if (p.w) v[c][j] *= g[j];
      const bool in = VEC ? elem(c, 0) < cols : elem(c, j) < cols;
      // Infinities and NaN have no part in the scale.
      if (in && fabsf(v[c][j]) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(v[c][j]));
    }
  }
  if (p.out_type != kOutE4m3) {
    void* out = row_at(p.out, p.out_type, r * p.out_stride);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (VEC) {
        if (elem(c, 0) < cols) store8(out, p.out_type, elem(c, 0), v[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (elem(c, j) < cols) store1(out, p.out_type, elem(c, j), v[c][j]);
      }
    }
    return;
  }
  amax = cta_reduce<NT, true>(amax, red[1]);
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
    if (VEC) {
      if (elem(c, 0) < cols) *reinterpret_cast<uint2*>(out + elem(c, 0)) = make_uint2(q[0], q[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (elem(c, j) < cols) out[elem(c, j)] = static_cast<uint8_t>(q[j >> 2] >> (8 * (j & 3)));
    }
  }
}

}  // namespace ca
