// Residual addition and RMSNorm of BF16 rows in one pass, with BF16 or MXFP8
// rows out, and its backward pass.
//
//   h = x + res                      stored in res's type (BF16 or FP32); no res: h = x
//   s = 1 / sqrt(mean(h^2) + eps)    of h as stored, so a backward pass needs h alone
//   y = h * s * w
//
// and, with z = dy * w,
//
//   dh = s * (z - h * s^2 * mean(z * h)) + dsum      dx = bf16(dh), dres = dh
//   dw = sum over rows of dy * h * s
//
// Everything between the loads and the stores is FP32; the only roundings are
// the stored sum and the result (unlike rmsnorm_rows_kernel, which repeats the
// BF16 roundings between the products of the module it replaces).
//
// The pass is bound by HBM: each tensor is read or written once.  A row is
// held in the registers of 32 * WPR threads (NC 16-byte chunks of BF16 each),
// so the statistics cost no second read; a CTA walks rows with a stride, which
// keeps w in registers for all of them.  MXFP8: four neighbouring lanes hold a
// block of 32, so its largest magnitude is two shuffles.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "mx.cuh"
#include "sm100.cuh"

namespace spx {

namespace {

constexpr int kNormThreads = 512;

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    v[2 * q] = __uint_as_float(w[q] << 16);
    v[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * q], v[2 * q + 1]);
    w[q] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void load8(const void* base, int64_t at, bool f32, float (&v)[8]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at), v);
  }
}

__device__ __forceinline__ void store8(void* base, int64_t at, bool f32, const float (&v)[8]) {
  if (f32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = pack8(v);
  }
}

// Sum of `n` floats over the 32 * WPR threads of a row.  `part` holds
// [2][rows per CTA][WPR][n]; the two halves alternate from row to row, so one
// barrier a row is enough.
template <int WPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* part, int group, int wr, int lane, uint32_t turn) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] += __shfl_xor_sync(0xFFFFFFFFu, s[j], off);
  }
  if constexpr (WPR > 1) {
    constexpr int kGroups = kNormThreads / (32 * WPR);
    float* p = part + ((turn & 1u) * kGroups + group) * WPR * N;
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < N; ++j) p[wr * N + j] = s[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) t += p[w * N + j];
      s[j] = t;
    }
  }
}

}  // namespace

template <int WPR, int NC>
__global__ void __launch_bounds__(kNormThreads) add_norm_kernel(const AddNormArgs a) {
  constexpr int kGroups = kNormThreads / (32 * WPR);
  __shared__ float part[2 * kGroups * WPR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wr = warp % WPR;
  const int nchunks = a.d / 8;
  const float inv_d = 1.0f / static_cast<float>(a.d);
  uint4 wv[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * WPR + wr) * 32 + lane;
    wv[i] = c < nchunks ? __ldg(reinterpret_cast<const uint4*>(a.w) + c) : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t turn = 0;
  // every warp of the CTA runs the same number of rows (row_sum has a barrier)
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * kGroups, ++turn) {
    const int64_t row = row0 + group;
    const bool live = row < a.rows;
    float h[NC][8];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (live && c < nchunks) {
        load8(a.x, row * a.ld_x + c * 8, false, h[i]);
        if (a.res != nullptr) {
          float r[8];
          load8(a.res, row * a.ld_res + c * 8, a.res_f32 != 0, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            h[i][j] += r[j];
            if (a.res_f32 == 0) h[i][j] = round_bf16(h[i][j]);
          }
          store8(a.sum, row * a.d + c * 8, a.res_f32 != 0, h[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(h[i][j], h[i][j], s[0]);
    }
    row_sum<WPR, 1>(s, part, group, wr, lane, turn);
    const float r = 1.0f / sqrtf(s[0] * inv_d + a.eps);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      const bool in = live && c < nchunks;
      float wf[8], y[8];
      unpack8(wv[i], wf);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = h[i][j] * r * wf[j];
      if (a.mx_values == nullptr) {
        if (in) store8(a.y, row * a.d + c * 8, false, y);
      } else {
        // blocks of 32 = four lanes; all lanes take part in the shuffles (d % 32 == 0, so a block is wholly in or out)
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        const uint32_t sb = mx_scale_byte(amax);
        const float m = mx_multiplier(sb);
        if (in) {
          const uint32_t q0 = mx_e4m3x2(y[0] * m, y[1] * m) | (mx_e4m3x2(y[2] * m, y[3] * m) << 16);
          const uint32_t q1 = mx_e4m3x2(y[4] * m, y[5] * m) | (mx_e4m3x2(y[6] * m, y[7] * m) << 16);
          *reinterpret_cast<uint2*>(a.mx_values + row * a.d + c * 8) = make_uint2(q0, q1);
          if ((c & 3) == 0) a.mx_scales[row * (a.d / kMxBlock) + c / 4] = static_cast<uint8_t>(sb);
        }
      }
    }
  }
}

// dw is summed per thread over the CTA's rows, then over the CTA's row groups
// in shared memory, then over CTAs by norm_dw_kernel: a fixed order, no atomics.
template <int WPR, int NC>
__global__ void __launch_bounds__(kNormThreads) add_norm_backward_kernel(const AddNormBackwardArgs a) {
  constexpr int kGroups = kNormThreads / (32 * WPR);
  constexpr int kCols = 32 * WPR * 8;  // columns of one chunk index
  __shared__ float part[2 * kGroups * WPR * 2];
  __shared__ float s_dw[kGroups > 1 ? kCols * (kGroups > 8 ? 8 : kGroups) : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wr = warp % WPR;
  const int nchunks = a.d / 8;
  const float inv_d = 1.0f / static_cast<float>(a.d);
  uint4 wv[NC];
  float dw[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * WPR + wr) * 32 + lane;
    wv[i] = c < nchunks ? __ldg(reinterpret_cast<const uint4*>(a.w) + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
  }
  uint32_t turn = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * kGroups, ++turn) {
    const int64_t row = row0 + group;
    const bool live = row < a.rows;
    float h[NC][8];
    uint4 g[NC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (live && c < nchunks) {
        g[i] = *reinterpret_cast<const uint4*>(a.dy + row * a.ld_dy + c * 8);
        load8(a.h, row * a.ld_h + c * 8, a.res_f32 != 0, h[i]);
      } else {
        g[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
      }
      float wf[8], gf[8];
      unpack8(wv[i], wf);
      unpack8(g[i], gf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[0] = fmaf(h[i][j], h[i][j], s[0]);
        s[1] = fmaf(gf[j] * wf[j], h[i][j], s[1]);
      }
    }
    row_sum<WPR, 2>(s, part, group, wr, lane, turn);
    const float r = 1.0f / sqrtf(s[0] * inv_d + a.eps);
    const float k = r * r * s[1] * inv_d;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (!live || c >= nchunks) continue;
      float wf[8], gf[8], dh[8];
      unpack8(wv[i], wf);
      unpack8(g[i], gf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] = fmaf(gf[j] * h[i][j], r, dw[i][j]);
        dh[j] = r * (gf[j] * wf[j] - h[i][j] * k);
      }
      if (a.dsum != nullptr) {
        float ds[8];
        load8(a.dsum, row * a.ld_dsum + c * 8, a.res_f32 != 0, ds);
#pragma unroll
        for (int j = 0; j < 8; ++j) dh[j] += ds[j];
      }
      store8(a.dx, row * a.d + c * 8, false, dh);
      if (a.dres != nullptr) store8(a.dres, row * a.d + c * 8, true, dh);
    }
  }
  if (a.dw_part == nullptr) return;
  float* out = a.dw_part + static_cast<int64_t>(blockIdx.x) * a.d;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * WPR + wr) * 32 + lane;
    if constexpr (kGroups > 1) {
      constexpr int kSlots = kGroups > 8 ? 8 : kGroups;
      __syncthreads();
      if constexpr (kGroups > kSlots) {  // the upper groups first hand theirs down
        if (group >= kSlots) {
#pragma unroll
          for (int j = 0; j < 8; ++j) s_dw[(group - kSlots) * kCols + j * (32 * WPR) + wr * 32 + lane] = dw[i][j];
        }
        __syncthreads();
        if (group < kSlots) {
#pragma unroll
          for (int j = 0; j < 8; ++j) dw[i][j] += s_dw[group * kCols + j * (32 * WPR) + wr * 32 + lane];
        }
        __syncthreads();
      }
      if (group < kSlots) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s_dw[group * kCols + j * (32 * WPR) + wr * 32 + lane] = dw[i][j];
      }
      __syncthreads();
      if (group == 0 && c < nchunks) {
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[j] = 0.0f;
#pragma unroll
          for (int q = 0; q < kSlots; ++q) t[j] += s_dw[q * kCols + j * (32 * WPR) + wr * 32 + lane];
        }
        store8(out, c * 8, true, t);
      }
    } else if (c < nchunks) {
      store8(out, c * 8, true, dw[i]);
    }
  }
}

// dw[c] = bf16(sum over the CTAs' partials), 32 columns x 8 row lanes a block.
__global__ void __launch_bounds__(256) norm_dw_kernel(const float* __restrict__ part, int nparts, int d,
                                                      uint16_t* __restrict__ dw) {
  __shared__ float s[8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  griddep_wait();
  float t = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int p = ry; p < nparts; p += 8) t += part[static_cast<int64_t>(p) * d + c];
  }
  s[ry][cx] = t;
  __syncthreads();
  if (ry == 0 && c < d) {
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += s[q][cx];
    dw[c] = f32_to_bf16_rne(v);
  }
}

namespace {

int norm_wpr(int d) { return d <= 1024 ? 1 : d <= 4096 ? 4 : 16; }

int norm_grid(int64_t rows, int wpr, int per_sm) {
  const int groups = kNormThreads / (32 * wpr);
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  return static_cast<int>(need < most ? need : most);
}

}  // namespace

// Rows of partial dw sums that launch_add_norm_backward writes (d floats each).
int add_norm_backward_parts(int64_t rows, int d) { return norm_grid(rows, norm_wpr(d), 2); }

int launch_add_norm(const AddNormArgs& a, cudaStream_t stream) {
  if (a.rows <= 0) return SPX_OK;
  const int wpr = norm_wpr(a.d);
  const int grid = norm_grid(a.rows, wpr, 4);
  const int nc = (a.d / 8 + 32 * wpr - 1) / (32 * wpr);
  auto run = [&](auto kernel) {
    kernel<<<grid, kNormThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  if (wpr == 1) return nc == 1 ? run(add_norm_kernel<1, 1>) : nc <= 3 ? run(add_norm_kernel<1, 3>) : run(add_norm_kernel<1, 4>);
  if (wpr == 4) return nc <= 2 ? run(add_norm_kernel<4, 2>) : run(add_norm_kernel<4, 4>);
  return nc <= 2 ? run(add_norm_kernel<16, 2>) : run(add_norm_kernel<16, 4>);
}

int launch_add_norm_backward(const AddNormBackwardArgs& a, uint16_t* dw, cudaStream_t stream) {
  if (a.rows <= 0) {
    if (dw == nullptr) return SPX_OK;
    return cudaMemsetAsync(dw, 0, static_cast<size_t>(a.d) * 2, stream) == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  }
  const int wpr = norm_wpr(a.d);
  const int grid = add_norm_backward_parts(a.rows, a.d);
  const int nc = (a.d / 8 + 32 * wpr - 1) / (32 * wpr);
  auto run = [&](auto kernel) {
    kernel<<<grid, kNormThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  int rc;
  if (wpr == 1)
    rc = nc == 1 ? run(add_norm_backward_kernel<1, 1>) : nc <= 3 ? run(add_norm_backward_kernel<1, 3>) : run(add_norm_backward_kernel<1, 4>);
  else if (wpr == 4)
    rc = nc <= 2 ? run(add_norm_backward_kernel<4, 2>) : run(add_norm_backward_kernel<4, 4>);
  else
    rc = nc <= 2 ? run(add_norm_backward_kernel<16, 2>) : run(add_norm_backward_kernel<16, 4>);
  if (rc != SPX_OK || dw == nullptr) return rc;
  return launch_pdl(norm_dw_kernel, dim3((a.d + 31) / 32), dim3(256), 0, stream, a.dw_part, grid, a.d, dw);
}

}  // namespace spx
