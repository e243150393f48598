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
// The pass is bound by HBM: each tensor is read or written once (65,536 rows of
// 768, BF16: forward 65 us, 6.2 TB/s; backward 75 us, 5.4 TB/s; 16,387 rows of 2,048
// to MXFP8 with an FP32 sum, 370 MB: 65 us, 5.7 TB/s).  A row is
// held in the registers of 32 * WPR threads (NC chunks of eight elements each),
// so the statistics cost no second read; a CTA walks rows with a stride, which
// keeps w in registers for all of them, and a row's loads are issued while the
// row before is worked on (loads between the stores of one row went one after
// another: 132 us and not 66 for 65,536 rows of 768, 403 MB).  MXFP8: four
// neighbouring lanes hold a block of 32, so its largest magnitude is two shuffles.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// Eight elements as they are stored: BF16 in one register quad, FP32 in two.
template <bool F32>
struct Raw8 {
  uint4 u[F32 ? 2 : 1];
};

template <bool F32>
__device__ __forceinline__ void load_raw(const void* base, int64_t at, Raw8<F32>& r) {
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at * (F32 ? 4 : 2));
#pragma unroll
  for (int i = 0; i < (F32 ? 2 : 1); ++i) r.u[i] = __ldg(p + i);
}

template <bool F32>
__device__ __forceinline__ void unpack8(const Raw8<F32>& r, float (&v)[8]) {
  if constexpr (F32) {
    const uint32_t w[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
  } else {
    unpack8(r.u[0], v);
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

// Two floats -> two E4M3 bytes, to nearest even and at most 448; a NaN stays one (mx_e4m3x2's clamp would make it -448).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3));
}

// Sums over the 32 * WPR threads of a row.  `part` holds
// [2][rows per CTA][WPR][n]; the two halves alternate from row to row, so one
// barrier a row is enough.
template <int WPR, int N, typename T>
__device__ __forceinline__ void row_sum(T (&s)[N], T* part, int group, int wr, int lane, uint32_t turn) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] += __shfl_xor_sync(0xFFFFFFFFu, s[j], off);
  }
  if constexpr (WPR > 1) {
    constexpr int kGroups = kNormThreads / (32 * WPR);
    T* p = part + ((turn & 1u) * kGroups + group) * WPR * N;
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < N; ++j) p[wr * N + j] = s[j];
    }
    // the row's warps alone
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * WPR) : "memory");
#pragma unroll
    for (int j = 0; j < N; ++j) {
      T t = 0;
#pragma unroll
      for (int w = 0; w < WPR; ++w) t += p[w * N + j];
      s[j] = t;
    }
  }
}

}  // namespace

// RES: 0 no residual, 1 BF16, 2 FP32.  MX: MXFP8 rows out.  A value that is to become
// E4M3 lies near a rounding border or not, and each bit of FP32 that y loses moves
// twice as many across; so there 1 / sqrt and the two products keep their remainders
// (16,387 rows of 2,048: 65 us, without 62).
template <int WPR, int NC, int RES, bool MX>
__global__ void __launch_bounds__(kNormThreads, 2) add_norm_kernel(const AddNormArgs a) {
  constexpr int kGroups = kNormThreads / (32 * WPR);
  __shared__ float part[2 * kGroups * WPR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wr = warp % WPR;
  const int nchunks = a.d / 8;
  const float inv_d = 1.0f / static_cast<float>(a.d);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  uint4 wv[NC];
  Raw8<false> xr[NC];
  Raw8<RES == 2> rr[NC];
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (c < nchunks) {
        load_raw<false>(a.x, row * a.ld_x + c * 8, xr[i]);
        if constexpr (RES != 0) load_raw<RES == 2>(a.res, row * a.ld_res + c * 8, rr[i]);
      }
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  constexpr bool kAhead = NC <= 2;
  if (kAhead) fetch(row);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * WPR + wr) * 32 + lane;
    wv[i] = c < nchunks ? __ldg(reinterpret_cast<const uint4*>(a.w) + c) : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t turn = 0;
  // every warp of the CTA runs the same number of rows (row_sum has a barrier)
  for (int64_t row0 = row - group; row0 < a.rows; row0 += step, row += step, ++turn) {
    const bool live = row < a.rows;
    if (!kAhead) fetch(row);
    float h[NC][8];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (live && c < nchunks) {
        unpack8(xr[i], h[i]);
        if constexpr (RES != 0) {
          float r[8];
          unpack8(rr[i], r);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            h[i][j] += r[j];
            if (RES == 1) h[i][j] = round_bf16(h[i][j]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
      }
      float sq = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(h[i][j], h[i][j], sq);
      s[0] += sq;
    }
    if (kAhead) fetch(row + step);
    if constexpr (RES != 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (i * WPR + wr) * 32 + lane;
        if (live && c < nchunks) store8(a.sum, row * a.d + c * 8, RES == 2, h[i]);
      }
    }
    row_sum<WPR, 1>(s, part, group, wr, lane, turn);
    const float ms = s[0] * inv_d + a.eps, r = 1.0f / sqrtf(ms);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      const bool in = live && c < nchunks;
      float wf[8], y[8];
      unpack8(wv[i], wf);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = h[i][j] * r * wf[j];
      if (a.y != nullptr && in) store8(a.y, row * a.d + c * 8, false, y);
      if constexpr (MX) {
        // what r lacks: 1 / sqrt(ms) = r (1 + e / 2), e = 1 - ms r^2
        const float mr = ms * r;
        const float r_rest = r > 0.0f ? 0.5f * r * (fmaf(-mr, r, 1.0f) - fmaf(ms, r, -mr) * r) : 0.0f;  // r = 0: ms overflowed
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p = h[i][j] * r;
          y[j] += fmaf(fmaf(h[i][j], r_rest, fmaf(h[i][j], r, -p)), wf[j], fmaf(p, wf[j], -y[j]));
        }
        // blocks of 32 = four lanes; all lanes take part in the shuffles (d % 32 == 0, so a block is wholly in or out)
        float amax = 0.0f;  // of the numbers: fmaxf passes over a NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        const uint32_t sb = mx_scale_byte(amax);
        const float m = mx_multiplier(sb);
        if (in) {
          const uint32_t q0 = e4m3x2(y[0] * m, y[1] * m) | (e4m3x2(y[2] * m, y[3] * m) << 16);
          const uint32_t q1 = e4m3x2(y[4] * m, y[5] * m) | (e4m3x2(y[6] * m, y[7] * m) << 16);
          *reinterpret_cast<uint2*>(a.mx_values + row * a.d + c * 8) = make_uint2(q0, q1);
          if ((c & 3) == 0) a.mx_scales[row * (a.d / kMxBlock) + c / 4] = static_cast<uint8_t>(sb);
        }
      }
    }
  }
}

// dw is summed per thread over the CTA's rows, then over the CTA's row groups
// in shared memory, then over CTAs by norm_dw_kernel: a fixed order, no atomics.
template <int WPR, int NC, bool F32>
__global__ void __launch_bounds__(kNormThreads, 1) add_norm_backward_kernel(const AddNormBackwardArgs a) {
  constexpr int kGroups = kNormThreads / (32 * WPR);
  constexpr int kCols = 32 * WPR * 8;  // columns of one chunk index
  __shared__ float part[2 * kGroups * WPR * 2];
  __shared__ float s_dw[kGroups > 1 ? kCols * (kGroups > 8 ? 8 : kGroups) : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / WPR, wr = warp % WPR;
  const int nchunks = a.d / 8;
  const float inv_d = 1.0f / static_cast<float>(a.d);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  uint4 wv[NC], gr[NC];
  Raw8<F32> hr[NC], sr[NC];
  float dw[NC][8];
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (c < nchunks) {
        gr[i] = __ldg(reinterpret_cast<const uint4*>(a.dy + row * a.ld_dy) + c);
        load_raw<F32>(a.h, row * a.ld_h + c * 8, hr[i]);
        if (a.dsum != nullptr) load_raw<F32>(a.dsum, row * a.ld_dsum + c * 8, sr[i]);
      }
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  constexpr bool kAhead = NC <= 3;
  if (kAhead) fetch(row);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * WPR + wr) * 32 + lane;
    wv[i] = c < nchunks ? __ldg(reinterpret_cast<const uint4*>(a.w) + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
  }
  uint32_t turn = 0;
  for (int64_t row0 = row - group; row0 < a.rows; row0 += step, row += step, ++turn) {
    const bool live = row < a.rows;
    if (!kAhead) fetch(row);
    Raw8<F32> h[NC], ds[NC];
    uint4 g[NC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      h[i] = hr[i], g[i] = gr[i], ds[i] = sr[i];
      if (!live || c >= nchunks) continue;
      float wf[8], gf[8], hf[8];
      unpack8(wv[i], wf);
      unpack8(g[i], gf);
      unpack8(h[i], hf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[0] = fmaf(hf[j], hf[j], s[0]);
        s[1] = fmaf(gf[j] * wf[j], hf[j], s[1]);
      }
    }
    if (kAhead) fetch(row + step);
    row_sum<WPR, 2>(s, part, group, wr, lane, turn);
    const float r = 1.0f / sqrtf(s[0] * inv_d + a.eps);
    const float k = r * r * s[1] * inv_d;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * WPR + wr) * 32 + lane;
      if (!live || c >= nchunks) continue;
      float wf[8], gf[8], hf[8], dh[8];
      unpack8(wv[i], wf);
      unpack8(g[i], gf);
      unpack8(h[i], hf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] = fmaf(gf[j] * hf[j], r, dw[i][j]);
        dh[j] = r * (gf[j] * wf[j] - hf[j] * k);
      }
      if (a.dsum != nullptr) {
        float sf[8];
        unpack8(ds[i], sf);
#pragma unroll
        for (int j = 0; j < 8; ++j) dh[j] += sf[j];
      }
      store8(a.dx, row * a.d + c * 8, false, dh);
      if (F32 && a.dres != nullptr) store8(a.dres, row * a.d + c * 8, true, dh);
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

// Warps of a row: up to two chunks a thread (registers for this row and the
// next), from one warp to sixteen; beyond that more chunks, loaded row by row.
// (One chunk a thread and twice the warps: 51 and 64 us, not 44 and 49, forward and
// backward over 2^25 elements in rows of 768.)  Where half of the warps hold the row
// in three chunks, the backward of BF16 residuals takes those: 45 us, not 49,
// as two chunks of two warps leave a quarter of the lanes idle.
int norm_wpr(int d, bool three) {
  int wpr = 1;
  while (wpr < 16 && 32 * wpr * 2 < d / 8) wpr *= 2;
  return three && wpr > 1 && 32 * (wpr / 2) * 3 >= d / 8 ? wpr / 2 : wpr;
}

// kernel(wpr, nc) as compile-time constants
template <bool THREE, typename F>
int with_shape(int d, F&& f) {
  const int wpr = norm_wpr(d, THREE);
  const int nc = (d / 8 + 32 * wpr - 1) / (32 * wpr);
  using std::integral_constant;
  auto pick = [&](auto w) {
    if constexpr (THREE && decltype(w)::value < 16) {
      if (nc == 3) return f(w, integral_constant<int, 3>{});
    }
    return nc <= 1 ? f(w, integral_constant<int, 1>{}) : f(w, integral_constant<int, 2>{});
  };
  switch (wpr) {
    case 1: return pick(integral_constant<int, 1>{});
    case 2: return pick(integral_constant<int, 2>{});
    case 4: return pick(integral_constant<int, 4>{});
    case 8: return pick(integral_constant<int, 8>{});
    default: return nc <= 2 ? pick(integral_constant<int, 16>{}) : f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  }
}

int norm_grid(int64_t rows, int wpr, int per_sm) {
  const int groups = kNormThreads / (32 * wpr);
  const int64_t need = (rows + groups - 1) / groups;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  return static_cast<int>(need < most ? need : most);
}

}  // namespace

// Rows of partial dw sums that launch_add_norm_backward writes at most (d floats each).
int add_norm_backward_parts(int64_t rows, int d) { return norm_grid(rows, norm_wpr(d, false), 1); }

int launch_add_norm(const AddNormArgs& a, cudaStream_t stream) {
  if (a.rows <= 0) return SPX_OK;
  const int grid = norm_grid(a.rows, norm_wpr(a.d, false), 2);
  return with_shape<false>(a.d, [&](auto w, auto n) {
    constexpr int W = decltype(w)::value, N = decltype(n)::value;
    auto run = [&](auto mx) {
      constexpr bool MX = decltype(mx)::value;
      if (a.res == nullptr)
        add_norm_kernel<W, N, 0, MX><<<grid, kNormThreads, 0, stream>>>(a);
      else if (a.res_f32 == 0)
        add_norm_kernel<W, N, 1, MX><<<grid, kNormThreads, 0, stream>>>(a);
      else
        add_norm_kernel<W, N, 2, MX><<<grid, kNormThreads, 0, stream>>>(a);
    };
    if (a.mx_values != nullptr)
      run(std::true_type{});
    else
      run(std::false_type{});
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  });
}

int launch_add_norm_backward(const AddNormBackwardArgs& a, uint16_t* dw, cudaStream_t stream) {
  if (a.rows <= 0) {
    if (dw == nullptr) return SPX_OK;
    return cudaMemsetAsync(dw, 0, static_cast<size_t>(a.d) * 2, stream) == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  }
  const int grid = norm_grid(a.rows, norm_wpr(a.d, a.res_f32 == 0), 1);
  const int rc = a.res_f32 == 0 ? with_shape<true>(a.d, [&](auto w, auto n) {
    add_norm_backward_kernel<decltype(w)::value, decltype(n)::value, false><<<grid, kNormThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  }) : with_shape<false>(a.d, [&](auto w, auto n) {
    add_norm_backward_kernel<decltype(w)::value, decltype(n)::value, true><<<grid, kNormThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  });
  if (rc != SPX_OK || dw == nullptr) return rc;
  return launch_pdl(norm_dw_kernel, dim3((a.d + 31) / 32), dim3(256), 0, stream, a.dw_part, grid, a.d, dw);
}

}  // namespace spx
