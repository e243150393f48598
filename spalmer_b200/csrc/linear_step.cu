// Linear attention, recurrent form for single tokens: for each request and head
//
//   S <- exp(g) S + k v^T          o = scale * S^T q
//
// with the FP32 state S [dk][dv] updated in place in a cache of states.
//
// Bound by HBM: the state is read once and written once (8 dk dv bytes a
// head); everything else is small.  A CTA holds the columns [c0, c0 + cols) of
// one state in registers, 16 bytes a load, neighbouring threads on
// neighbouring columns of a row; the sum over rows ends in shared memory.
// 256 requests of 12 heads of 128 x 128 (400 MB) take 64 us, 6.3 TB/s.
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "sm100.cuh"

namespace spx {

namespace {

constexpr int kStepThreads = 128;  // at least kLaMaxD
constexpr int kStepLoads = 8;      // 16-byte loads of a thread at most
static_assert(kStepThreads >= kLaMaxD, "a thread per element of a head");

__device__ __forceinline__ float decay_at(const void* g, bool f32, int64_t at) {
  return f32 ? reinterpret_cast<const float*>(g)[at] : bf16_to_f32(reinterpret_cast<const uint16_t*>(g)[at]);
}

}  // namespace

// NL: 16-byte loads of the state per thread.
template <int NL>
__global__ void __launch_bounds__(kStepThreads) la_step_kernel(const LaStepArgs a, int cols) {
  __shared__ float s_q[kLaMaxD], s_k[kLaMaxD], s_v[kLaMaxD];
  __shared__ float4 s_o[kStepThreads];
  const int h = blockIdx.y;
  const int64_t b = blockIdx.x;
  const int c0 = blockIdx.z * cols;
  const int nc = min(cols, a.dv - c0);      // columns of this CTA, a multiple of 4
  const int c4 = nc / 4;
  const int rows = kStepThreads / c4;       // state rows side by side
  const int tid = threadIdx.x;
  const int64_t slot = a.slot != nullptr ? a.slot[b] : b;
  uint16_t* out = a.out + (b * a.H + h) * a.dv + c0;
  if (slot < 0 || slot >= a.slots) {  // an empty row of the batch
    for (int i = tid; i < nc; i += kStepThreads) out[i] = 0;
    return;
  }
  const int col = tid % c4, r0 = tid / c4;
  float* S = a.state + (slot * a.H + h) * static_cast<int64_t>(a.dk) * a.dv + c0 + 4 * col;
  float4 s[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = r0 + i * rows;
    if (r0 < rows && r < a.dk) s[i] = *reinterpret_cast<const float4*>(S + static_cast<int64_t>(r) * a.dv);
  }
  const uint16_t* q = a.q.p + b * a.q.sb + (h / a.q.group) * a.q.sh;
  const uint16_t* k = a.k.p + b * a.k.sb + (h / a.k.group) * a.k.sh;
  const uint16_t* v = a.v.p + b * a.v.sb + (h / a.v.group) * a.v.sh + c0;
  if (tid < a.dk) {
    s_q[tid] = bf16_to_f32(q[tid]);
    s_k[tid] = bf16_to_f32(k[tid]);
  }
  if (tid < nc) s_v[tid] = bf16_to_f32(v[tid]);
  const float dec = expf(decay_at(a.g, a.g_f32 != 0, b * a.g_sb + h * a.g_sh));
  __syncthreads();
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (r0 < rows) {
    const float4 vv = make_float4(s_v[4 * col], s_v[4 * col + 1], s_v[4 * col + 2], s_v[4 * col + 3]);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = r0 + i * rows;
      if (r < a.dk) {
        const float kk = s_k[r], qq = s_q[r];
        s[i].x = fmaf(dec, s[i].x, kk * vv.x);
        s[i].y = fmaf(dec, s[i].y, kk * vv.y);
        s[i].z = fmaf(dec, s[i].z, kk * vv.z);
        s[i].w = fmaf(dec, s[i].w, kk * vv.w);
        *reinterpret_cast<float4*>(S + static_cast<int64_t>(r) * a.dv) = s[i];
        o.x = fmaf(qq, s[i].x, o.x);
        o.y = fmaf(qq, s[i].y, o.y);
        o.z = fmaf(qq, s[i].z, o.z);
        o.w = fmaf(qq, s[i].w, o.w);
      }
    }
    s_o[tid] = o;
  }
  __syncthreads();
  if (tid < nc) {
    const float* f = reinterpret_cast<const float*>(s_o);
    float t = 0.0f;
    for (int r = 0; r < rows; ++r) t += f[(r * c4) * 4 + tid];
    out[tid] = f32_to_bf16_rne(t * a.scale);
  }
}

int launch_la_step(const LaStepArgs& a, cudaStream_t stream) {
  if (a.batch <= 0) return SPX_OK;
  if (a.batch > 0x7FFFFFFF || a.H > 65535) return SPX_ERR_UNSUPPORTED;
  // Columns per CTA: all of them, or fewer while a thread would need more than eight loads or the CTAs would
  // leave SMs idle.  256 requests of 12 heads of 128 x 128: 64 us with 8 loads a thread, 78 with 16 and 70 with 4; two
  // requests of 32 heads: 4.7 us split, 5.1 not.
  int cols = a.dv;
  const int64_t heads = a.batch * a.H;
  auto loads = [&](int c) {
    const int rows = kStepThreads / (c / 4);
    return (a.dk + rows - 1) / rows;
  };
  while (cols > 16 && (loads(cols) > kStepLoads || heads * ((a.dv + cols - 1) / cols) < device_sm_count()))
    cols = ((cols + 1) / 2 + 3) / 4 * 4;
  const int need = loads(cols);
  const dim3 grid(static_cast<unsigned>(a.batch), a.H, (a.dv + cols - 1) / cols);
  auto run = [&](auto kernel) {
    kernel<<<grid, kStepThreads, 0, stream>>>(a, cols);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  // the last slice may be narrower: it then has more rows side by side and needs fewer loads
  return need <= 2 ? run(la_step_kernel<2>) : need <= 4 ? run(la_step_kernel<4>) : run(la_step_kernel<kStepLoads>);
}

}  // namespace spx
