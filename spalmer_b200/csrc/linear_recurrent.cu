// Linear attention with a decay per head, token by token (a job of LaArgs):
//
//   forward   S <- exp(g_t) S + b_t c_t^T,  out_t = scale S^T a_t
//   reverse   S <- S + b_t c_t^T, out_t = scale S^T a_t, S <- exp(g_t) S
//
// One CTA per (job, sequence, head); thread j keeps column j of the FP32
// state in registers.  Bound by the chain of tokens, not by memory.
//
// Also the two small passes after a backward: the decay's gradient from the
// jobs' dots, and the sum of a shared head's gradients over its query heads.
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "sm100.cuh"

namespace spx {

namespace {

constexpr int kRecThreads = 128;

// Tokens [start, start + len) of sequence s in the flattened [total] order; false if cu is not sound.
__device__ __forceinline__ bool sequence_of(const int32_t* cu, int64_t T, int64_t total, int s, int64_t* start,
                                            int64_t* len) {
  if (cu == nullptr) {
    *start = s * T;
    *len = T;
    return true;
  }
  const int64_t lo = cu[s], hi = cu[s + 1];
  *start = lo;
  *len = hi - lo;
  return lo >= 0 && hi >= lo && hi <= total;
}

}  // namespace

template <int DA>
__global__ void __launch_bounds__(kRecThreads) la_recurrent_kernel(const __grid_constant__ LaArgs args) {
  __shared__ float s_a[2][DA], s_b[2][DA];
  __shared__ float s_dot[2][kRecThreads / 32];
  const LaJob& j = args.job[blockIdx.y];
  const int h = blockIdx.x % args.H;
  const int seq = blockIdx.x / args.H;
  const int tid = threadIdx.x;
  int64_t start, len;
  if (!sequence_of(args.cu, args.T, args.total, seq, &start, &len)) {
    if (tid == 0) record_error(args.status, SPX_DEV_BAD_TILE);
    return;
  }
  const int64_t batch = args.cu == nullptr ? seq : 0, t_in = args.cu == nullptr ? 0 : start;
  const uint16_t* pa = j.a.p + batch * j.a.sb + t_in * j.a.st + (h / j.a.group) * j.a.sh;
  const uint16_t* pb = j.b.p + batch * j.b.sb + t_in * j.b.st + (h / j.b.group) * j.b.sh;
  const uint16_t* pc = j.c.p + batch * j.c.sb + t_in * j.c.st + (h / j.c.group) * j.c.sh;
  const uint16_t* pe = j.e.p == nullptr ? nullptr : j.e.p + batch * j.e.sb + t_in * j.e.st + (h / j.e.group) * j.e.sh;
  const int64_t g0 = batch * args.g_sb + t_in * args.g_st + h * args.g_sh;
  const bool col = tid < j.dc;
  const int64_t state0 = (static_cast<int64_t>(seq) * args.H + h) * j.da * j.dc;
  float S[DA];
#pragma unroll
  for (int r = 0; r < DA; ++r)
    S[r] = j.init != nullptr && col && r < j.da ? j.init_scale * j.init[state0 + r * j.s_row + tid * j.s_col] : 0.0f;
  for (int64_t i = 0; i < len; ++i) {
    const int64_t t = j.reverse != 0 ? len - 1 - i : i;
    const int buf = static_cast<int>(i & 1);
    if (tid < DA) {
      s_a[buf][tid] = tid < j.da ? bf16_to_f32(pa[t * j.a.st + tid]) : 0.0f;
      s_b[buf][tid] = tid < j.da ? bf16_to_f32(pb[t * j.b.st + tid]) : 0.0f;
    }
    const float c = col ? bf16_to_f32(pc[t * j.c.st + tid]) : 0.0f;
    const int64_t ga = g0 + t * args.g_st;
    const float dec = expf(args.g_f32 != 0 ? reinterpret_cast<const float*>(args.g)[ga]
                                           : bf16_to_f32(reinterpret_cast<const uint16_t*>(args.g)[ga]));
    const float before = j.reverse != 0 ? 1.0f : dec, after = j.reverse != 0 ? dec : 1.0f;
    __syncthreads();
    float o = 0.0f;
#pragma unroll
    for (int r = 0; r < DA; ++r) {
      const float s = fmaf(before, S[r], s_b[buf][r] * c);
      o = fmaf(s_a[buf][r], s, o);
      S[r] = s * after;
    }
    o *= args.scale;
    const int64_t at = ((start + t) * args.H + h) * j.dc + tid;
    if (col) {
      if (j.out_f32 != 0)
        reinterpret_cast<float*>(j.out)[at] = o;
      else
        reinterpret_cast<uint16_t*>(j.out)[at] = f32_to_bf16_rne(o);
    }
    if (pe != nullptr) {
      float d = col ? o * bf16_to_f32(pe[t * j.e.st + tid]) : 0.0f;
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, off);
      if ((tid & 31) == 0) s_dot[buf][tid >> 5] = d;
      __syncthreads();
      if (tid == 0) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRecThreads / 32; ++w) sum += s_dot[buf][w];
        j.dots[h * args.total + start + t] = sum;
      }
    }
  }
  if (j.fin != nullptr && col) {
#pragma unroll
    for (int r = 0; r < DA; ++r)
      if (r < j.da) j.fin[state0 + r * j.s_row + tid * j.s_col] = j.fin_scale * S[r];
  }
}

int launch_la_recurrent(const LaArgs& a, cudaStream_t stream) {
  if (a.nseq <= 0 || a.H <= 0) return SPX_OK;
  int da = 0;
  for (int i = 0; i < a.njobs; ++i) da = a.job[i].da > da ? a.job[i].da : da;
  const int64_t items = static_cast<int64_t>(a.nseq) * a.H;
  if (items > 0x7FFFFFFF) return SPX_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(items), a.njobs);
  auto run = [&](auto kernel) {
    kernel<<<grid, kRecThreads, 0, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  return da <= 32 ? run(la_recurrent_kernel<32>) : da <= 64 ? run(la_recurrent_kernel<64>) : run(la_recurrent_kernel<128>);
}

// ---------------------------------------------------------------- decay gradient
// One CTA per (sequence, head): a suffix sum over its tokens.  Thread i takes
// a run of consecutive tokens; the sums are FP64, because terms of both signs
// cancel over the whole sequence.
namespace {
constexpr int kDgThreads = 1024;
constexpr int kDgEach = 4;  // tokens a thread
}

__global__ void __launch_bounds__(kDgThreads) la_decay_grad_kernel(const LaDecayGradArgs a) {
  __shared__ double s_part[32];
  const int h = blockIdx.x % a.H, seq = blockIdx.x / a.H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t start, len;
  if (!sequence_of(a.cu, a.T, a.total, seq, &start, &len)) return;  // the jobs recorded it
  auto block_sum = [&](double v) {  // every thread gets the CTA's sum
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    __syncthreads();
    if (lane == 0) s_part[warp] = v;
    __syncthreads();
    double t = s_part[lane];
    for (int off = 16; off >= 1; off >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, off);
    return t;
  };
  double carry = 0.0;
  if (a.last != nullptr) {
    const float* x = a.last + (static_cast<int64_t>(seq) * a.H + h) * a.state_elems;
    const float* y = a.d_last + (static_cast<int64_t>(seq) * a.H + h) * a.state_elems;
    double s = 0.0;
    for (int64_t i = tid; i < a.state_elems; i += kDgThreads) s += static_cast<double>(x[i]) * y[i];
    carry = block_sum(s);
  }
  const int64_t base = h * a.total + start;
  const int64_t plane = static_cast<int64_t>(a.H) * a.total;
  // Tiles of kDgThreads x kDgEach tokens from the end.  A thread sums its own
  // tokens, and one scan over the CTA's threads joins them: with one token a
  // thread 16 sequences of 4,096 tokens, 12 heads, took 25.7 us, now 16.9.
  for (int64_t hi = len; hi > 0; hi -= kDgThreads * kDgEach) {
    const int64_t t0 = hi - 1 - static_cast<int64_t>(tid) * kDgEach;  // thread 0 takes the last tokens
    double v[kDgEach];
#pragma unroll
    for (int e = 0; e < kDgEach; ++e) v[e] = 0.0;
    auto add = [&](const float* dots, int slices, float sign) {
      for (int s = 0; s < slices; ++s) {
        float x[kDgEach];
#pragma unroll
        for (int e = 0; e < kDgEach; ++e) x[e] = t0 - e >= 0 ? dots[s * plane + base + t0 - e] : 0.0f;
#pragma unroll
        for (int e = 0; e < kDgEach; ++e) v[e] += static_cast<double>(sign * x[e]);
      }
    };
    add(a.q_dots, a.q_slices, 1.0f);
    add(a.k_dots, a.k_slices, -1.0f);
#pragma unroll
    for (int e = 1; e < kDgEach; ++e) v[e] += v[e - 1];
    double up = v[kDgEach - 1];  // of the warp's threads up to this one
    for (int off = 1; off < 32; off <<= 1) {
      const double u = __shfl_up_sync(0xFFFFFFFFu, up, off);
      if (lane >= off) up += u;
    }
    __syncthreads();
    if (lane == 31) s_part[warp] = up;
    __syncthreads();
    double warps = s_part[lane];  // of the warps up to the lane's
    for (int off = 1; off < 32; off <<= 1) {
      const double u = __shfl_up_sync(0xFFFFFFFFu, warps, off);
      if (lane >= off) warps += u;
    }
    const double all = __shfl_sync(0xFFFFFFFFu, warps, 31);
    const double earlier = __shfl_sync(0xFFFFFFFFu, warps, warp > 0 ? warp - 1 : 0);
    const double mine = __shfl_up_sync(0xFFFFFFFFu, up, 1);
    const double before = carry + (warp > 0 ? earlier : 0.0) + (lane > 0 ? mine : 0.0);
#pragma unroll
    for (int e = 0; e < kDgEach; ++e) {
      if (t0 - e < 0) continue;
      // nothing decays into a first token that no state comes before: zero, not what rounding leaves of it
      const float r = t0 - e == 0 && a.from_zero != 0 ? 0.0f : static_cast<float>(before + v[e]);
      const int64_t at = (start + t0 - e) * a.H + h;
      if (a.g_f32 != 0)
        reinterpret_cast<float*>(a.dg)[at] = r;
      else
        reinterpret_cast<uint16_t*>(a.dg)[at] = f32_to_bf16_rne(r);
    }
    carry += all;
  }
}

int launch_la_decay_grad(const LaDecayGradArgs& a, cudaStream_t stream) {
  const int64_t items = static_cast<int64_t>(a.nseq) * a.H;
  if (items <= 0) return SPX_OK;
  if (items > 0x7FFFFFFF) return SPX_ERR_UNSUPPORTED;
  la_decay_grad_kernel<<<static_cast<unsigned>(items), kDgThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
}

// ---------------------------------------------------------------- shared heads
// One warp per (token, shared head): the sum over its query heads' gradients,
// and with `e` (the shared tensor itself) each query head's dot with it.
__global__ void __launch_bounds__(256) la_group_sum_kernel(const LaGroupSumArgs a) {
  const int lane = threadIdx.x & 31;
  const int kv = a.H / a.group;
  const int64_t n = a.total * kv;
  const bool col = 4 * lane < a.d;
  for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < n; i += gridDim.x * 8ll) {
    const int64_t t = i / kv;
    const int h = static_cast<int>(i - t * kv);
    float4 ev = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.e.p != nullptr && col) {
      const int64_t b = t / a.T;
      const uint2 u = *reinterpret_cast<const uint2*>(a.e.p + b * a.e.sb + (t - b * a.T) * a.e.st + h * a.e.sh + 4 * lane);
      ev = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
    }
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int q = 0; q < a.group; ++q) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (col) v = *reinterpret_cast<const float4*>(a.in + (i * a.group + q) * a.d + 4 * lane);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      if (a.e.p != nullptr) {
        float d = fmaf(v.x, ev.x, fmaf(v.y, ev.y, fmaf(v.z, ev.z, v.w * ev.w)));
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, off);
        if (lane == 0) a.dots[static_cast<int64_t>(h * a.group + q) * a.total + t] = d;
      }
    }
    if (col) {
      const uint2 b = make_uint2(f32_to_bf16_rne(s.x) | (static_cast<uint32_t>(f32_to_bf16_rne(s.y)) << 16),
                                 f32_to_bf16_rne(s.z) | (static_cast<uint32_t>(f32_to_bf16_rne(s.w)) << 16));
      *reinterpret_cast<uint2*>(a.out + i * a.d + 4 * lane) = b;
    }
  }
}

int launch_la_group_sum(const LaGroupSumArgs& a, cudaStream_t stream) {
  const int64_t n = a.total * (a.H / a.group);
  if (n <= 0) return SPX_OK;
  int64_t blocks = (n + 7) / 8;
  if (blocks > 148 * 16) blocks = 148 * 16;
  la_group_sum_kernel<<<static_cast<int>(blocks), 256, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
}

}  // namespace spx
