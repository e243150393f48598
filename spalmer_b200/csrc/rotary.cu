// Rotary positions of queries and keys: pair p of a head at position t turns
// by the angle t * freq[p],
//
//   (a, b) -> factor * (a cos - b sin, b cos + a sin)
//
// over the first 2 * pairs elements of each head (pairs are (p, p + pairs) or,
// interleaved, (2p, 2p + 1)); the others are copied.  The gradient is the same
// rotation with the sine negated.
//
// Bound by HBM: each element is read and written once.  A CTA takes a few
// tokens, computes their sines and cosines once for all heads into shared
// memory, then streams the heads through 16-byte loads and stores.  The angle
// needs more than FP32's 24 bits (a position of 10^6 leaves FP32 an error of
// 0.06), so it is taken in turns in FP64 -- three operations per (token, pair)
// -- and only the fraction of a turn goes on in FP32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "sm100.cuh"

namespace spx {

namespace {

constexpr int kRotMaxThreads = 512;
constexpr int kRotAngles = 2048;  // (token, pair) angles a CTA holds: 16 KB
constexpr int kRotUnroll = 4;

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

__device__ __forceinline__ float lo_f(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_f(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

}  // namespace

// One unit of work: VEC = 8: a 16-byte chunk (interleaved, or copied), or the
// two chunks of eight half-layout pairs; VEC = 1: one pair, or one copied
// element.  A thread keeps its unit (head and place in it) and walks tokens.
template <int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotMaxThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 s_cs[];  // [tokens per CTA][pairs]: cos, sin
  const int pairs = a.pairs;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_cta;
  const int nt = static_cast<int>(a.tokens - t0 < a.tokens_per_cta ? a.tokens - t0 : a.tokens_per_cta);
  // units of a head: the rotated ones first, then the copied ones
  const int rot_units = VEC == 8 ? (INTERLEAVED ? pairs / 4 : pairs / 8) : pairs;
  const int units = rot_units + (a.d - 2 * pairs) / VEC;
  const int total = (a.heads_q + a.heads_k) * units;  // of a token
  const int side = total <= static_cast<int>(blockDim.x) ? static_cast<int>(blockDim.x) / total : 1;  // tokens side by side
  int i = threadIdx.x, t_first = 0;
  if (side > 1) {
    t_first = i / total;
    i -= t_first * total;
    if (t_first >= side) i = total;  // no unit is left for this thread
  }
  const uint16_t* src = nullptr;
  uint16_t* dst = nullptr;
  const float2* cs0 = nullptr;
  int64_t sst = 0, dst_st = 0;
  bool turned = false;
  auto choose = [&]() {  // unit i
    const int h = i / units, unit = i - h * units;
    const bool is_q = h < a.heads_q;
    const int hh = is_q ? h : h - a.heads_q;
    turned = unit < rot_units;
    // first element of the unit
    const int e = turned ? (VEC == 8 ? unit * 8 : (INTERLEAVED ? 2 * unit : unit)) : 2 * pairs + (unit - rot_units) * VEC;
    sst = is_q ? a.q_st : a.k_st;
    dst_st = static_cast<int64_t>(is_q ? a.heads_q : a.heads_k) * a.d;
    src = (is_q ? a.q + hh * a.q_sh : a.k + hh * a.k_sh) + t0 * sst + e;
    dst = (is_q ? a.q_out : a.k_out) + t0 * dst_st + static_cast<int64_t>(hh) * a.d + e;
    cs0 = s_cs + (VEC == 8 ? (INTERLEAVED ? unit * 4 : unit * 8) : unit);
  };
  uint4 u[kRotUnroll], w[kRotUnroll];
  auto load = [&](int tb) {
#pragma unroll
    for (int r = 0; r < kRotUnroll; ++r) {
      const int t = tb + r * side;
      if (t >= nt) break;
      if constexpr (VEC == 8) {
        u[r] = __ldg(reinterpret_cast<const uint4*>(src + t * sst));
        if (!INTERLEAVED && turned) w[r] = __ldg(reinterpret_cast<const uint4*>(src + t * sst + pairs));
      } else {
        u[r].x = src[t * sst];
        if (turned) w[r].x = src[t * sst + (INTERLEAVED ? 1 : pairs)];
      }
    }
  };
  if (i < total) {  // the first loads travel while the angles are computed
    choose();
    load(t_first);
  }
  for (int n = threadIdx.x; n < nt * pairs; n += blockDim.x) {
    const int t = n / pairs, p = n - t * pairs;
    const int64_t at = (t0 + t) % a.pos_period;
    const int64_t pos = a.pos64 != 0 ? reinterpret_cast<const int64_t*>(a.pos)[at]
                                     : static_cast<int64_t>(reinterpret_cast<const int32_t*>(a.pos)[at]);
    const double turns = static_cast<double>(pos) * (a.freq[p] * 0.15915494309189533577);  // 1 / (2 pi)
    const float frac = static_cast<float>(turns - rint(turns));  // [-1/2, 1/2]
    // inside [-pi, pi] the fast functions are off by 2^-21 at most: nothing beside the result's BF16 rounding
    float sn, cs;
    __sincosf(6.28318530717958647692f * frac, &sn, &cs);
    s_cs[n] = make_float2(cs * a.factor, (a.inverse != 0 ? -sn : sn) * a.factor);
  }
  __syncthreads();
  for (; i < total; i += blockDim.x) {
    if (i != static_cast<int>(threadIdx.x) && side == 1) {
      choose();
      load(0);
    }
    for (int tb = t_first; tb < nt; tb += side * kRotUnroll) {
      if (tb != t_first) load(tb);
#pragma unroll
      for (int r = 0; r < kRotUnroll; ++r) {
        const int t = tb + r * side;
        if (t >= nt) break;
        uint16_t* out = dst + t * dst_st;
        const float2* cs = cs0 + t * pairs;
        if constexpr (VEC == 8) {
          if (turned && INTERLEAVED) {
            uint32_t x[4] = {u[r].x, u[r].y, u[r].z, u[r].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 c = cs[j];
              const float p = lo_f(x[j]), q = hi_f(x[j]);
              x[j] = pack2(p * c.x - q * c.y, q * c.x + p * c.y);
            }
            u[r] = make_uint4(x[0], x[1], x[2], x[3]);
          } else if (turned) {
            uint32_t x[4] = {u[r].x, u[r].y, u[r].z, u[r].w}, y[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 c = *reinterpret_cast<const float4*>(cs + 2 * j);  // pairs % 8 == 0: 16-byte aligned
              const float p0 = lo_f(x[j]), p1 = hi_f(x[j]), q0 = lo_f(y[j]), q1 = hi_f(y[j]);
              x[j] = pack2(p0 * c.x - q0 * c.y, p1 * c.z - q1 * c.w);
              y[j] = pack2(q0 * c.x + p0 * c.y, q1 * c.z + p1 * c.w);
            }
            u[r] = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(out + pairs) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          *reinterpret_cast<uint4*>(out) = u[r];
        } else if (turned) {
          const float2 c = cs[0];
          const float p = lo_f(u[r].x), q = lo_f(w[r].x);
          out[0] = f32_to_bf16_rne(p * c.x - q * c.y);
          out[INTERLEAVED ? 1 : pairs] = f32_to_bf16_rne(q * c.x + p * c.y);
        } else {
          out[0] = static_cast<uint16_t>(u[r].x);
        }
      }
    }
    if (side > 1) break;
  }
}

int launch_rotary(RotaryArgs a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.heads_q + a.heads_k <= 0) return SPX_OK;
  // 16-byte units need every head and every half to start on 16 bytes (8,192 tokens of 12 + 12 heads of 64: 14.5 us,
  // interleaved 12.7; one pair at a time 25.8 and 23.1)
  const auto aligned = [](const void* p, int64_t st, int64_t sh) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st % 8 == 0 && sh % 8 == 0;
  };
  const bool vec = a.d % 8 == 0 && (a.interleaved != 0 ? (2 * a.pairs) % 8 == 0 : a.pairs % 8 == 0) &&
                   (a.heads_q == 0 || (aligned(a.q, a.q_st, a.q_sh) && aligned(a.q_out, 0, 0))) &&
                   (a.heads_k == 0 || (aligned(a.k, a.k_st, a.k_sh) && aligned(a.k_out, 0, 0)));
  // threads: as many whole tokens' units as fit into about 384
  const int64_t units = vec ? (a.interleaved != 0 ? a.pairs / 4 : a.pairs / 8) + (a.d - 2 * a.pairs) / 8 : a.d - a.pairs;
  const int64_t total = units * (a.heads_q + a.heads_k);
  int threads = 256;
  if (total <= kRotMaxThreads) {
    const int64_t side = total <= 384 ? 384 / total : 1;
    threads = static_cast<int>((side * total + 31) / 32 * 32);
  }
  // tokens a CTA: one batch of loads a thread, at most kRotAngles angles
  int64_t tpc = (total <= threads ? threads / total : 1) * kRotUnroll;
  const int64_t cap = a.pairs > 0 ? kRotAngles / a.pairs : 64;
  tpc = tpc > cap ? cap : tpc;
  // a small batch is spread over the SMs (256 tokens: 4.1 us, in whole CTAs' loads 5.6)
  const int64_t spread = (a.tokens + device_sm_count() - 1) / device_sm_count();
  tpc = tpc > spread ? spread : tpc;
  tpc = tpc < 1 ? 1 : tpc;
  a.tokens_per_cta = static_cast<int>(tpc);
  const int64_t grid = (a.tokens + tpc - 1) / tpc;
  if (grid > 0x7FFFFFFF) return SPX_ERR_UNSUPPORTED;
  const size_t smem = static_cast<size_t>(tpc) * a.pairs * sizeof(float2);
  auto run = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(grid), threads, smem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  if (vec) return a.interleaved != 0 ? run(rotary_kernel<8, true>) : run(rotary_kernel<8, false>);
  return a.interleaved != 0 ? run(rotary_kernel<1, true>) : run(rotary_kernel<1, false>);
}

}  // namespace spx
