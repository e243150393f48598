// Linear attention with a decay per head on tcgen05 tensor cores: the chunked
// form of a job of LaArgs (kernels.h).  For a chunk of 128 tokens with G_i =
// the sum of the log decays up to token i inside the chunk,
//
//   out = scale ( tril(e^{G_i - G_j} a_i . b_j) C + e^{G_i} a_i S )
//   S'  = e^{G_128} S + sum_j e^{G_128 - G_j} b_j c_j^T
//
// (reverse: triu, e^{G_j - G_i}, e^{G_128 - G_i} and e^{G_j}).  The forward
// pass and the three gradients are jobs of this one form, so a backward pass is
// one launch of three times the work and stores no states.
//
// A CTA walks its chunks in order for one (job, sequence, head, 64 columns of
// C), a "lane"; the FP32 state stays in registers from chunk to chunk.  64 columns
// leave room in shared memory to load the next chunk (two or three stages) and give
// twice as many CTAs at 128-wide heads; a . b is then computed once per 64 columns,
// which the tensor cores have time for (they are busy for a quarter of it).
//
// Operand precision.  a, b, c are exact BF16.  What is not is split into BF16
// parts that are multiplied one after another into the same FP32 accumulator:
//   c scaled by its decay (into the state): three parts where a caller keeps the
//     last state (exact), else two (2^-18; the first state's gradient too);
//   the decayed a . b matrix and the state (into out): one part in the forward
//     pass, whose output is rounded to BF16 as coarsely (2.3e-3 from 64 bits, one
//     rounding alone 1.7e-3; two parts: 158 us and not 133 for 65,536 tokens of 12
//     heads of 64, and no room for them beside three parts of c at 128 wide), two in
//     the gradients, because d decay is a long sum of q . dq - k . dk that cancels.
//
// Decay factors are exponentials of sums <= 0, never quotients, so no decay
// overflows: inside a 32-token block the sum between two tokens, across blocks a
// factor up to the block's edge and one from there.  A token's log2 decay is
// clamped to -150, which is zero in FP32; sums start at block edges, and those to and
// from an edge are taken directly, so that a token that forgets everything costs the
// other blocks and the state no digits, and a NaN reaches no token on its other side.
// Between two tokens of one block the sum is the difference of two such sums and off by
// about 2^-24 of them: factors by 3e-5 at most in a block that decays by 2^-150 in all,
// 4e-4 after 26 tokens that forget everything.
//
// How lanes meet SMs.  Too few lanes: the sequence is cut into segments; a pass
// over b and c alone gives each segment's state from zero, a small kernel chains
// them, and the full pass starts every segment from its own first state
// (segments_for).  A few more lanes than SMs: even shares of chunks (even_shares).
// Packed sequences: longest first from a queue (37 ragged prompts of 20,011 tokens
// in all, 12 heads of 64: 83 us, in the order given and a fixed stride 115; with
// the later steps 72).
//
// What bounds it: neither HBM nor the tensor cores, but instructions.  A chunk of
// 64-wide heads takes about 6,000 cycles, in the gradients too (1.75 GHz under this
// kernel), in which four schedulers issue 48 to 57% of the time and wait for
// instruction fetch in a quarter of the rest: a dozen roles run at once, so that their
// code has to stay small, and unrolling or prefetching more made every loop slower.
// 65,536 tokens of 12 heads of 64: forward 142 us (403 MB, 2.8 TB/s), the three
// gradients 431 us.  8,190 tokens of 16 heads of 128 over 4 shared ones: 88 and 213 us.
//
// Warps: 0-7 the decayed a . b matrix (TMEM -> registers -> TMEM operand), 8-15
// scaled c, 16-19 the state, 20-27 the epilogue, 28 and 31 TMA, 29 MMA, 30
// decays.  One warp gets through an instruction every three or four cycles here,
// so the longer roles have two warpgroups, and registers move between them.  (A
// second MMA warp, a . b and its product apart from the state's, cost more
// instructions than its shorter waits gave back: 173, not 154 us.)
// Every wait is bounded (status word, then return).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kernels.h"
#include "sm100.cuh"

namespace spx {

namespace {

constexpr int kC = 128;              // tokens of a chunk
constexpr int kTile = kC * 128;      // bytes of a [128 tokens][64] BF16 tile
constexpr int kLaThreads = 32 * 32;  // eight warpgroups
constexpr int64_t kWaitCycles = 4000000000;  // about two seconds
// Registers of the warpgroups' threads: the launch gives each 64 (1024 x 64 = 65,536).
constexpr int kRegsC = 48, kRegsRest = 40;
constexpr int kOrderMax = 4096;  // more sequences are taken as they come
constexpr uint32_t kBarBytes = 416;
constexpr uint32_t kTmP = 0, kTmOI = 256, kTmOX = 320, kTmKV = 384, kTmCols = 512;

struct alignas(64) LaChunkArgs {
  CUtensorMap map[3][3];
  LaArgs la;
  int lanes[4];          // first lane of each job; lanes[njobs] = all of them
  int slices[3];
  int nseg, state_only, run_segs;
  const int* order;      // packed: the sequences, longest first | null
  int* queue;            // with order: the next item to take
  float* seg_state;      // [lane][nseg][128][64]
  float* seg_decay;      // [lane][nseg]
  // Even shares (or null): every CTA takes as many chunks, and a lane that two of
  // them share is handed on by its state, [CTA][128][64], and a flag per warp of it.
  float* hand;
  int* handed;
};

// Decays of a chunk, each sum taken directly (a small one as the difference of
// large ones would lose its digits): log2 decays from the token's 32-token block's
// start up to it (reverse: from it to the block's end), the factor over the rest of
// the block, and the blocks' totals.
struct DecayTable {
  float a[kC];
  float cf[kC];
  float total[4];
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The other blocks of the chunk on the token's far side: those before its own (reverse: after it), or the others.
__device__ __forceinline__ float blocks(const DecayTable& t, int quad, bool before) {
  float x = 0.0f;
#pragma unroll
  for (int q = 0; q < 4; ++q) x += (before ? q < quad : q > quad) ? t.total[q] : 0.0f;
  return x;
}
// Between the state at the chunk's near end and the token (on a . S), and between the token and the far end (on c).
__device__ __forceinline__ float into_token(const DecayTable& t, int quad, int row, bool rev) {
  return ex2(t.a[row] + blocks(t, quad, !rev));
}
__device__ __forceinline__ float out_of_token(const DecayTable& t, int quad, int row, bool rev) {
  return t.cf[row] * ex2(blocks(t, quad, rev));
}

template <int DKB, bool PRECISE, int PARTS>
struct Cfg {
  static constexpr int kStages = DKB == 1 ? 3 : 2;
  static constexpr int kParts = PARTS;            // of scaled c
  static constexpr int kSParts = PRECISE ? 2 : 1; // of the state
  // 64 rows of state in the 128 lanes of an accumulator: computed twice, so that each of the four warps
  // keeps half of the columns of 32 rows and not two of them all (training backward 459 -> 412 us for 65,536
  // tokens, 12 heads; packed prompts 79 -> 72).
  static constexpr int kStateCols = DKB == 1 ? 32 : 64;
  static constexpr int kRegsState = DKB == 1 ? 88 : 120;
  static_assert(4 * 64 + 2 * kRegsC + kRegsState + kRegsRest <= 8 * 64, "registers of a CTA");
  static constexpr uint32_t kStage = (2 * DKB + 1) * kTile;
  static constexpr uint32_t kSTile = DKB * 64 * 128;
  static constexpr uint32_t kOffS = kStages * kStage;
  static constexpr uint32_t kOffV = kOffS + kSParts * kSTile;
  // rows on their way to global memory: a tile of their own where there is room, else the chunk's tile of c
  static constexpr bool kOwnOut = DKB == 1;
  static constexpr uint32_t kOffOut = kOffV + kParts * kTile;
  static constexpr uint32_t kOffT = kOffOut + (kOwnOut ? kTile : 0);
  static constexpr uint32_t kOffBar = kOffT + 2 * sizeof(DecayTable);
  static constexpr uint32_t kBytes = kOffBar + kBarBytes;
};
static_assert(Cfg<2, false, 3>::kBytes <= 232448 && Cfg<2, true, 2>::kBytes <= 232448, "shared memory of a CTA");

struct Item {
  int job, seq, h, slice, seg, lane;
  int start, len;   // tokens of the sequence in the flattened order
  int n;            // this item's chunks
  int first, step;  // first token of the first of them in the sequence, and to the next one's
  bool resume, save;  // goes on from the CTA before; is gone on with by the next one
};

// A CTA's share of all lanes' chunks in a row.  It is at least one lane, so that
// a lane is cut at most once: the share is the end of a lane, whole lanes, and
// the start of another.
struct Share {
  int lane0, at0, lane1, at1;  // from chunk at0 of lane0 up to chunk at1 of lane1
  __device__ __forceinline__ void set(int lanes, int chunks) {
    const int64_t all = static_cast<int64_t>(lanes) * chunks, cta = blockIdx.x, ctas = gridDim.x;
    const int64_t lo = cta * all / ctas, hi = (cta + 1) * all / ctas;
    lane0 = static_cast<int>(lo / chunks);
    at0 = static_cast<int>(lo - static_cast<int64_t>(lane0) * chunks);
    lane1 = static_cast<int>(hi / chunks);
    at1 = static_cast<int>(hi - static_cast<int64_t>(lane1) * chunks);
  }
  __device__ __forceinline__ int whole() const { return lane0 + (at0 > 0 ? 1 : 0); }  // the first one
  __device__ __forceinline__ int items() const { return lane1 - whole() + 2; }
};

__device__ __forceinline__ bool item_of(const LaChunkArgs& a, const Share& s, int idx, Item* it) {
  const int all = a.lanes[a.la.njobs];
  int from = 0, till = 0;  // of its chunks, with even shares
  if (a.hand != nullptr) {
    // the start that another CTA goes on from comes first, and the end that needs another's state last
    const int chunks = static_cast<int>((a.la.T + kC - 1) / kC);
    const int last = s.items() - 1;
    it->save = idx == 0;
    it->resume = idx == last;
    it->lane = idx == 0 ? min(s.lane1, all - 1) : idx == last ? s.lane0 : s.whole() + idx - 1;
    from = idx == last ? s.at0 : 0;
    till = idx == 0 ? s.at1 : idx == last && s.at0 == 0 ? 0 : chunks;
    it->seg = 0;
  } else {
    it->save = it->resume = false;
    it->seg = idx / all;
    it->lane = idx - it->seg * all;
  }
  int j = 0;
  while (j + 1 < a.la.njobs && it->lane >= a.lanes[j + 1]) ++j;
  it->job = j;
  int r = it->lane - a.lanes[j];
  it->slice = r % a.slices[j];
  r /= a.slices[j];
  it->h = r % a.la.H;
  it->seq = r / a.la.H;
  if (a.order != nullptr) it->seq = __ldg(a.order + it->seq);
  bool ok = true;
  if (a.la.cu == nullptr) {
    it->start = static_cast<int>(it->seq * a.la.T);
    it->len = static_cast<int>(a.la.T);
  } else {
    const int lo = __ldg(a.la.cu + it->seq), hi = __ldg(a.la.cu + it->seq + 1);
    ok = lo >= 0 && hi >= lo && hi <= a.la.total;
    it->start = ok ? lo : 0;
    it->len = ok ? hi - lo : 0;
  }
  const int nch = (it->len + kC - 1) / kC;
  const int per = (nch + a.nseg - 1) / a.nseg;
  const int p0 = a.hand != nullptr ? from : min(it->seg * per, nch);
  it->n = a.hand != nullptr ? till - from : min(per, nch - p0);
  const bool rev = a.la.job[j].reverse != 0;
  it->first = (rev ? nch - 1 - p0 : p0) * kC;
  it->step = rev ? -kC : kC;
  return ok;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// mbar_wait that counts cycles instead of reading the timer: the kernel's 32
// warps run through a dozen loops at once, and what the instruction cache does
// not hold is fetched again for every chunk, so its hot code has to stay small.
// A wait that gives up leaves its code in shared memory; the CTA's end records it.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* failed, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const int64_t start = clock64();
  do {
    if (mbar_try_wait(bar, parity)) return true;
  } while (clock64() - start < kWaitCycles);
  *failed = code;
  return false;
}

// Registers move between warpgroups; every warp of one executes the same instruction.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Whether a phase is over, at once (a try_wait may sleep first).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0u;
}

// A wait whose first poll was made earlier, so that its latency has passed.
__device__ __forceinline__ bool wait_after(bool polled, uint64_t* bar, uint32_t parity, int* failed, int code) {
  if (__all_sync(0xFFFFFFFFu, polled) != 0) return true;
  return __all_sync(0xFFFFFFFFu, wait_for(bar, parity, failed, code)) != 0;
}

// A flag in global memory that another CTA sets.
__device__ __forceinline__ bool wait_flag(const int* flag, int* failed) {
  const int64_t start = clock64();
  int set;
  do {
    asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(set) : "l"(flag) : "memory");
  } while (set == 0 && clock64() - start < kWaitCycles);
  if (set == 0) *failed = SPX_DEV_TIMEOUT_PRODUCER;
  return __all_sync(0xFFFFFFFFu, set != 0) != 0;
}

// Every lane polls; the warp goes on together, or gives up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* failed, int code) {
  return __all_sync(0xFFFFFFFFu, wait_for(bar, parity, failed, code)) != 0;
}

__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// One lane of the warp, the same one every time.  MMAs are issued in branches on
// this and not on a lane number, and everything around them runs in the whole
// warp: only then does the compiler know the branch as one thread's and the
// descriptors as uniform, and an MMA of 64, 128 or 256 columns issues every 48,
// 64 or 126 cycles instead of every 75 and more.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0u;
}

// D[tmem] (+)= A[tmem] * B[smem]^T, BF16: A holds two K elements per column.
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[16]) {  // the first eight
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major operand of [128-byte rows along K][64 MN elements] tiles, 128-byte
// swizzle; the next 64 MN elements are `lbo` bytes on.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// Byte offset of 16-byte chunk `c` of 128-byte row `row` in a 128B-swizzled tile.
__device__ __forceinline__ uint32_t swz(int row, int c) {
  return static_cast<uint32_t>(row) * 128u + static_cast<uint32_t>((c ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair(uint32_t x, uint32_t y) { return pair(__uint_as_float(x), __uint_as_float(y)); }
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Two floats as NP packed BF16 parts whose sum they are: one part is the
// rounding, two leave 2^-18 of the value, three are exact (three truncations of
// eight bits each).
template <int NP>
__device__ __forceinline__ void split2(uint64_t v, uint32_t (&part)[NP]) {
  float x, y;
  unpair(v, x, y);
  if constexpr (NP < 3) {
    part[0] = pack_bf16(x, y);
    if constexpr (NP == 2) {
      unpair(add2(v, pair((part[0] << 16) ^ 0x80000000u, (part[0] & 0xFFFF0000u) ^ 0x80000000u)), x, y);
      part[1] = pack_bf16(x, y);
    }
  } else {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
      part[p] = __byte_perm(ux, uy, 0x7632);
      if (p < 2) {
        v = add2(v, pair((ux & 0xFFFF0000u) ^ 0x80000000u, (uy & 0xFFFF0000u) ^ 0x80000000u));
        unpair(v, x, y);
      }
    }
  }
}

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst_smem, const void* src, bool copy) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(copy ? 16 : 0) : "memory");
}

struct Bars {
  uint64_t full_ab[3], full_c[3], empty_a[3], empty_b[3], empty_c[3];  // per stage
  uint64_t gfull[2], gfree[2];
  uint64_t pacc[2], pop[2];
  uint64_t tail[2];  // at most one tail is fixed ahead of the one being waited for
  uint64_t kvgo[2], kv[2];  // by the chunk's parity: scaled c is there and the accumulator free; the product done
  uint64_t qsgo, qs;        // the state's operand is there and the output's accumulators free; a . S done
  uint64_t o, drained;
  uint64_t qfull[4], qfree[4];  // of the items taken from the queue
  int taken[4];
  int items;
  Share share;
  uint32_t tmem;
  int failed;
};
static_assert(sizeof(Bars) <= kBarBytes, "barriers");

}  // namespace

template <int DKB, bool PRECISE, int PARTS>
__global__ void __launch_bounds__(kLaThreads, 1) la_chunk_kernel(const __grid_constant__ LaChunkArgs args) {
  using K = Cfg<DKB, PRECISE, PARTS>;
  extern __shared__ __align__(1024) uint8_t la_smem[];
  const uint32_t base = smem_u32(la_smem);
  int* const status = args.la.status;
  if ((base & 1023u) != 0u) {  // the swizzled tiles need it; uniform over the CTA
    if (threadIdx.x == 0) record_error(status, SPX_DEV_BAD_TILE);
    return;
  }
  Bars& bar = *reinterpret_cast<Bars*>(la_smem + K::kOffBar);
  int* const failed = &bar.failed;
  DecayTable* const tables = reinterpret_cast<DecayTable*>(la_smem + K::kOffT);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform to the compiler
  const bool full_pass = args.state_only == 0;
  const int item0 = args.hand != nullptr ? 0 : blockIdx.x, item_step = args.hand != nullptr ? 1 : gridDim.x;
  // The state-only pass has room for two chunks' parts of scaled c (the second in
  // the places of a and of the state's operand) and two accumulators, so that
  // scaling, product and update of neighbouring chunks overlap.
  const uint32_t depth = full_pass ? 1u : 2u;
  auto part_at = [&](uint32_t n, uint32_t part) {  // the part's tile for chunk n
    if (full_pass || (n & 1u) == 0u) return base + K::kOffV + part * kTile;
    if constexpr (DKB == 1) return base + part * K::kStage;
    return part < 2u ? base + part * kTile : base + K::kOffS;
  };
  auto acc_at = [&](uint32_t n) { return full_pass || (n & 1u) == 0u ? kTmKV : kTmP; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 3; ++s) {
      mbar_init(&bar.full_ab[s], 1);
      mbar_init(&bar.full_c[s], 1);
      mbar_init(&bar.empty_a[s], 1);
      mbar_init(&bar.empty_b[s], 1);
      mbar_init(&bar.empty_c[s], full_pass && !K::kOwnOut ? 9 : 1);  // the MMAs, and the epilogue's warps
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar.gfull[s], 1);
      mbar_init(&bar.gfree[s], full_pass ? 28 : 12);
      mbar_init(&bar.pacc[s], 1);
      mbar_init(&bar.pop[s], 8);
      mbar_init(&bar.tail[s], 8);
      mbar_init(&bar.kvgo[s], 12);
      mbar_init(&bar.kv[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bar.qfull[s], 1);
      mbar_init(&bar.qfree[s], full_pass ? 31 : 15);  // every warp that takes items but the one that fetches them
    }
    mbar_init(&bar.qsgo, 12);
    mbar_init(&bar.qs, 1);
    mbar_init(&bar.o, 1);
    mbar_init(&bar.drained, 1);
    bar.failed = 0;
    bar.items = args.lanes[args.la.njobs] * args.run_segs;
    if (args.hand != nullptr) {
      bar.share.set(bar.items, static_cast<int>((args.la.T + kC - 1) / kC));
      bar.items = bar.share.items();
    }
    fence_mbar_init();
  }
  if (warp == 29) {
    tmem_alloc(&bar.tmem, kTmCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const int items = bar.items;
  const int quad = warp & 3;
  const uint32_t tm_lane = static_cast<uint32_t>(quad * 32) << 16;
  const int row = quad * 32 + lane;  // this thread's TMEM lane / tile row
  bool ok = true;
  uint32_t it = 0;  // chunks so far, the same count in every role
  uint32_t st = 0, ph = 0;  // it % kStages, and the parity of it / kStages
  auto advance = [&]() {
    ++it;
    if (++st == K::kStages) {
      st = 0;
      ph ^= 1u;
    }
  };
  // Items: a fixed stride, or for packed sequences (longest first) a queue that all
  // CTAs take from; the warp of c's TMA fetches one ahead and hands it to the others.
  uint32_t nitem = 0;  // taken so far, the CTA's first item (its index) apart
  auto next_item = [&](int idx) {
    if (args.order == nullptr) return idx + item_step;
    const uint32_t slot = nitem & 3u;
    if (!(ok = warp_wait(&bar.qfull[slot], (nitem >> 2) & 1u, failed, SPX_DEV_TIMEOUT_PRODUCER))) return items;
    const int got = *const_cast<volatile int*>(&bar.taken[slot]);
    warp_arrive(&bar.qfree[slot], lane);
    ++nitem;
    return got;
  };

  if (warp < 8) {
    // ---------------- the decayed a . b matrix: 16 columns of each 32-token block
    const int half = warp >> 2;
    for (int idx = item0; full_pass && ok && idx < items; idx = next_item(idx)) {
      Item w;
      item_of(args, bar.share, idx, &w);
      const bool rev = w.step < 0;
      // of this row's words in the diagonal block: a masked entry is zero whatever it holds
      uint32_t mask[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int c = 16 * half + 2 * q;
        mask[q] = ((rev ? c >= lane : c <= lane) ? 0xFFFFu : 0u) | ((rev ? c + 1 >= lane : c + 1 <= lane) ? 0xFFFF0000u : 0u);
      }
      for (int p = 0; p < w.n; ++p, ++it) {
        const uint32_t b = it & 1u, ph = (it >> 1) & 1u;
        const DecayTable& t = tables[b];
        if (!(ok = warp_wait(&bar.gfull[b], ph, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        const float a = t.a[row];
        if (!(ok = warp_wait(&bar.pacc[b], ph, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        // The operand takes the accumulator's place: 16 FP32 columns become 8 of BF16
        // pairs (PRECISE: 8 more of their second parts).  From the diagonal block
        // outwards; `run` is the decay between this row and the near edge of the block.
        const uint32_t acc = tmem + kTmP + b * 128u + tm_lane;
        const float own = t.total[quad];
        // inside the diagonal block the two factors are on either side of 1; a block
        // that decays by more than 2^100 takes the exponential of each difference
        float run = a - own;
        const bool steep = !(own >= -100.0f);
        uint32_t x[16];  // a block's columns; once they are multiplied, the next block's are on their way
        tmem_ld16(acc + 32u * quad + 16u * half, x);
#pragma unroll 1
        for (int n = 0; n < 4; ++n) {
          const int j = (rev ? quad + n : quad - n) & 3;
          const int c0 = 32 * j + 16 * half;
          uint32_t words[16];
          if (rev ? j < quad : j > quad) {
#pragma unroll
            for (int q = 0; q < 16; ++q) words[q] = 0u;
          } else {
            const float rf = ex2(run);
            const uint64_t rf2 = pair(rf, rf);
            run = n == 0 ? a : run + t.total[j];  // its own block's part directly, whatever comes after the row
            const ulonglong2* f4 = reinterpret_cast<const ulonglong2*>(t.cf + c0);
            uint64_t f[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const ulonglong2 v = f4[q];
              f[2 * q] = mul2(v.x, rf2);
              f[2 * q + 1] = mul2(v.y, rf2);
            }
            if (n == 0 && steep) {
#pragma unroll
              for (int q = 0; q < 8; ++q) f[q] = pair(ex2(a - t.a[c0 + 2 * q]), ex2(a - t.a[c0 + 2 * q + 1]));
            }
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = mul2(pair(x[2 * q], x[2 * q + 1]), f[q]);
            if (rev ? j < 3 : j > 0) tmem_ld16(acc + (rev ? c0 + 32 : c0 - 32), x);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              uint32_t part[PRECISE ? 2 : 1];
              split2<PRECISE ? 2 : 1>(f[q], part);
              words[q] = part[0];
              if constexpr (PRECISE) words[8 + q] = part[1];
            }
            if (n == 0) {
#pragma unroll
              for (int q = 0; q < (PRECISE ? 16 : 8); ++q) words[q] &= mask[q & 7];
            }
          }
          if constexpr (PRECISE)
            tmem_st16(acc + c0, words);
          else
            tmem_st8(acc + c0, words);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&bar.gfree[b], lane);
        warp_arrive(&bar.pop[b], lane);
      }
    }
  } else if (warp < 16) {
    regs_down<kRegsC>();
    const int half = warp >> 2 & 1;  // 32 of the 64 columns
    // ---------------- scaled c
    uint32_t tails = 0;
    for (int idx = item0; ok && idx < items; idx = next_item(idx)) {
      Item w;
      item_of(args, bar.share, idx, &w);
      const bool rev = w.step < 0;
      int left = w.len - w.first;  // tokens from the chunk's first one on
      for (int p = 0; p < w.n; ++p, advance(), left -= w.step) {
        const uint32_t b = it & 1u;
        const int len = left;
        if (!(ok = warp_wait(&bar.full_c[st], ph, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        const uint32_t stage = base + st * K::kStage;
        const uint32_t sc_row = stage + 2 * DKB * kTile + swz(row, 0);  // ^ (c << 4): the row's chunk c
        if (len < kC && args.la.cu != nullptr) {
          // packed: the rows past the sequence are another's (or nobody's); nothing of them may enter a sum.  A thread
          // zeroes the chunks of c that it scales below: the row's other half is another warp's.
          if (!(ok = warp_wait(&bar.full_ab[st], ph, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
          if (row >= len) {
#pragma unroll
            for (int x = 0; x < DKB + 1; ++x)
#pragma unroll
              for (int c = 0; c < 4; ++c) sts16(stage + (DKB + x) * kTile + swz(row, 4 * half + c), 0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          if (full_pass) warp_arrive(&bar.tail[tails++ & 1u], lane);  // else the product alone reads them, after vp
        }
        if (!(ok = warp_wait(&bar.gfull[b], (it >> 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        const float wgt = out_of_token(tables[b], quad, row, rev);
        warp_arrive(&bar.gfree[b], lane);
        const uint64_t wgt2 = pair(wgt, wgt);
        // the parts' last reader: the state product of the chunk before (or the one before that)
        if (it >= depth && !(ok = warp_wait(&bar.kv[(it - depth) & 1u], ((it - depth) >> 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        uint32_t dst[K::kParts];
#pragma unroll
        for (int part = 0; part < K::kParts; ++part) dst[part] = part_at(it, part) + swz(row, 0);
#pragma unroll 1
        for (int c = 4 * half; c < 4 * half + 4; ++c) {
          const uint4 u = lds16(sc_row ^ (c << 4));
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
          uint32_t q[4][K::kParts];
#pragma unroll
          for (int e = 0; e < 4; ++e) split2<K::kParts>(mul2(pair(uw[e] << 16, uw[e] & 0xFFFF0000u), wgt2), q[e]);
#pragma unroll
          for (int part = 0; part < K::kParts; ++part)
            sts16(dst[part] ^ (c << 4), q[0][part], q[1][part], q[2][part], q[3][part]);
        }
        fence_proxy_async_smem();
        warp_arrive(&bar.kvgo[b], lane);
      }
    }
  } else if (warp < 20) {
    regs_up<K::kRegsState>();
    // ---------------- the state: 64 (or 32) columns of one row of da, in registers
    constexpr int kN = K::kStateCols / 2;  // pairs of columns
    const int row = (DKB == 1 ? quad & 1 : quad) * 32 + lane;
    const int part_col = DKB == 1 ? (quad >> 1) * 32 : 0;
    for (uint32_t n = 0; n < depth; ++n) warp_arrive(&bar.kvgo[n], lane);  // the accumulators are free at first
    for (int idx = item0; ok && idx < items; idx = next_item(idx)) {
      Item w;
      const bool sound = item_of(args, bar.share, idx, &w);
      if (args.hand != nullptr && w.n == 0) continue;
      const LaJob& j = args.la.job[w.job];
      if (!sound && threadIdx.x == 512) *failed = SPX_DEV_BAD_TILE;  // and it counts as an empty sequence
      uint64_t s[kN];
      const int64_t st0 = (static_cast<int64_t>(w.seq) * args.la.H + w.h) * j.da * j.dc;
      const int col0 = w.slice * 64 + part_col;
      const bool live = row < j.da;
      float* const seg = args.seg_state == nullptr ? nullptr : args.seg_state + ((static_cast<int64_t>(w.lane) * args.nseg + w.seg) * 128 + row) * 64 + part_col;
      if ((args.nseg > 1 && full_pass) || w.resume) {
        const float* from = seg;
        if (w.resume) {  // its start was its CTA's first item, so that it has long been done
          from = args.hand + (static_cast<int64_t>(blockIdx.x - 1) * 128 + row) * 64 + part_col;
          if (!(ok = wait_flag(args.handed + (blockIdx.x - 1) * 4 + quad, failed))) break;
        }
        const float4* f = reinterpret_cast<const float4*>(from);
#pragma unroll
        for (int q = 0; q < kN / 2; ++q) {
          const float4 v = live ? __ldcg(f + q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          s[2 * q] = pair(v.x, v.y);
          s[2 * q + 1] = pair(v.z, v.w);
        }
      } else {
        const float* f = j.init + st0 + row * j.s_row + col0 * j.s_col;
        const int n = j.init != nullptr && args.nseg == 1 && live ? j.dc - col0 : 0;
        if (j.s_col == 1) {  // a thread's columns side by side: widths are multiples of 8
#pragma unroll
          for (int c = 0; c < kN; c += 2) {
            const float4 v = 2 * c < n ? __ldg(reinterpret_cast<const float4*>(f + 2 * c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            s[c] = pair(j.init_scale * v.x, j.init_scale * v.y);
            s[c + 1] = pair(j.init_scale * v.z, j.init_scale * v.w);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kN; ++c, f += 2 * j.s_col)
            s[c] = 2 * c < n ? pair(j.init_scale * f[0], j.init_scale * f[j.s_col]) : 0;
        }
      }
      float decay = 1.0f;
      auto write_operand = [&]() {  // BF16 parts of the state for the next chunk's a . S
#pragma unroll
        for (int c = 0; c < kN / 4; ++c) {
          uint32_t q[4][K::kSParts];
#pragma unroll
          for (int e = 0; e < 4; ++e) split2<K::kSParts>(s[4 * c + e], q[e]);
#pragma unroll
          for (int part = 0; part < K::kSParts; ++part)
            sts16(base + K::kOffS + part * K::kSTile + swz(row, part_col / 8 + c), q[0][part], q[1][part], q[2][part], q[3][part]);
        }
        fence_proxy_async_smem();
        warp_arrive(&bar.qsgo, lane);
      };
      for (int p = 0; p < w.n; ++p, ++it) {
        const uint32_t b = it & 1u;
        if (full_pass) {
          // the operand before this chunk; its last reader was the chunk before
          if (it > 0 && !(ok = warp_wait(&bar.qs, (it - 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
          write_operand();
        }
        if (!(ok = warp_wait(&bar.gfull[b], (it >> 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        const float* tt = tables[b].total;
        const float gamma = ex2((tt[0] + tt[1]) + (tt[2] + tt[3]));
        warp_arrive(&bar.gfree[b], lane);
        const uint64_t gamma2 = pair(gamma, gamma);
        decay *= gamma;
        if (!(ok = warp_wait(&bar.kv[b], (it >> 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        const uint32_t acc = tmem + acc_at(it) + tm_lane + part_col;
        tc_fence_after();
#pragma unroll
        for (int part = 0; part < kN / 8; ++part) {
          uint32_t x[16], y[16];
          tmem_ld16(acc + 16u * part, x);
          if constexpr (K::kParts == 2) tmem_ld16(acc + 64u + 16u * part, y);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint64_t add = pair(x[2 * c], x[2 * c + 1]);
            if constexpr (K::kParts == 2) add = add2(add, pair(y[2 * c], y[2 * c + 1]));
            s[8 * part + c] = fma2(gamma2, s[8 * part + c], add);
          }
        }
        tc_fence_before();
        warp_arrive(&bar.kvgo[(it + depth) & 1u], lane);  // for the chunk `depth` on
      }
      if (!ok) break;
      if (!full_pass || w.save) {
        float4* f = reinterpret_cast<float4*>(
            w.save ? args.hand + (static_cast<int64_t>(blockIdx.x) * 128 + row) * 64 + part_col : seg);
        if (live) {
#pragma unroll
          for (int q = 0; q < kN / 2; ++q) *reinterpret_cast<ulonglong2*>(f + q) = make_ulonglong2(s[2 * q], s[2 * q + 1]);
        }
        if (w.save) {
          __threadfence();
          __syncwarp();
          if (lane == 0) atomicExch(args.handed + blockIdx.x * 4 + quad, 1);
        } else if (threadIdx.x == 512) args.seg_decay[static_cast<int64_t>(w.lane) * args.nseg + w.seg] = decay;
      } else if (j.fin != nullptr && w.seg == args.nseg - 1 && live) {
        float* f = j.fin + st0 + row * j.s_row + col0 * j.s_col;
        const int n = j.dc - col0;
        const bool wide = j.s_col == 1;
#pragma unroll
        for (int c = 0; c < kN; c += 2, f += 4 * j.s_col) {
          if (2 * c >= n) break;
          float4 v;
          unpair(s[c], v.x, v.y);
          unpair(s[c + 1], v.z, v.w);
          v = make_float4(j.fin_scale * v.x, j.fin_scale * v.y, j.fin_scale * v.z, j.fin_scale * v.w);
          if (wide) {
            *reinterpret_cast<float4*>(f) = v;
          } else {
            f[0] = v.x;
            f[j.s_col] = v.y;
            f[2 * j.s_col] = v.z;
            f[3 * j.s_col] = v.w;
          }
        }
      }
    }
  } else if (warp < 28) {
    const int half = warp >> 2 & 1;  // 32 of the 64 columns
    // ---------------- epilogue: 32 columns of one token a thread
    if (full_pass) warp_arrive(&bar.qsgo, lane);  // the accumulators are free at first
    for (int idx = item0; full_pass && ok && idx < items; idx = next_item(idx)) {
      Item w;
      item_of(args, bar.share, idx, &w);
      const LaJob& j = args.la.job[w.job];
      const bool rev = w.step < 0, f32 = PRECISE && j.out_f32 != 0;
      const int col0 = w.slice * 64;
      const int valid = min(64, j.dc - col0);  // a multiple of 8
      const bool packed = args.la.cu != nullptr;
      const uint16_t* pe = nullptr;
      if constexpr (PRECISE) {
        if (j.e.p != nullptr)
          pe = j.e.p + (packed ? 0 : w.seq) * j.e.sb + (packed ? w.start : 0) * j.e.st + (w.h / j.e.group) * j.e.sh + col0;
      }
      const int64_t stride = static_cast<int64_t>(args.la.H) * j.dc;
      const int r0 = quad * 32 + (lane >> 2), c4 = 4 * half + (lane & 3);  // rows r0, r0 + 8, ...; 16-byte column
      // the row's decay for the a . S part; read a chunk ahead, so that this role, the
      // last to need a table, does not keep the others waiting for the next
      float factor = 0.0f;
      auto read_factor = [&](uint32_t n) {
        const uint32_t b = n & 1u;
        if (!warp_wait(&bar.gfull[b], (n >> 1) & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE)) return false;
        factor = into_token(tables[b], quad, row, rev);
        warp_arrive(&bar.gfree[b], lane);
        return true;
      };
      if (w.n > 0) ok = read_factor(it);
      int first = w.first;  // the chunk's first token
      int64_t at = (static_cast<int64_t>(w.start) + first + r0) * stride + w.h * j.dc + col0;
      for (int p = 0; ok && p < w.n; ++p, advance(), first += w.step, at += w.step * stride) {
        const int left = w.len - first;  // tokens from there on
        // Rows go through shared memory on their way to and from global memory (four
        // lanes this warp's 64 bytes of a row): a thread's own row would touch 32 lines an
        // instruction and hold up every barrier and shared-memory access of the CTA.
        const uint32_t tile = base + (K::kOwnOut ? K::kOffOut : st * K::kStage + 2 * DKB * kTile);
        auto fetch_e = [&]() {  // rows past the sequence and columns past the width read as zero
          const uint16_t* src = pe + (first + r0) * j.e.st + 8 * c4;
#pragma unroll
          for (int q = 0; q < 4; ++q, src += 8 * j.e.st) {
            const bool in = r0 + 8 * q < left && 8 * c4 < valid;
            cp_async16_or_zero(tile + swz(r0 + 8 * q, c4), in ? src : pe, in);
          }
        };
        if constexpr (PRECISE && K::kOwnOut) {
          if (pe != nullptr) fetch_e();
        }
        const float sc = args.la.scale, sx = sc * factor;
        const uint64_t sc2 = pair(sc, sc), sx2 = pair(sx, sx);
        if (p + 1 < w.n && !(ok = read_factor(it + 1))) break;
        if (!(ok = warp_wait(&bar.o, it & 1u, failed, SPX_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        if constexpr (PRECISE) {
          if (pe != nullptr) {
            if constexpr (!K::kOwnOut) fetch_e();  // the tile is the chunk's c, free now
            cp_async_wait_all();
            __syncwarp();
          }
        }
        uint64_t dot[2] = {0, 0};  // four FP32 sums
        uint32_t x[16], y[16];
        const uint32_t tm = tmem + tm_lane + 32u * half;
#pragma unroll 1
        for (uint32_t part = 0; part < 2; ++part) {  // 16 columns
          tmem_ld16(tm + kTmOI + 16u * part, x);
          tmem_ld16(tm + kTmOX + 16u * part, y);
          tmem_wait_ld();
          if (part == 1u) {
            // the accumulators are free before the stores: the next chunk's products wait for them
            tc_fence_before();
            warp_arrive(&bar.qsgo, lane);
          }
          uint64_t v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fma2(sx2, pair(y[2 * i], y[2 * i + 1]), mul2(sc2, pair(x[2 * i], x[2 * i + 1])));
          if constexpr (PRECISE) {
            if (f32) {  // (no dots then) 16 columns at a time fill this warp's half of the tile
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float z[4];
                unpair(v[2 * q], z[0], z[1]);
                unpair(v[2 * q + 1], z[2], z[3]);
                sts16(tile + swz(row, 4 * half + q), __float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]),
                      __float_as_uint(z[3]));
              }
              __syncwarp();
              const int c = 32 * half + 16 * part + 4 * (lane & 3);
              float* dst = reinterpret_cast<float*>(j.out) + at + c;
#pragma unroll
              for (int q = 0; q < 4; ++q, dst += 8 * stride)
                if (r0 + 8 * q < left && c < valid) *reinterpret_cast<uint4*>(dst) = lds16(tile + swz(r0 + 8 * q, c4));
              __syncwarp();
            } else if (pe != nullptr) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint4 u = lds16(tile + swz(row, 4 * half + 2 * part + q));
                const uint32_t ew[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  dot[i & 1] = fma2(v[4 * q + i], pair(ew[i] << 16, ew[i] & 0xFFFF0000u), dot[i & 1]);
              }
            }
          }
          if (!f32) {  // over the e that has just been read
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t o[4][1];
#pragma unroll
              for (int i = 0; i < 4; ++i) split2<1>(v[4 * q + i], o[i]);
              sts16(tile + swz(row, 4 * half + 2 * part + q), o[0][0], o[1][0], o[2][0], o[3][0]);
            }
          }
        }
        uint4 rows[4];
        if (!f32) {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) rows[q] = lds16(tile + swz(r0 + 8 * q, c4));
        }
        if constexpr (K::kOwnOut) {
          __syncwarp();  // before the next chunk's rows
        } else {
          fence_proxy_async_smem();  // before the next copy lands here
          warp_arrive(&bar.empty_c[st], lane);
        }
        if (!f32) {
          uint16_t* dst = reinterpret_cast<uint16_t*>(j.out) + at + 8 * c4;
#pragma unroll
          for (int q = 0; q < 4; ++q, dst += 8 * stride)
            if (r0 + 8 * q < left && 8 * c4 < valid) *reinterpret_cast<uint4*>(dst) = rows[q];
        }
        if constexpr (PRECISE) {
          if (pe != nullptr && row < left) {
            float d0, d1;
            unpair(add2(dot[0], dot[1]), d0, d1);
            j.dots[(static_cast<int64_t>(2 * w.slice + half) * args.la.H + w.h) * args.la.total + w.start + first + row] = d0 + d1;
          }
        }
      }
    }
  } else {
    regs_down<kRegsRest>();
    if (warp == 28 || warp == 31) {
    // ---------------- TMA: a and b, and in a warp of its own c, whose tile is free later
    const bool ab = warp == 28;
    uint64_t* const full = ab ? bar.full_ab : bar.full_c;
    // The next item, from the queue into its place: at once if the place is free, and at the latest after this
    // item's copies, which the roles that are to free it may be waiting for.
    auto hand_out = [&](int got, bool wait) {
      const uint32_t slot = nitem & 3u, parity = ((nitem >> 2) & 1u) ^ 1u;
      if (!(wait ? wait_for(&bar.qfree[slot], parity, failed, SPX_DEV_TIMEOUT_PRODUCER) : mbar_test(&bar.qfree[slot], parity)))
        return false;
      bar.taken[slot] = got < items ? got : items;
      mbar_arrive(&bar.qfull[slot]);
      return true;
    };
    const bool queue = args.order != nullptr && !ab;
    int idx = item0;
    while (ok && idx < items) {
      Item w;
      item_of(args, bar.share, idx, &w);
      if (lane == 0) {
        const int got = queue ? atomicAdd(args.queue, 1) : 0;
        const bool handed = !queue || hand_out(got, false);
        const LaJob& j = args.la.job[w.job];
        const bool packed = args.la.cu != nullptr;
        const int batch = packed ? 0 : w.seq;
        int t = (packed ? w.start : 0) + w.first;
        for (int p = 0; p < w.n; ++p, advance(), t += w.step) {
          const uint32_t stage = base + st * K::kStage;
          if (!ab) {
            if (!(ok = wait_for(&bar.empty_c[st], ph ^ 1u, failed, SPX_DEV_TIMEOUT_PRODUCER))) break;
            mbar_arrive_expect_tx(&full[st], kTile);
            tma_load_4d(stage + 2 * DKB * kTile, &args.map[w.job][2], &full[st], 64 * w.slice, w.h / j.c.group, t, batch);
            continue;
          }
          if (!(ok = wait_for(&bar.empty_b[st], ph ^ 1u, failed, SPX_DEV_TIMEOUT_PRODUCER))) break;
          mbar_arrive_expect_tx(&full[st], (full_pass ? 2 * DKB : DKB) * kTile);
          for (int x = 0; x < DKB; ++x)
            tma_load_4d(stage + (DKB + x) * kTile, &args.map[w.job][1], &full[st], 64 * x, w.h / j.b.group, t, batch);
          if (full_pass) {
            // with b's copies on their way the count has to come to its end: a's follow even after a failed wait
            ok = wait_for(&bar.empty_a[st], ph ^ 1u, failed, SPX_DEV_TIMEOUT_PRODUCER);
            for (int x = 0; x < DKB; ++x)
              tma_load_4d(stage + x * kTile, &args.map[w.job][0], &full[st], 64 * x, w.h / j.a.group, t, batch);
            if (!ok) {
              advance();
              break;
            }
          }
        }
        if (ok && !handed) ok = hand_out(got, true);
      }
      ok = __all_sync(0xFFFFFFFFu, ok) != 0;
      __syncwarp();
      if (!queue) {
        idx = next_item(idx);
      } else {
        idx = *const_cast<volatile int*>(&bar.taken[nitem & 3u]);
        ++nitem;
      }
    }
    if (lane == 0 && !ok) {  // leave no copy in flight behind an abandoned pipeline
      for (int s = 0; s < K::kStages && static_cast<uint32_t>(s) < it; ++s) {
        const uint32_t last = it - 1 - ((it - 1 - s) % K::kStages);  // the newest chunk loaded into stage s
        wait_for(&full[s], (last / K::kStages) & 1u, failed, SPX_DEV_TIMEOUT_PRODUCER);
      }
    }
    } else if (warp == 29) {
    // ---------------- MMA
    {
      const uint32_t id_ab = idesc_bf16_f32(128, 128);
      const uint32_t id_o = idesc_bf16_f32(128, 64) | (1u << 16);               // B MN-major
      const uint32_t id_kv = idesc_bf16_f32(128, K::kParts == 3 ? 64 : 128) | (1u << 15) | (1u << 16);  // A and B MN-major
      uint32_t tails = 0;
      uint32_t ast = 0, aph = 0;  // stage and parity of the chunk to start
      auto product_ab = [&](uint32_t n) {  // a . b of chunk n
        const uint32_t sa = base + ast * K::kStage;
        const uint64_t da = desc_kmajor_sw128(sa), db = desc_kmajor_sw128(sa + DKB * kTile);
        const uint32_t acc = tmem + kTmP + (n & 1u) * 128u;
        if (elect_one()) {
#pragma unroll
          for (uint32_t k = 0; k < 4 * DKB; ++k) {
            const uint32_t at = ((k >> 2) * kTile + (k & 3u) * 32u) >> 4;
            mma_bf16_ss(acc, da + at, db + at, id_ab, k != 0u ? 1u : 0u);
          }
          mma_commit(&bar.pacc[n & 1u]);
        }
        __syncwarp();
      };
      // a . b runs one chunk ahead, over item borders
      int nidx = item0, np = 0;  // the next chunk to start
      Item nw{};
      bool more = nidx < items;
      if (more) item_of(args, bar.share, nidx, &nw);
      // Looks for the item of the next chunk.  The queue frees a place only when every role is through with an older
      // item, and they may wait for this warp's products: it waits for the queue only when it owes them none.
      auto settle = [&](bool owing) {
        while (more && np >= nw.n) {
          if (owing && args.order != nullptr &&
              __all_sync(0xFFFFFFFFu, mbar_test(&bar.qfull[nitem & 3u], (nitem >> 2) & 1u)) == 0)
            return;
          nidx = next_item(nidx);
          np = 0;
          if ((more = nidx < items)) item_of(args, bar.share, nidx, &nw);
        }
      };
      uint32_t ahead = 0;  // chunks whose a . b has been issued (state-only: whose tiles are there)
      auto start_next = [&](bool polled) {
        if (!more || np >= nw.n) return true;
        if (!wait_after(polled, &bar.full_ab[ast], aph, failed, SPX_DEV_TIMEOUT_MMA)) return false;
        // the tail of a packed sequence: its rows are zeroed first
        if (full_pass && args.la.cu != nullptr && nw.len - (nw.first + np * nw.step) < kC) {
          if (!warp_wait(&bar.tail[tails & 1u], (tails >> 1) & 1u, failed, SPX_DEV_TIMEOUT_MMA)) return false;
          ++tails;
        }
        tc_fence_after();
        // its accumulator's last reader is the product with c two chunks before: done, as the
        // epilogue of that chunk has freed the output for the a . S issued before this
        if (full_pass) product_ab(ahead);
        ++ahead;
        ++np;
        if (++ast == K::kStages) {
          ast = 0;
          aph ^= 1u;
        }
        return true;
      };
      bool kv_ready = false, qs_ready = false, ab_ready = false, pop_ready = false;
      while (ok) {
        const bool owing = it < ahead;
        const uint32_t b = it & 1u, ph2 = (it >> 1) & 1u;
        const uint32_t stage = base + st * K::kStage;
        if (owing) {
          // A satisfied wait still takes a few hundred cycles of a busy CTA: each is polled one product ahead.
          // state product b^T (scaled c)
          if (!(ok = wait_after(kv_ready, &bar.kvgo[b], ph2, failed, SPX_DEV_TIMEOUT_MMA))) break;
          tc_fence_after();
          qs_ready = full_pass && mbar_test(&bar.qsgo, it & 1u);
          ab_ready = mbar_test(&bar.full_ab[ast], aph);
          const uint64_t db = desc_mn(stage + DKB * kTile, DKB == 1 ? 0u : kTile);  // 64 columns: the same rows twice
          uint64_t dv[K::kParts];  // (two parts: the first, with the distance to the second)
#pragma unroll
          for (uint32_t part = 0; part < K::kParts; ++part) dv[part] = desc_mn(part_at(it, part), part_at(it, 1) - part_at(it, 0));
          const uint32_t acc = tmem + acc_at(it);
          if (elect_one()) {
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
              // two parts side by side are one MMA of 128 columns, which reads b once; three go one after another
              // into the same 64 (MMAs of different shapes on one accumulator have no order)
#pragma unroll
              for (uint32_t part = 0; part < (K::kParts == 3 ? 3u : 1u); ++part)
                mma_bf16_ss(acc, db + q * 128u, dv[part] + q * 128u, id_kv, (part | q) != 0u ? 1u : 0u);
            }
            mma_commit(&bar.kv[b]);
            mma_commit(&bar.empty_b[st]);  // a . b of this chunk was issued before
            if (!full_pass) mma_commit(&bar.empty_c[st]);
          }
          __syncwarp();
          if (full_pass) {
            // a . S
            if (!(ok = wait_after(qs_ready, &bar.qsgo, it & 1u, failed, SPX_DEV_TIMEOUT_MMA))) break;
            tc_fence_after();
            pop_ready = mbar_test(&bar.pop[b], ph2);
            const uint64_t da = desc_kmajor_sw128(stage), ds = desc_mn(base + K::kOffS, kTile);
            if (elect_one()) {
#pragma unroll
              for (uint32_t n = 0; n < 4 * DKB; ++n) {
#pragma unroll
                for (uint32_t part = 0; part < K::kSParts; ++part)
                  mma_bf16_ss(tmem + kTmOX, da + (((n >> 2) * kTile + (n & 3u) * 32u) >> 4),
                              ds + (part * (K::kSTile >> 4) + n * 128u), id_o, (part | n) != 0u ? 1u : 0u);
              }
              mma_commit(&bar.qs);
              mma_commit(&bar.empty_a[st]);
            }
            __syncwarp();
          }
        }
        settle(owing);
        if (!(ok = ok && start_next(ab_ready))) break;
        kv_ready = mbar_test(&bar.kvgo[b ^ 1u], ((it + 1) >> 1) & 1u);
        if (!owing) {
          if (it == ahead) break;  // there is no next one
          kv_ready = false;
          continue;
        }
        if (full_pass) {
          // (decayed a . b) c
          if (!(ok = wait_after(pop_ready, &bar.pop[b], ph2, failed, SPX_DEV_TIMEOUT_MMA))) break;
          tc_fence_after();
          const uint64_t dc = desc_mn(stage + 2 * DKB * kTile, kTile);
          if (elect_one()) {
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
#pragma unroll
              for (uint32_t part = 0; part < (PRECISE ? 2u : 1u); ++part)
                mma_bf16_ts(tmem + kTmOI, tmem + kTmP + b * 128u + q * 16u + part * 8u, dc + q * 128u, id_o,
                            (part | q) != 0u ? 1u : 0u);
            }
            mma_commit(&bar.o);
            mma_commit(&bar.empty_c[st]);
          }
          __syncwarp();
        }
        advance();
      }
      if (elect_one()) mma_commit(&bar.drained);  // arrives once everything issued above has completed
      __syncwarp();
    }
    } else if (warp == 30) {
    // ---------------- decay tables: lane l of block b is token 32 b + l
    for (int idx = item0; ok && idx < items; idx = next_item(idx)) {
      Item w;
      item_of(args, bar.share, idx, &w);
      const bool rev = w.step < 0;
      const bool packed = args.la.cu != nullptr;
      const int64_t g0 = (packed ? 0 : w.seq) * args.la.g_sb + (packed ? w.start : 0) * args.la.g_st + w.h * args.la.g_sh;
      uint32_t next[4];  // raw: nothing of a load is used before the next chunk
      const bool f32 = args.la.g_f32 != 0;
      int t = w.first + lane;
      auto fetch = [&]() {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          next[q] = 0u;  // past the sequence: no decay
          if (t + 32 * q < w.len) {
            const int64_t at = g0 + (t + 32 * q) * args.la.g_st;
            if (f32)
              next[q] = __ldg(reinterpret_cast<const uint32_t*>(args.la.g) + at);
            else
              next[q] = __ldg(reinterpret_cast<const uint16_t*>(args.la.g) + at);
          }
        }
        t += w.step;
      };
      if (w.n > 0) fetch();
      for (int p = 0; p < w.n; ++p, ++it) {
        const uint32_t b = it & 1u;
        float up[4], down[4];  // sums up to the lane's token, and after it
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = __uint_as_float(f32 ? next[q] : next[q] << 16) * 1.44269504088896340736f;  // log2 e
          up[q] = x < -150.0f ? -150.0f : x;                                                         // a NaN stays
          const float after = __shfl_down_sync(0xFFFFFFFFu, up[q], 1);
          down[q] = lane == 31 ? 0.0f : after;
        }
        if (p + 1 < w.n) fetch();
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float u = __shfl_up_sync(0xFFFFFFFFu, up[q], off), v = __shfl_down_sync(0xFFFFFFFFu, down[q], off);
            if (lane >= off) up[q] += u;
            if (lane < 32 - off) down[q] += v;
          }
        }
        if (!(ok = warp_wait(&bar.gfree[b], ((it >> 1) & 1u) ^ 1u, failed, SPX_DEV_TIMEOUT_PRODUCER))) break;
        DecayTable& t = tables[b];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          t.a[32 * q + lane] = rev ? down[q] : up[q];
          t.cf[32 * q + lane] = ex2(rev ? up[q] : down[q]);
          if (lane == 31) t.total[q] = up[q];
        }
        warp_arrive(&bar.gfull[b], lane);
      }
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 29) {
    // no MMA may still write the accumulators when they are freed
    if (lane == 0) wait_for(&bar.drained, 0u, failed, SPX_DEV_TIMEOUT_MMA);
    __syncwarp();
    tc_fence_after();
    if (lane == 0 && *failed != 0) record_error(status, *failed);
    tmem_dealloc(tmem, kTmCols);
  }
}

// What packed sequences need first.  The last block sorts them by their number of
// chunks, longest first (ties by index): a rank is the count of those that come
// before; and sets the queue's start.  The others zero the rows of the outputs that no
// sequence holds, which nobody else writes: with sound offsets those before the first
// and after the last, else all of them, before the sound sequences write theirs.
__global__ void __launch_bounds__(1024) la_prepare_kernel(const __grid_constant__ LaArgs a, int* __restrict__ order,
                                                          int* __restrict__ queue, int first_state, int first_full) {
  __shared__ int chunks[kOrderMax];
  const int n = a.nseq;
  if (blockIdx.x + 1 < gridDim.x) {
    bool sound = true;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int lo = a.cu[i], hi = a.cu[i + 1];
      sound = sound && lo >= 0 && hi >= lo && hi <= a.total;
    }
    sound = __syncthreads_and(sound) != 0;
    const int64_t lo = sound ? a.cu[0] : a.total, hi = sound ? a.cu[n] : a.total;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x - 1) * blockDim.x;
    auto zero = [&](auto* p, int64_t row) {  // elements of a token's row
      for (int64_t i = at; i < lo * row; i += step) p[i] = {};
      for (int64_t i = hi * row + at; i < a.total * row; i += step) p[i] = {};
    };
    for (int j = 0; j < a.njobs; ++j)  // rows are multiples of 16 bytes
      zero(static_cast<uint4*>(a.job[j].out), static_cast<int64_t>(a.H) * a.job[j].dc / (a.job[j].out_f32 != 0 ? 4 : 8));
    if (a.dg != nullptr) zero(static_cast<uint16_t*>(a.dg), static_cast<int64_t>(a.H) * (a.g_f32 != 0 ? 2 : 1));
    return;
  }
  if (order == nullptr) return;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int lo = a.cu[i], hi = a.cu[i + 1];
    chunks[i] = lo >= 0 && hi >= lo && hi <= a.total ? (hi - lo + kC - 1) / kC : 0;
  }
  if (threadIdx.x == 0) {  // each pass has its own, behind the items that its CTAs start with
    queue[0] = first_state;
    queue[1] = first_full;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int mine = chunks[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += chunks[k] > mine || (chunks[k] == mine && k < i) ? 1 : 0;
    order[rank] = i;
  }
}

// Segment states from zero -> each segment's first state, in place.
__global__ void __launch_bounds__(256) la_chain_kernel(const __grid_constant__ LaChunkArgs args) {
  const int lane_id = blockIdx.x;
  Item w;
  item_of(args, Share{}, lane_id, &w);
  const LaJob& j = args.la.job[w.job];
  const int64_t st0 = (static_cast<int64_t>(w.seq) * args.la.H + w.h) * j.da * j.dc;
  float* seg = args.seg_state + static_cast<int64_t>(lane_id) * args.nseg * 8192;
  const int i = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (i >= j.da * 64) return;
  const int r = i / 64, c = w.slice * 64 + (i & 63);
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    x[e] = j.init != nullptr && c + e < j.dc ? j.init_scale * j.init[st0 + r * j.s_row + (c + e) * j.s_col] : 0.0f;
  float4 next = *reinterpret_cast<const float4*>(seg + i);
  for (int s = 0; s + 1 < args.nseg; ++s) {
    const float4 v = next;
    float4* p = reinterpret_cast<float4*>(seg + static_cast<int64_t>(s) * 8192 + i);
    if (s + 2 < args.nseg) next = p[2048];  // the next segment's, before this one's place is written
    const float d = args.seg_decay[static_cast<int64_t>(lane_id) * args.nseg + s];
    *p = make_float4(x[0], x[1], x[2], x[3]);
    x[0] = fmaf(d, x[0], v.x);
    x[1] = fmaf(d, x[1], v.y);
    x[2] = fmaf(d, x[2], v.z);
    x[3] = fmaf(d, x[3], v.w);
  }
  *reinterpret_cast<float4*>(seg + static_cast<int64_t>(args.nseg - 1) * 8192 + i) = make_float4(x[0], x[1], x[2], x[3]);
}

namespace {

int64_t lanes_of(const LaArgs& a, int (&slices)[3], int64_t (&first)[4]) {
  int64_t n = 0;
  for (int i = 0; i < a.njobs; ++i) {
    slices[i] = (a.job[i].dc + 63) / 64;
    first[i] = n;
    n += static_cast<int64_t>(a.nseq) * a.H * slices[i];
  }
  first[a.njobs] = n;
  return n;
}

int64_t mean_tokens(const LaArgs& a) { return a.cu == nullptr ? a.T : (a.total + a.nseq - 1) / (a.nseq > 0 ? a.nseq : 1); }

// Even shares pay where whole lanes would leave many SMs idle: 192 lanes of 32 chunks on 148 SMs take 143 us, not
// 166 (forward, 64 wide), and 218, not 254 (gradients, 128 wide).  They cost something themselves, as neighbouring
// heads no longer read the same tokens at the same time: 576 lanes, which fill four rounds to 97%, 466, not 420.  So a
// sixth of the rounds has to be idle.
bool even_shares(const LaArgs& a, int64_t lanes, int sms) {
  return a.cu == nullptr && a.T > kC && lanes > sms && (lanes + sms - 1) / sms * sms * 5 > lanes * 6;
}

// Segments per sequence that leave the shortest time, in units of one chunk
// of the full pass (the state-only pass costs about 0.6 of it, the chaining and
// the two extra launches about ten).  One sequence of 65,536 tokens, 6 heads of 128:
// 233 us in 12 segments, 1,363 in one piece.
int segments_for(const LaArgs& a, int64_t lanes, int sms) {
  const int64_t chunks = (mean_tokens(a) + kC - 1) / kC;
  auto waves = [&](int64_t n) { return (n + sms - 1) / sms; };
  int best = 1;
  double least = even_shares(a, lanes, sms) ? static_cast<double>(lanes * chunks) / sms + 1.0
                                            : static_cast<double>(waves(lanes) * chunks);
  for (int s = 2; s <= 64 && s <= chunks; ++s) {
    const int64_t per = (chunks + s - 1) / s;
    const double t = static_cast<double>(waves(lanes * s) * per) + 0.6 * static_cast<double>(waves(lanes * (s - 1)) * per) + 10.0;
    if (t < 0.95 * least) {
      least = t;
      best = s;
    }
  }
  return best;
}

}  // namespace

namespace {
bool ordered(const LaArgs& a) { return a.cu != nullptr && a.nseq > 1 && a.nseq <= kOrderMax; }
size_t order_bytes(const LaArgs& a) { return ordered(a) ? (static_cast<size_t>(a.nseq) + 2 + 3) / 4 * 16 : 0; }
}  // namespace

namespace {
size_t hand_bytes(int sms) { return static_cast<size_t>(sms) * (8192 * sizeof(float) + 4 * sizeof(int)); }
}  // namespace

size_t la_chunk_workspace(const LaArgs& a) {
  int slices[3];
  int64_t first[4];
  const int64_t lanes = lanes_of(a, slices, first);
  const int nseg = segments_for(a, lanes, device_sm_count());
  if (nseg == 1) return order_bytes(a) + (even_shares(a, lanes, device_sm_count()) ? hand_bytes(device_sm_count()) : 0);
  return order_bytes(a) + static_cast<size_t>(lanes) * nseg * (8192 + 1) * sizeof(float);
}

int launch_la_chunk(const LaArgs& a, bool precise, void* workspace, cudaStream_t stream) {
  LaChunkArgs c{};
  int64_t first[4];
  const int64_t lanes = lanes_of(a, c.slices, first);
  if (lanes == 0) return SPX_OK;
  const int sms = device_sm_count();
  c.nseg = segments_for(a, lanes, sms);
  if (lanes * c.nseg > 0x7FFFFFFF - sms) return SPX_ERR_UNSUPPORTED;  // a step past the last item is an int too
  c.la = a;
  int dkb = 1;
  for (int i = 0; i < a.njobs; ++i) {
    const LaJob& j = a.job[i];
    if (j.da > 64) dkb = 2;
    const LaOperand* op[3] = {&j.a, &j.b, &j.c};
    const int width[3] = {j.da, j.da, j.dc};
    for (int x = 0; x < 3; ++x) {
      if (a.total == 0) continue;  // only empty sequences: no tile is loaded
      if (int rc = encode_heads(&c.map[i][x], op[x]->p, width[x], a.H / op[x]->group, a.cu != nullptr ? a.total : a.T,
                                a.cu != nullptr ? 1 : a.nseq, op[x]->sh, op[x]->st, op[x]->sb, kC);
          rc != SPX_OK)
        return rc;
    }
  }
  for (int i = 0; i <= a.njobs; ++i) c.lanes[i] = static_cast<int>(first[i]);
  const bool even = c.nseg == 1 && even_shares(a, lanes, sms);
  if (workspace == nullptr && (c.nseg > 1 || even || ordered(a))) return SPX_ERR_WORKSPACE;
  if (even) {
    c.hand = static_cast<float*>(workspace);
    c.handed = reinterpret_cast<int*>(c.hand + static_cast<int64_t>(sms) * 8192);
    if (cudaMemsetAsync(c.handed, 0, static_cast<size_t>(sms) * 4 * sizeof(int), stream) != cudaSuccess) return SPX_ERR_CUDA;
  }
  if (a.cu != nullptr) {
    int* const order = ordered(a) ? static_cast<int*>(workspace) + 2 : nullptr;
    c.order = order;
    c.queue = order != nullptr ? order - 2 : nullptr;
    const int state_ctas = static_cast<int>(std::min<int64_t>(lanes * (c.nseg - 1), sms));
    const int full_ctas = static_cast<int>(std::min<int64_t>(lanes * c.nseg, sms));
    la_prepare_kernel<<<sms, 1024, 0, stream>>>(a, order, c.queue, state_ctas, full_ctas);
    if (cudaGetLastError() != cudaSuccess) return SPX_ERR_CUDA;
  }
  if (c.nseg > 1) {
    c.seg_state = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + order_bytes(a));
    c.seg_decay = c.seg_state + lanes * c.nseg * 8192;
  }
  auto run = [&](auto kernel, size_t smem) {
    if (int rc = ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel)); rc != SPX_OK) return rc;
    const int64_t items = lanes * c.run_segs;
    kernel<<<static_cast<unsigned>(std::min<int64_t>(items, sms)), kLaThreads, smem, stream>>>(c);
    return cudaGetLastError() == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
  };
  // a last state that the caller keeps is FP32 to the end; one that only feeds BF16 outputs needs two parts
  const int parts = !precise && a.job[0].fin != nullptr ? 3 : 2;
  auto pass = [&]() {
    if (dkb == 1) {
      if (precise) return run(la_chunk_kernel<1, true, 2>, Cfg<1, true, 2>::kBytes);
      return parts == 3 ? run(la_chunk_kernel<1, false, 3>, Cfg<1, false, 3>::kBytes)
                        : run(la_chunk_kernel<1, false, 2>, Cfg<1, false, 2>::kBytes);
    }
    if (precise) return run(la_chunk_kernel<2, true, 2>, Cfg<2, true, 2>::kBytes);
    return parts == 3 ? run(la_chunk_kernel<2, false, 3>, Cfg<2, false, 3>::kBytes)
                      : run(la_chunk_kernel<2, false, 2>, Cfg<2, false, 2>::kBytes);
  };
  if (c.nseg > 1) {
    c.state_only = 1;
    c.run_segs = c.nseg - 1;
    if (int rc = pass(); rc != SPX_OK) return rc;
    la_chain_kernel<<<dim3(static_cast<unsigned>(lanes), 8), 256, 0, stream>>>(c);
    if (cudaGetLastError() != cudaSuccess) return SPX_ERR_CUDA;
  }
  c.state_only = 0;
  c.run_segs = c.nseg;
  if (c.queue != nullptr) ++c.queue;
  return pass();
}

}  // namespace spx
