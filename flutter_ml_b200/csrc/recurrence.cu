// Gated linear recurrence over sequences and its backward pass (an extension beside lib/layertypes/lstmLayer.dart, whose
// gates read the state that they form and so cannot be scanned).
//
//   GATED:  a = sigmoid(f), s = 1 - a        h_t = a_t h_{t-1} + s_t x_t
//   LINEAR: a = f                            h_t = a_t h_{t-1} + x_t
// Backward, from the last step to the first, with c the gradient that flows into a state from the steps behind it
// (c = dh_last at the end):
//   G_t = dy_t + c    c <- a_t G_t           GATED: dx = s G, df = G (h_{t-1} - x) a s      LINEAR: dx = G, df = G h_{t-1}
// dh0 = c at the beginning.  Both directions are first-order recurrences of one state a channel, "state <- a state + b" and
// "state <- a (state + b)", so one scheme serves both, the backward one with time turned round.
//
// Bound: memory, 12 bytes an element forward (f, x in, h out), 24 backward (f, x, h, dy in, df, dx out; LINEAR 20, without x).
//
// Layout: a lane owns one, two or four neighbouring channels (what alignment allows) and SEG consecutive steps of them, loaded
// into registers; LANES lanes make a row, so a warp covers 32 / LANES segments.  Each segment is reduced to its pair (A, B)
// with "state <- A state + B"; the pairs are joined across the lanes of the same channels by shuffles, across the warps of the
// CTA through shared memory, across the CTAs of a cluster (which split the steps when there are too few channels to fill the
// GPU) by asynchronous stores into one another's shared memory; then every lane runs its own steps again from the state it
// now knows, in registers, and writes.  The data crosses the memory bus once.  The order of all joins depends on the sizes, the
// addresses and strides (which decide how wide the loads are) and the device (how many clusters it holds), never on timing: a
// call repeats bit for bit.  Single steps (token by token use) and other very short sequences take one thread a channel.
//
// Measured (us; bytes at the copy's rate in brackets): 128 sequences of 128 x 512 forward 18 (15); 32 ragged ones of 512 x 1024
// 21 forward (14), 37 backward (29); 8 of 2048 x 1024 35 (31) and 69 (61); one of 16384 x 1024, in clusters of four, 44 (31) and
// 80 (61); one of 65521 x 250, in clusters of thirteen, LINEAR, 57 (30) and 95 (50); one of 52433 x 192, in clusters of sixteen,
// 43 (18) and 75 (37).  The first are bound by memory, with about 5 us for the first loads and last stores; the clusters by the
// chain of a round, which 16 warps an SM do not hide.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_CLUSTER = 16;   // above 8 where the device says that such a cluster fits
constexpr int WAIT_CODE = 130;   // fml_device_status: a cluster's pairs did not arrive

struct Params {
  const float *f, *x, *h0, *h, *dy, *dh_last;
  const int* lens;
  float *out, *last;            // forward: h, h_last
  float *df, *dx, *dh0;         // backward
  long long ss_in, ts_in, ss_h, ts_h;
  int n_seq, seq_len, dim, ctiles, accumulate;
  int cluster;                  // CTAs that share the steps of a sequence, 16 at most; above bit 8: the self test's limit
  int* status;
};
// Self test of the wait for a cluster's pairs: CTA 1 sends none, and the others wait for so many microseconds
constexpr int TEST_SHIFT = 8, TEST_CTA = 1;

// a = 1 / (1 + e), s = 1 - a = e a with e = exp(-f): neither is a difference, both keep their relative precision (4 u of the
// exponential, 1.2 |f| u of its argument in base 2, 2 u of the reciprocal, u = 2^-24).  Gates below -80 count as -80: e stays
// finite, a is 2e-35.  The hardware's exponential and reciprocal, six instructions: with expf and a division the forward
// scan issued 40 instructions an element and was bound by them.
template <bool GATED>
__device__ __forceinline__ void gate(float f, float& a, float& s) {
  if (GATED) {
    float g, r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(g) : "f"(f), "f"(-80.f));
    const float e = fml_exp2_ftz(-1.4426950408889634f * g);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    a = r;
    s = e * r;
  } else {
    a = f;
    s = 1.f;
  }
}

// "state <- A state + B".  GATED decays are positive, and a product of them that has underflowed counts as the smallest number
// above zero: an infinite state stays infinite, a finite one is off by 2^-149 of itself.  (A gate that is NaN shows in B.)
// LINEAR ones may be above one: a zero state stays clear of a product of them that has overflowed.
template <bool GATED>
__device__ __forceinline__ float through(float A, float B, float state) {
  if (GATED) return fmaf(fmaxf(A, 0x1p-149f), state, B);
  return state == 0.f ? B : fmaf(A, state, B);
}

// A pair into the shared memory of CTA `rank` of the cluster, counted by that CTA's barrier: neither side needs a fence, which
// would wait for the results of the round before as well (the cluster's own barrier did).
__device__ __forceinline__ void send_pair(const float2* here, const uint64_t* bar, uint32_t rank, float2 v) {
  uint32_t to, sig;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(fml_tc::smem_u32(here)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(sig) : "r"(fml_tc::smem_u32(bar)), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(v.x), "f"(v.y), "r"(sig)
               : "memory");
}

// Waits for a set's bytes, `limit_ns` at most: false when they did not come, or not for another thread of the CTA.  The status
// word then has a code, and the results are whatever they are.
__device__ __forceinline__ bool wait_pairs(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, unsigned long long limit_ns) {
  unsigned long long t0 = 0;
  for (uint32_t spins = 0;; spins++) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if (spins == 0) t0 = fml_tc::globaltimer_ns();
    if ((spins & 0xFF) != 0xFF) continue;
    if (*gave_up) return false;
    if (fml_tc::globaltimer_ns() - t0 > limit_ns) {
      *gave_up = 1;
      atomicCAS(status, 0, WAIT_CODE);
      return false;
    }
  }
}

__device__ __forceinline__ int length_of(const Params& p, int seq) {
  if (!p.lens) return p.seq_len;
  const int n = p.lens[seq];
  if (n < 0 || n > p.seq_len) fml_flag_bad_index(p.status, FML_BAD_INDEX_LENGTH);
  return min(max(n, 0), p.seq_len);
}

template <int VEC>
__device__ __forceinline__ void load_row(float* dst, const float* src) {
  if (VEC == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(src);
  else if (VEC == 2) *reinterpret_cast<float2*>(dst) = *reinterpret_cast<const float2*>(src);
  else *dst = *src;
}
template <int VEC>
__device__ __forceinline__ void store_row(float* dst, const float* src) {
  if (VEC == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(src);
  else if (VEC == 2) *reinterpret_cast<float2*>(dst) = *reinterpret_cast<const float2*>(src);
  else *dst = *src;
}

// CTAs an SM that a scan is compiled for.  Forward 128 registers a thread (128 sequences of 128 x 512: 18.5 us; left alone the
// compiler takes 200 and it is 23).  Backward the next round's four rows need them: 35 us with any number, 47 with 128.  At 128
// registers sixteen of the 120 instances spill 4 to 8 bytes, five forward ones of four channels a lane 12 to 48.
constexpr int min_ctas(int warps, bool team, bool bwd) { return team ? 2 : bwd ? 1 : 16 / warps; }

// What a lane has read of its segment, SEG steps of VEC channels, in scan direction.
template <int VEC, int SEG, bool BWD>
struct Raw {
  float f[SEG][VEC], x[SEG][VEC];
  float dy[BWD ? SEG : 1][VEC], hp[BWD ? SEG : 1][VEC];
};

// Steps behind the end become a gate of one and an input of zero: the state passes through them.
template <int VEC, int SEG, bool GATED, bool BWD>
__device__ __forceinline__ void load_segment(const Params& p, Raw<VEC, SEG, BWD>& r, const float* f, const float* x, const float* h,
                                             const float* dy, const float* first, int p0, int len, bool on) {
  const int t0 = BWD ? len - 1 - p0 : p0;             // the first step's place; backward they descend
  const long long di = BWD ? -p.ts_in : p.ts_in;
  f += t0 * p.ts_in;
  x += t0 * p.ts_in;
  if (BWD) {
    h += (t0 - 1) * p.ts_h;                           // the state before the step
    dy += t0 * p.ts_h;
  }
  // wholly inside (backward: without step 0, whose state before is h0): no tests
  if (on && p0 + SEG + (BWD ? 1 : 0) <= len && (!BWD || p.dy)) {
#pragma unroll
    for (int i = 0; i < SEG; i++) {
      load_row<VEC>(r.f[i], f + i * di);
      if (GATED || !BWD) load_row<VEC>(r.x[i], x + i * di);
      if (BWD) {
        load_row<VEC>(r.hp[i], h - i * p.ts_h);
        load_row<VEC>(r.dy[i], dy - i * p.ts_h);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < SEG; i++) {
    const bool there = on && p0 + i < len;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      r.f[i][v] = GATED ? INFINITY : 1.f;
      r.x[i][v] = 0.f;
      if (BWD) {
        r.dy[i][v] = 0.f;
        r.hp[i][v] = first[v];
      }
    }
    if (!there) continue;
    load_row<VEC>(r.f[i], f + i * di);
    if (GATED || !BWD) load_row<VEC>(r.x[i], x + i * di);
    if (BWD) {
      if (p.dy) load_row<VEC>(r.dy[i], dy - i * p.ts_h);
      if (p0 + i < len - 1) load_row<VEC>(r.hp[i], h - i * p.ts_h);
    }
  }
}

template <int WARPS, int LANES, int VEC, int SEG, bool GATED, bool BWD, bool AHEAD, bool TEAM>
__global__ void __launch_bounds__(32 * WARPS, min_ctas(WARPS, TEAM, BWD)) scan_kernel(const Params p) {
  constexpr int SUBS = 32 / LANES;                    // segments of a warp that share their channels
  constexpr int CW = LANES * VEC;                     // channels of a CTA
  constexpr int TILE = WARPS * SUBS * SEG;            // steps of a CTA's round
  __shared__ __align__(16) float wtot[2][WARPS][2][CW];   // the warps' pairs; two sets, so one barrier a round is enough
  // The CTAs' pairs, written by their owners into every CTA.  Two sets: a CTA sends round r + 2's pairs when it has every
  // CTA's of round r + 1, and those were sent when their owners had read round r's.
  __shared__ __align__(16) float2 ctot[TEAM ? 2 : 1][TEAM ? MAX_CLUSTER : 1][CW];
  __shared__ uint64_t arrived[2];                     // counts the bytes of a set
  __shared__ int gave_up;                             // a thread's wait has run out
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ch = (lane % LANES) * VEC, sub = lane / LANES;
  const int cs = TEAM ? p.cluster & ((1 << TEST_SHIFT) - 1) : 1, rank = TEAM ? (int)fml_tc::cluster_ctarank() : 0;
  const int unit = blockIdx.x / cs;
  const int seq = unit / p.ctiles, c = (unit - seq * p.ctiles) * CW + ch;
  const bool on = c < p.dim;
  fml_chain_next();
  fml_chain_wait();
  const int len = length_of(p, seq);
  const float* f = p.f + seq * p.ss_in + c;
  const float* x = p.x + seq * p.ss_in + c;
  const float* h = p.h + seq * p.ss_h + c;
  const float* dy = p.dy + seq * p.ss_h + c;
  const long long edge = (long long)seq * p.dim + c;  // of h0, h_last and their gradients
  float state[VEC], first[VEC];                       // first: h before step 0
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    first[v] = on && p.h0 ? p.h0[edge + v] : 0.f;
    state[v] = !BWD ? first[v] : on && p.dh_last ? p.dh_last[edge + v] : 0.f;
  }
  Raw<VEC, SEG, BWD> raw;
  if (TEAM) {
    if (threadIdx.x == 0) {
      gave_up = 0;
      for (int i = 0; i < 2; i++) fml_tc::mbar_init(fml_tc::smem_u32(&arrived[i]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fml_tc::cluster_sync_all();                       // every CTA's barriers are there, and every CTA has read h0 and dh_last
  }
  int p0 = ((rank * WARPS + warp) * SUBS + sub) * SEG;   // first step of the segment, counted in scan direction
  if (AHEAD) load_segment<VEC, SEG, GATED, BWD>(p, raw, f, x, h, dy, first, p0, len, on);
  uint32_t phase = 0;
  bool arriving = true;                               // a thread that has waited in vain waits, and arms a barrier, no more
  for (int base = 0, buf = 0; base < len; base += TILE * cs, p0 += TILE * cs, buf ^= 1) {
    if (!AHEAD) load_segment<VEC, SEG, GATED, BWD>(p, raw, f, x, h, dy, first, p0, len, on);
    // forward: decay and input; backward: decay, incoming gradient, and what G is multiplied by for dx and df
    float a[SEG][VEC], b[SEG][VEC], s[BWD && GATED ? SEG : 1][VEC], w[BWD ? SEG : 1][VEC];
    float A[VEC], B[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      A[v] = 1.f;
      B[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < SEG; i++)
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        float s1;
        gate<GATED>(raw.f[i][v], a[i][v], s1);
        if (!BWD) {
          b[i][v] = GATED ? s1 * raw.x[i][v] : raw.x[i][v];
          B[v] = fmaf(a[i][v], B[v], b[i][v]);
        } else {
          b[i][v] = raw.dy[i][v];
          B[v] = a[i][v] * (B[v] + b[i][v]);
          if (GATED) s[i][v] = s1;
          w[i][v] = GATED ? (raw.hp[i][v] - raw.x[i][v]) * (a[i][v] * s1) : raw.hp[i][v];
        }
        A[v] *= a[i][v];
      }
    if (AHEAD) load_segment<VEC, SEG, GATED, BWD>(p, raw, f, x, h, dy, first, p0 + TILE * cs, len, on);
    // over the segments of the warp: the pair of everything before this one, and the warp's
    float Ae[VEC], Be[VEC];
    if (SUBS > 1) {
#pragma unroll
      for (int o = 1; o < SUBS; o <<= 1)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          const float Ap = __shfl_up_sync(0xffffffffu, A[v], o * LANES), Bp = __shfl_up_sync(0xffffffffu, B[v], o * LANES);
          if (sub >= o) {
            B[v] = through<GATED>(A[v], B[v], Bp);
            A[v] *= Ap;
          }
        }
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        Ae[v] = __shfl_up_sync(0xffffffffu, A[v], LANES);
        Be[v] = __shfl_up_sync(0xffffffffu, B[v], LANES);
      }
    }
    if (sub == SUBS - 1) {
      store_row<VEC>(&wtot[buf][warp][0][ch], A);
      store_row<VEC>(&wtot[buf][warp][1][ch], B);
    }
    __syncthreads();
    float run[VEC];                                   // the state before the lane's steps; `state`: after the round
    if (TEAM) {
      const uint32_t bar = fml_tc::smem_u32(&arrived[buf]);
      if (threadIdx.x == 0 && arriving) fml_tc::mbar_expect_tx(bar, (uint32_t)(cs * CW * sizeof(float2)));
      const unsigned test_us = (unsigned)p.cluster >> TEST_SHIFT;
      for (int i = !arriving || (test_us && rank == TEST_CTA) ? cs * CW : (int)threadIdx.x; i < cs * CW; i += 32 * WARPS) {
        const int r = i / CW, k = i - r * CW;
        float At = 1.f, Bt = 0.f;
#pragma unroll
        for (int q = 0; q < WARPS; q++) {
          const float Aq = wtot[buf][q][0][k];
          Bt = through<GATED>(Aq, wtot[buf][q][1][k], Bt);
          At *= Aq;
        }
        send_pair(&ctot[buf][rank][k], &arrived[buf], r, make_float2(At, Bt));
      }
      if (arriving) arriving = wait_pairs(bar, phase, &gave_up, p.status, test_us ? test_us * 1000ull : fml_tc::WAIT_LIMIT_NS);
      phase ^= buf;                                   // each set is used every other round
      for (int r = 0; r < cs; r++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          const float2 pr = ctot[buf][r][ch + v];
          if (r == rank) run[v] = state[v];
          state[v] = through<GATED>(pr.x, pr.y, state[v]);
        }
#pragma unroll
      for (int q = 0; q < WARPS - 1; q++)
        if (q < warp) {
          float Aq[VEC], Bq[VEC];
          load_row<VEC>(Aq, &wtot[buf][q][0][ch]);
          load_row<VEC>(Bq, &wtot[buf][q][1][ch]);
#pragma unroll
          for (int v = 0; v < VEC; v++) run[v] = through<GATED>(Aq[v], Bq[v], run[v]);
        }
    } else {
#pragma unroll
      for (int q = 0; q < WARPS; q++) {
        float Aq[VEC], Bq[VEC];
        load_row<VEC>(Aq, &wtot[buf][q][0][ch]);
        load_row<VEC>(Bq, &wtot[buf][q][1][ch]);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          if (q == warp) run[v] = state[v];
          state[v] = through<GATED>(Aq[v], Bq[v], state[v]);
        }
      }
    }
    if (SUBS > 1 && sub > 0) {
#pragma unroll
      for (int v = 0; v < VEC; v++) run[v] = through<GATED>(Ae[v], Be[v], run[v]);
    }
#pragma unroll
    for (int i = 0; i < SEG; i++)
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        if (!BWD) {
          run[v] = b[i][v] = fmaf(a[i][v], run[v], b[i][v]);
        } else {
          const float G = b[i][v] + run[v];
          run[v] = a[i][v] * G;
          b[i][v] = GATED ? s[i][v] * G : G;          // dx
          w[i][v] *= G;                               // df
        }
      }
    if (!on || p0 >= len) continue;
    const int there = len - p0;                       // steps of the segment that exist, or more
    if (!BWD) {
      float* to = p.out + seq * p.ss_h + p0 * p.ts_h + c;
#pragma unroll
      for (int i = 0; i < SEG; i++)
        if (i < there) store_row<VEC>(to + i * p.ts_h, b[i]);
    } else {
      const long long at = seq * p.ss_in + (len - 1 - p0) * p.ts_in + c;
      float *tx = p.dx + at, *tf = p.df + at;
#pragma unroll
      for (int i = 0; i < SEG; i++) {
        if (i >= there) break;
        if (p.accumulate) {
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            b[i][v] = __fadd_rn(tx[v - i * p.ts_in], b[i][v]);
            w[i][v] = __fadd_rn(tf[v - i * p.ts_in], w[i][v]);
          }
        }
        store_row<VEC>(tx - i * p.ts_in, b[i]);
        store_row<VEC>(tf - i * p.ts_in, w[i]);
      }
    }
  }
  if (TEAM) fml_tc::cluster_sync_all();               // nobody leaves while something may still arrive
  float* last = BWD ? p.dh0 : p.last;
  if (last && on && rank == 0 && warp == 0 && sub == 0) {
#pragma unroll
    for (int v = 0; v < VEC; v++) last[edge + v] = BWD && p.accumulate ? __fadd_rn(last[edge + v], state[v]) : state[v];
  }
}

// One thread a channel: single tokens and very short sequences.
template <bool GATED, bool BWD>
__global__ void __launch_bounds__(THREADS) step_kernel(const Params p) {
  const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
  fml_chain_next();
  fml_chain_wait();
  if (i >= (long long)p.n_seq * p.dim) return;
  const int seq = (int)(i / p.dim), c = (int)(i - (long long)seq * p.dim);
  const int len = length_of(p, seq);
  const float first = p.h0 ? p.h0[i] : 0.f;
  float state = BWD ? (p.dh_last ? p.dh_last[i] : 0.f) : first;
  for (int q = 0; q < len; q++) {
    const int t = BWD ? len - 1 - q : q;
    const long long in = seq * p.ss_in + t * p.ts_in + c, at = seq * p.ss_h + t * p.ts_h + c;
    float a, s;
    gate<GATED>(p.f[in], a, s);
    if (!BWD) {
      state = fmaf(a, state, s * p.x[in]);
      p.out[at] = state;
    } else {
      const float G = (p.dy ? p.dy[at] : 0.f) + state, hp = t > 0 ? p.h[at - p.ts_h] : first;
      state = a * G;
      const float gx = GATED ? s * G : G, gf = GATED ? G * (hp - p.x[in]) * (a * s) : G * hp;
      p.dx[in] = p.accumulate ? __fadd_rn(p.dx[in], gx) : gx;
      p.df[in] = p.accumulate ? __fadd_rn(p.df[in], gf) : gf;
    }
  }
  float* last = BWD ? p.dh0 : p.last;
  if (last) last[i] = BWD && p.accumulate ? __fadd_rn(last[i], state) : state;
}

// ---- host side: what a call may hand over
struct Box {                  // n_seq x seq_len rows of dim elements at two strides
  const float* p;
  long long ss, ts;
};
// every element at an address of its own
bool distinct(const Params& p, long long ss, long long ts) {
  if (p.n_seq == 1 && p.seq_len == 1) return true;
  if (p.n_seq == 1) return ts >= p.dim;
  if (p.seq_len == 1) return ss >= p.dim;
  const long long lo = std::min(ss, ts), hi = std::max(ss, ts), n_lo = ss < ts ? p.n_seq : p.seq_len;
  return lo >= p.dim && hi >= lo * (n_lo - 1) + p.dim;
}
long long extent(const Params& p, const Box& b) { return (p.n_seq - 1) * b.ss + (p.seq_len - 1) * b.ts + p.dim; }
bool overlap(const Params& p, const Box& a, const Box& b) {
  if (!a.p || !b.p) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + 4 * extent(p, a) <= pb || pb + 4 * extent(p, b) <= pa) return false;
  if (a.ss != b.ss || a.ts != b.ts || p.n_seq == 1 || p.seq_len == 1) {
    // rows of one stride (the halves of a fused projection, one sequence or one step): column by column
    const long long st = p.n_seq == 1 ? a.ts : a.ss, st2 = p.n_seq == 1 ? b.ts : b.ss;
    if ((p.n_seq > 1 && p.seq_len > 1) || st != st2 || st < 1) return true;
    const long long off = ((long long)(pb - pa) / 4 % st + st) % st;
    return off < p.dim || off + p.dim > st;
  }
  // the same strides: some difference of rows that meets the difference of the addresses to less than a row
  const long long diff = (long long)(pb - pa) / 4;
  const bool few_seqs = p.n_seq <= p.seq_len;
  const long long n = few_seqs ? p.n_seq : p.seq_len, m = few_seqs ? p.seq_len : p.n_seq;
  const long long sn = few_seqs ? a.ss : a.ts, sm = few_seqs ? a.ts : a.ss;
  for (long long i = 1 - n; i < n; i++) {
    const long long rest = diff - i * sn;
    long long j = sm > 0 ? rest / sm : 0;
    for (long long k = j - 1; k <= j + 1; k++)
      if (k > -m && k < m && std::llabs(rest - k * sm) < p.dim) return true;
  }
  return false;
}
bool ranges_meet(const float* a, long long na, const float* b, long long nb) {
  if (!a || !b) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return pa < pb + 4 * nb && pb < pa + 4 * na;
}

int32_t check(fml_ctx* ctx, const Params& p, int32_t form) {
  FML_REQUIRE(ctx, form == FML_RECURRENCE_GATED || form == FML_RECURRENCE_LINEAR, "fml_gated_recurrence: unknown form");
  FML_REQUIRE(ctx, p.n_seq >= 0 && p.seq_len >= 0 && p.seq_len <= (1 << 30) && p.dim >= 1, "fml_gated_recurrence: bad sizes");
  FML_REQUIRE(ctx, (long long)p.n_seq * ((p.dim + 7) / 8) <= (1ll << 27), "fml_gated_recurrence: too many sequences and channels for one call");
  FML_REQUIRE(ctx, p.ss_in >= 0 && p.ts_in >= 0 && p.ss_h >= 0 && p.ts_h >= 0, "fml_gated_recurrence: strides must not be negative");
  const auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  const uintptr_t all = at(p.f) | at(p.x) | at(p.h0) | at(p.lens) | at(p.out) | at(p.last) | at(p.h) | at(p.dy) | at(p.dh_last) | at(p.df) | at(p.dx) | at(p.dh0);
  FML_REQUIRE(ctx, (all & 3) == 0, "fml_gated_recurrence: misaligned buffer");
  return FML_OK;
}

template <int WARPS, int LANES, int VEC, int SEG, bool GATED, bool BWD, bool AHEAD, bool TEAM>
int32_t launch_scan(fml_ctx* ctx, Params& p, int cluster) {
  p.ctiles = (p.dim + LANES * VEC - 1) / (LANES * VEC);
  p.cluster = cluster | (p.cluster & ~((1 << TEST_SHIFT) - 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.n_seq * p.ctiles * cluster));
  cfg.blockDim = dim3(32 * WARPS);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  if (TEAM) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  } else {   // set up while the kernel before drains; with clusters that was slower (203 us against 165 on the long sequence)
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FML_CUDA(ctx, cudaLaunchKernelEx(&cfg, scan_kernel<WARPS, LANES, VEC, SEG, GATED, BWD, AHEAD, TEAM>, (const Params)p));
  return FML_OK;
}

// elements that one load may take: rows, row strides and addresses all allow it
int vector_width(const Params& p) {
  uintptr_t all = 0;
  for (const float* q : {p.f, p.x, p.h, p.dy, (const float*)p.out, (const float*)p.df, (const float*)p.dx}) all |= reinterpret_cast<uintptr_t>(q);
  const long long n = p.dim | p.ss_in | p.ts_in | p.ss_h | p.ts_h;
  return (all & 15) == 0 && n % 4 == 0 ? 4 : (all & 7) == 0 && n % 2 == 0 ? 2 : 1;
}

// How many clusters of this size the device holds at once (none where it cannot form one); asked for once a device and size.
template <int LANES, int VEC, int SEG, bool GATED, bool BWD>
int32_t clusters_at_once(fml_ctx* ctx, int size, long long* out) {
  static std::atomic<int> known[FML_MAX_DEVICES][MAX_CLUSTER + 1];   // one more than the answer
  const bool slot = ctx->device >= 0 && ctx->device < FML_MAX_DEVICES;
  int n = slot ? known[ctx->device][size].load(std::memory_order_acquire) : 0;
  if (n == 0) {
    auto* kernel = scan_kernel<8, LANES, VEC, SEG, GATED, BWD, false, true>;
    FML_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(256);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)size, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess) {
      fit = 0;
      (void)cudaGetLastError();
    }
    n = std::max(fit, 0) + 1;
    if (slot) known[ctx->device][size].store(n, std::memory_order_release);
  }
  *out = n - 1;
  return FML_OK;
}

// Few channels: eight warps, rows of LANES, long segments forward, and a cluster along the steps: two CTAs an SM, or where eight
// CTAs a cluster do not give one an SM, up to sixteen and one and a half; no more of them than the same number of rounds needs,
// and only as many as let all clusters run at once.
// One sequence of 16384 x 1024: 44 and 80 us with four, of 52433 x 192: 43 and 75 with sixteen (56 and 105 with eight), of
// 18285 x 256: 21 and 37 with twelve (27 and 44).  14 of 2899 x 112, 98 units of which 93 clusters of three run at once: 19 and
// 33 with two, 23 and 37 with three.
template <int LANES, int VEC, bool GATED, bool BWD>
int32_t launch_team(fml_ctx* ctx, Params& p) {
  constexpr int SEG = (BWD ? 16 : 32) / VEC, TILE = 8 * (32 / LANES) * SEG;
  const long long units = (long long)p.n_seq * ((p.dim + LANES * VEC - 1) / (LANES * VEC)), sms = ctx->sm_count;
  long long cluster = units * 8 < sms ? std::min<long long>(MAX_CLUSTER, 3 * sms / 2 / units) : std::min(8ll, 2 * sms / units);
  for (; cluster > 1; cluster--) {
    const long long rounds = (p.seq_len + TILE * cluster - 1) / (TILE * cluster);
    cluster = (p.seq_len + TILE * rounds - 1) / (TILE * rounds);
    if (cluster == 1) break;
    long long fit;
    const int32_t rc = clusters_at_once<LANES, VEC, SEG, GATED, BWD>(ctx, (int)cluster, &fit);
    if (rc) return rc;
    if (units <= fit) break;
  }
  if (cluster > 1) return launch_scan<8, LANES, VEC, SEG, GATED, BWD, false, true>(ctx, p, (int)cluster);
  return launch_scan<8, LANES, VEC, SEG, GATED, BWD, false, false>(ctx, p, 1);
}

template <int VEC, bool GATED, bool BWD>
int32_t launch_lanes(fml_ctx* ctx, Params& p) {
  constexpr int SEG = 16 / VEC;
  auto units = [&](int lanes) { return (long long)p.n_seq * ((p.dim + lanes * VEC - 1) / (lanes * VEC)); };
  const int sms = ctx->sm_count;
  // Channels enough: each CTA goes over all steps of its channels, the next round's rows in registers meanwhile.  Rows as wide as
  // leave three to four CTAs of four warps an SM, at least 32 channels of them, else eight warps.  Measured (us, forward and
  // backward): 128 sequences of 128 x 512, 32 lanes of four: 18 and 35.  32 of 512 x 1024: 34 and 65 with 16 lanes, 35 and 68
  // with 8; ragged 25 and 37, 21 and 37 (the one ragged size that was compared).  8 of 2048 x 1024, eight warps of 8 lanes: 36 and 69, four warps 49 and 68.  Two
  // channels a lane, 8 of 2048 x 1022: eight warps of 16 lanes 37 and 74, of 8 40 and 84.  One, 32 of 512 x 1001: 32 lanes 39
  // and 84, 8 46 and 108; 100 of 300 x 77: 16 lanes 10 and 20, 8 13 and 29.
#define FML_SCAN(warps, lanes) return launch_scan<warps, lanes, VEC, SEG, GATED, BWD, true, false>(ctx, p, 1)
  if (VEC == 4) {
    if (units(32) >= 3 * sms) FML_SCAN(4, 32);
    if (units(16) >= (p.lens ? 4 : 3) * sms) FML_SCAN(4, 16);
    if (units(8) >= 4 * sms) FML_SCAN(4, 8);
  } else {
    if (units(32) >= 4 * sms) FML_SCAN(4, 32);
    if (units(16) >= (VEC == 2 ? 4 : 3) * sms) FML_SCAN(4, 16);
    if (2 * units(16) >= (VEC == 2 ? 3 : 2) * sms) FML_SCAN(8, 16);
  }
  if constexpr (BWD) {
    // A CTA of eight warps fills an SM: few more of them than SMs, and a second wave would go nearly empty.  6 of 3000 x 800
    // 78 us for 88, 8 of 2500 x 800 the other way 86 and 75; single floats, 10 of 3000 x 197: 39 for 44.
    if (units(8) >= sms && 4 * units(8) < (VEC == 1 ? 7 : 5) * sms) return launch_team<16, VEC, GATED, BWD>(ctx, p);
  }
  if (units(8) >= sms) FML_SCAN(8, 8);
#undef FML_SCAN
  if constexpr (VEC == 4) {
    if (units(4) * MAX_CLUSTER < sms) return launch_team<2, VEC, GATED, BWD>(ctx, p);   // rows of one sector
    // rows of two sectors, as long as two CTAs share a sequence (one of 9000 x 2600 with four lanes 73 and 215 us, with eight
    // 62 and 114; of 6618 x 1472 the other way 35 and 59, 31 and 49)
    if (units(4) <= sms) return launch_team<4, VEC, GATED, BWD>(ctx, p);
  }
  if constexpr (VEC == 2) {   // one of 60000 x 50: 25 and 41 us with four lanes, 33 and 60 with eight; of 52433 x 190 49 and 82, 43 and 70
    if (units(4) * MAX_CLUSTER < 2 * sms) return launch_team<4, VEC, GATED, BWD>(ctx, p);   // rows of one sector
  }
  return launch_team<8, VEC, GATED, BWD>(ctx, p);
}

template <bool GATED, bool BWD>
int32_t launch(fml_ctx* ctx, Params& p) {
  if (p.n_seq == 0) return FML_OK;
  if (p.seq_len <= 4) {
    const unsigned blocks = (unsigned)(((long long)p.n_seq * p.dim + THREADS - 1) / THREADS);
    const cudaError_t e = fml_launch_chained(step_kernel<GATED, BWD>, dim3(blocks), dim3(THREADS), 0, ctx->stream, p);
    return e == cudaSuccess ? FML_OK : fml_fail(ctx, FML_ERR_CUDA, std::string("step_kernel: ") + cudaGetErrorString(e));
  }
  const int vec = vector_width(p);
  if (vec == 4) return launch_lanes<4, GATED, BWD>(ctx, p);
  if (vec == 2) return launch_lanes<2, GATED, BWD>(ctx, p);
  return launch_lanes<1, GATED, BWD>(ctx, p);
}

}  // namespace

extern "C" {

int32_t fml_gated_recurrence_fwd(fml_ctx* ctx, int32_t form, int32_t n_seq, int32_t seq_len, int32_t dim, const float* f, const float* x,
                                 int64_t seq_stride_in, int64_t step_stride_in, const float* h0, const int32_t* lens, float* h,
                                 int64_t seq_stride_h, int64_t step_stride_h, float* h_last) {
  FML_REQUIRE(ctx, ctx, "fml_gated_recurrence_fwd: no context");
  FML_ENTER(ctx);
  Params p = {};
  p.f = f; p.x = x; p.h0 = h0; p.lens = lens; p.out = h; p.last = h_last;
  p.ss_in = seq_stride_in; p.ts_in = step_stride_in; p.ss_h = seq_stride_h; p.ts_h = step_stride_h;
  p.n_seq = n_seq; p.seq_len = seq_len; p.dim = dim; p.status = ctx->d_status;
  const int32_t rc = check(ctx, p, form);
  if (rc || n_seq == 0) return rc;
  FML_REQUIRE(ctx, seq_len == 0 || (f && x && h), "fml_gated_recurrence_fwd: missing buffer");
  const long long ends = (long long)n_seq * dim;
  if (seq_len > 0) {
    FML_REQUIRE(ctx, distinct(p, p.ss_h, p.ts_h), "fml_gated_recurrence_fwd: rows of h overlap");
    const Box out = {h, p.ss_h, p.ts_h};
    for (const float* in : {f, x})
      FML_REQUIRE(ctx, !overlap(p, out, {in, p.ss_in, p.ts_in}), "fml_gated_recurrence_fwd: h overlaps an input");
    FML_REQUIRE(ctx, !ranges_meet(h, extent(p, out), h0, ends) && !ranges_meet(h, extent(p, out), h_last, ends),
                "fml_gated_recurrence_fwd: h overlaps an end state");
    for (const float* in : {f, x})
      FML_REQUIRE(ctx, !ranges_meet(in, extent(p, {in, p.ss_in, p.ts_in}), h_last, ends), "fml_gated_recurrence_fwd: h_last overlaps an input");
  }
  FML_REQUIRE(ctx, h0 == h_last || !ranges_meet(h0, ends, h_last, ends), "fml_gated_recurrence_fwd: h_last overlaps h0 without being it");
  return form == FML_RECURRENCE_GATED ? launch<true, false>(ctx, p) : launch<false, false>(ctx, p);
}

int32_t fml_gated_recurrence_bwd(fml_ctx* ctx, int32_t form, int32_t n_seq, int32_t seq_len, int32_t dim, const float* f, const float* x,
                                 int64_t seq_stride_in, int64_t step_stride_in, const float* h0, const int32_t* lens, const float* h,
                                 const float* dy, int64_t seq_stride_h, int64_t step_stride_h, const float* dh_last, float* df,
                                 float* dx, float* dh0, int32_t accumulate) {
  FML_REQUIRE(ctx, ctx, "fml_gated_recurrence_bwd: no context");
  FML_ENTER(ctx);
  Params p = {};
  p.f = f; p.x = x; p.h0 = h0; p.lens = lens; p.h = h; p.dy = dy; p.dh_last = dh_last; p.df = df; p.dx = dx; p.dh0 = dh0;
  p.ss_in = seq_stride_in; p.ts_in = step_stride_in; p.ss_h = seq_stride_h; p.ts_h = step_stride_h;
  p.n_seq = n_seq; p.seq_len = seq_len; p.dim = dim; p.accumulate = accumulate != 0; p.status = ctx->d_status;
  const int32_t rc = check(ctx, p, form);
  if (rc || n_seq == 0) return rc;
  FML_REQUIRE(ctx, seq_len == 0 || (f && x && h && df && dx), "fml_gated_recurrence_bwd: missing buffer");
  const long long ends = (long long)n_seq * dim;
  if (seq_len > 0) {
    FML_REQUIRE(ctx, distinct(p, p.ss_in, p.ts_in), "fml_gated_recurrence_bwd: rows of df and dx overlap");
    const Box bf = {df, p.ss_in, p.ts_in}, bx = {dx, p.ss_in, p.ts_in};
    FML_REQUIRE(ctx, !overlap(p, bf, bx), "fml_gated_recurrence_bwd: df and dx overlap");
    for (const Box& out : {bf, bx}) {
      for (const Box& in : {Box{f, p.ss_in, p.ts_in}, Box{x, p.ss_in, p.ts_in}, Box{h, p.ss_h, p.ts_h}, Box{dy, p.ss_h, p.ts_h}})
        FML_REQUIRE(ctx, !overlap(p, out, in), "fml_gated_recurrence_bwd: an output overlaps an input");
      for (const float* e : {h0, dh_last, (const float*)dh0})
        FML_REQUIRE(ctx, !ranges_meet(out.p, extent(p, out), e, ends), "fml_gated_recurrence_bwd: an output overlaps an end state");
    }
    for (const Box& in : {Box{f, p.ss_in, p.ts_in}, Box{x, p.ss_in, p.ts_in}, Box{h, p.ss_h, p.ts_h}, Box{dy, p.ss_h, p.ts_h}})
      FML_REQUIRE(ctx, !in.p || !ranges_meet(in.p, extent(p, in), dh0, ends), "fml_gated_recurrence_bwd: dh0 overlaps an input");
  }
  FML_REQUIRE(ctx, (dh_last == dh0 && !accumulate) || !ranges_meet(dh_last, ends, dh0, ends), "fml_gated_recurrence_bwd: dh0 overlaps dh_last");
  FML_REQUIRE(ctx, !ranges_meet(h0, ends, dh0, ends), "fml_gated_recurrence_bwd: dh0 overlaps h0");
  return form == FML_RECURRENCE_GATED ? launch<true, true>(ctx, p) : launch<false, true>(ctx, p);
}

int32_t fml_selftest_cluster_wait(fml_ctx* ctx, int32_t backward, int32_t limit_us) {
  FML_REQUIRE(ctx, ctx && limit_us > 0 && limit_us <= 1000000, "fml_selftest_cluster_wait: the limit must be 1 .. 1000000 us");
  FML_ENTER(ctx);
  FML_REQUIRE(ctx, !ctx->capturing, "fml_selftest_cluster_wait: not while a graph is being recorded");
  Params p = {};
  p.n_seq = 1; p.seq_len = 40000; p.dim = 8; p.status = ctx->d_status;   // three rounds of a cluster
  p.ss_in = p.ss_h = (long long)p.seq_len * p.dim; p.ts_in = p.ts_h = p.dim;
  p.cluster = limit_us << TEST_SHIFT;
  const long long n = p.ss_in;
  float* b = nullptr;
  int32_t rc = fml_alloc(ctx, 6 * n, &b);
  if (rc) return rc;
  rc = fml_zero(ctx, b, 6 * n);
  p.f = b; p.x = b + n; p.h = p.dy = b + 2 * n; p.out = b + 3 * n; p.df = b + 4 * n; p.dx = b + 5 * n;
  if (!rc) rc = backward ? launch<true, true>(ctx, p) : launch<true, false>(ctx, p);
  if (!rc && (p.cluster & ((1 << TEST_SHIFT) - 1)) < 2) rc = fml_fail(ctx, FML_ERR_INVALID, "fml_selftest_cluster_wait: the device forms no clusters");
  const int32_t freed = fml_free(ctx, b);
  return rc ? rc : freed;
}

}  // extern "C"
