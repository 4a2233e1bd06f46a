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
// Bound: memory, 12 bytes an element forward (f, x in, h out), 24 backward (f, x, h, dy in, df, dx out).
//
// Layout: a lane owns one channel and SEG consecutive steps of it, loaded into registers, so a warp's load covers CW
// neighbouring channels of 32 / CW steps.  Each segment is reduced to its pair (A, B) with "state <- A state + B"; the pairs
// are joined across the lanes that share a channel by shuffles, across the warps of the CTA through shared memory, across
// the CTAs of a cluster (which split the time axis when there are too few channels to fill the GPU) through distributed
// shared memory; then every lane runs its own steps again from the state it now knows, in registers, and writes.  The data
// crosses the memory bus once.  The order of all joins depends on the sizes alone: results repeat bit for bit.
// A single step (token by token use) and other very short sequences take one thread a channel.
#include <math.h>

#include <algorithm>
#include <cstdlib>

#include "common.cuh"

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int MAX_CLUSTER = 8;

struct Params {
  const float *f, *x, *h0, *h, *dy, *dh_last;
  const int* lens;
  float *out, *last;            // forward: h, h_last
  float *df, *dx, *dh0;         // backward
  long long ss_in, ts_in, ss_h, ts_h;
  int n_seq, seq_len, dim, ctiles, cluster, accumulate;
  int* status;
};

// a and s = 1 - a without the difference: whichever is small comes from the exponential itself
template <bool GATED>
__device__ __forceinline__ void gate(float f, float& a, float& s) {
  if (GATED) {
    const float e = expf(-fabsf(f)), big = __fdividef(1.f, 1.f + e), small = e * big;
    a = f >= 0.f ? big : small;
    s = f >= 0.f ? small : big;
  } else {
    a = f;
    s = 1.f;
  }
}

// "state <- A state + B"; a zero state stays clear of a product of decays that has overflowed
__device__ __forceinline__ float through(float A, float B, float state) { return state == 0.f ? B : fmaf(A, state, B); }

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_remote(const float2* here, uint32_t rank, float2 v) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(here);
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
}

__device__ __forceinline__ int length_of(const Params& p, int seq) {
  if (!p.lens) return p.seq_len;
  const int n = p.lens[seq];
  if (n < 0 || n > p.seq_len) fml_flag_bad_index(p.status, FML_BAD_INDEX_LENGTH);
  return min(max(n, 0), p.seq_len);
}

template <int CW, int SEG, bool GATED, bool BWD>
__global__ void __launch_bounds__(THREADS) scan_kernel(const Params p) {
  constexpr int SUBS = 32 / CW;                       // lanes that share a channel
  constexpr int TILE = WARPS * SUBS * SEG;            // steps of a CTA's round
  __shared__ float2 wtot[2][WARPS][CW];               // the warps' pairs; two sets, so one barrier a round is enough
  __shared__ float2 ctot[2][MAX_CLUSTER][CW];         // the CTAs' pairs, written by their owners into every CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ch = lane % CW, sub = lane / CW;
  const int cs = p.cluster;
  const int rank = cs > 1 ? (int)cluster_rank() : 0;
  const int unit = blockIdx.x / cs;
  const int seq = unit / p.ctiles, c = (unit - seq * p.ctiles) * CW + ch;
  const bool on = c < p.dim;
  const int len = length_of(p, seq);
  const float* f = p.f + seq * p.ss_in + c;
  const float* x = p.x + seq * p.ss_in + c;
  const long long edge = (long long)seq * p.dim + c;  // of h0, h_last and their gradients
  float state = 0.f;
  const float first = on && p.h0 ? p.h0[edge] : 0.f;  // h before step 0
  if (!BWD) state = first;
  else if (on && p.dh_last) state = p.dh_last[edge];
  if (cs > 1) cluster_sync();                         // every CTA is there before the first remote store
  int buf = 0;
  for (int base = 0; base < len; base += TILE * cs, buf ^= 1) {
    const int p0 = base + ((rank * WARPS + warp) * SUBS + sub) * SEG;   // first step of the segment, counted in scan direction
    float a[SEG], s[SEG], xv[SEG], b[SEG], hp[SEG];   // what a form or direction does not use, the compiler drops
#pragma unroll
    for (int i = 0; i < SEG; i++) {
      const int q = p0 + i;
      const bool there = on && q < len;
      const int t = BWD ? len - 1 - q : q;
      a[i] = there ? f[t * p.ts_in] : 0.f;
      xv[i] = there && (GATED || !BWD) ? x[t * p.ts_in] : 0.f;
      if (BWD) {
        b[i] = there && p.dy ? p.dy[seq * p.ss_h + t * p.ts_h + c] : 0.f;
        hp[i] = there && t > 0 ? p.h[seq * p.ss_h + (t - 1) * p.ts_h + c] : first;
      }
    }
    float A = 1.f, B = 0.f;
#pragma unroll
    for (int i = 0; i < SEG; i++) {
      gate<GATED>(a[i], a[i], s[i]);
      if (!(p0 + i < len)) a[i] = 1.f;                // behind the end: the state passes through (b and xv are 0)
      if (!BWD) b[i] = s[i] * xv[i];
      A *= a[i];
      B = BWD ? a[i] * (B + b[i]) : fmaf(a[i], B, b[i]);
    }
    // over the lanes of a channel: the pair of everything before this lane in the warp, and the warp's
    float Ae = 1.f, Be = 0.f;
    if (SUBS > 1) {
#pragma unroll
      for (int o = 1; o < SUBS; o <<= 1) {
        const float Ap = __shfl_up_sync(0xffffffffu, A, o * CW), Bp = __shfl_up_sync(0xffffffffu, B, o * CW);
        if (sub >= o) {
          B = through(A, B, Bp);
          A *= Ap;
        }
      }
      Ae = __shfl_up_sync(0xffffffffu, A, CW);
      Be = __shfl_up_sync(0xffffffffu, B, CW);
    }
    if (sub == SUBS - 1) wtot[buf][warp][ch] = make_float2(A, B);
    __syncthreads();
    if (cs > 1) {
      float At = 1.f, Bt = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float2 v = wtot[buf][w][ch];
        Bt = through(v.x, v.y, Bt);
        At *= v.x;
      }
      for (int r = warp; r < cs; r += WARPS)
        if (sub == 0) store_remote(&ctot[buf][rank][ch], r, make_float2(At, Bt));
      __syncwarp();
      cluster_sync();
    }
    float mine = state;                               // the state before this CTA's steps
    if (cs > 1) {
      for (int r = 0; r < cs; r++) {
        const float2 v = ctot[buf][r][ch];
        if (r == rank) mine = state;
        state = through(v.x, v.y, state);
      }
    }
    float run = mine;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      if (w == warp) run = mine;
      const float2 v = wtot[buf][w][ch];
      mine = through(v.x, v.y, mine);
    }
    if (cs == 1) state = mine;
    if (SUBS > 1 && sub > 0) run = through(Ae, Be, run);
#pragma unroll
    for (int i = 0; i < SEG; i++) {
      const int q = p0 + i;
      const bool there = on && q < len;
      if (!BWD) {
        run = fmaf(a[i], run, b[i]);
        if (there) p.out[seq * p.ss_h + q * p.ts_h + c] = run;
      } else {
        const float G = b[i] + run;
        run = a[i] * G;
        const float gx = GATED ? s[i] * G : G;
        const float gf = GATED ? G * (hp[i] - xv[i]) * (a[i] * s[i]) : G * hp[i];
        if (there) {
          const long long at = seq * p.ss_in + (len - 1 - q) * p.ts_in + c;
          p.dx[at] = p.accumulate ? __fadd_rn(p.dx[at], gx) : gx;
          p.df[at] = p.accumulate ? __fadd_rn(p.df[at], gf) : gf;
        }
      }
    }
  }
  float* last = BWD ? p.dh0 : p.last;
  if (last && on && rank == 0 && warp == 0 && sub == 0) last[edge] = BWD && p.accumulate ? __fadd_rn(last[edge], state) : state;
}

// One thread a channel: single tokens and very short sequences.
template <bool GATED, bool BWD>
__global__ void __launch_bounds__(THREADS) step_kernel(const Params p) {
  const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
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
  return FML_OK;
}

template <int CW, int SEG, bool GATED, bool BWD>
int32_t launch_scan(fml_ctx* ctx, Params& p, int cluster) {
  p.ctiles = (p.dim + CW - 1) / CW;
  p.cluster = cluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.n_seq * p.ctiles * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  FML_CUDA(ctx, cudaLaunchKernelEx(&cfg, scan_kernel<CW, SEG, GATED, BWD>, (const Params)p));
  return FML_OK;
}

template <bool GATED, bool BWD>
int32_t launch(fml_ctx* ctx, Params& p) {
  if (p.n_seq == 0) return FML_OK;
  if (p.seq_len <= 4) {
    step_kernel<GATED, BWD><<<(unsigned)(((long long)p.n_seq * p.dim + THREADS - 1) / THREADS), THREADS, 0, ctx->stream>>>(p);
    FML_LAUNCH_CHECK(ctx, "step_kernel");
    return FML_OK;
  }
  constexpr int SEG = BWD ? 8 : 16;
  // Few channels: narrower tiles and a cluster along the time axis, until there are four CTAs an SM or no more steps to split
  const long long want = 4ll * ctx->sm_count;
  int cw = 32;
  while (cw > 8 && (long long)p.n_seq * ((p.dim + cw - 1) / cw) * MAX_CLUSTER < want) cw >>= 1;
  const long long units = (long long)p.n_seq * ((p.dim + cw - 1) / cw);
  const int tile = WARPS * (32 / cw) * SEG;
  int cluster = 1;
  while (cluster < MAX_CLUSTER && units * cluster < want && (long long)tile * cluster < p.seq_len) cluster <<= 1;
  if (cw == 32) return launch_scan<32, SEG, GATED, BWD>(ctx, p, cluster);
  if (cw == 16) return launch_scan<16, SEG, GATED, BWD>(ctx, p, cluster);
  return launch_scan<8, SEG, GATED, BWD>(ctx, p, cluster);
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

}  // extern "C"
