// Root-mean-square norm of every query and key head, its gain, and the position rotation, in one pass; and the backward
// pass.  It stands between the projections and the attention kernels (lib/layertypes/singleHeadAttentionLayer.dart:77-86
// has neither; an extension).
//
//   r = 1 / sqrt(mean(x^2) + eps)    xh = x r    z = gain xh    y = R(pos) z
//   R turns the pairs of the first rot_dim elements by pos base^(-2 i / rot_dim): pairs (i, i + rot_dim / 2), or neighbours
//   dz = R^T dy    dgain += sum dz xh    dx = r (gain dz - xh mean(gain dz xh))
//
// Bound: memory, 8 bytes an element forward (x in, y out), 12 backward (x, dy in, dx out).  Nothing is saved between the
// two passes: r comes again from the head, which the backward pass has in registers anyway.
//
// Layout: 4, 8, 16 or 32 lanes hold a head (d_head up to 32, 64, 128, 256), eight elements each: two float4, in the rotated
// part four elements of its first half and their partners of the second, so a pair never leaves its lane; the only exchange
// is the reduction.  A warp takes 32 / lanes heads at once, the heads of a CTA's rows counted through, and the loads of the
// next such item are under way while one is used.  The cosines and sines of a CTA's rows are formed once, into shared memory, for
// all heads: the angle in turns in double (pos times a frequency keeps no fraction in 24 bits at far positions), its fraction
// in float.  Addresses or row strides that float4 cannot take are read float by float in the same places; head widths and
// rotated parts that are no multiple of eight run the same steps with one warp a head, pairs of floats.
// dgain: each CTA leaves its sums in the caller's scratch, a second launch adds them in a fixed order.
//
// Measured on 16384 rows of 16 + 16 heads of 64: forward 47 us (0.88 of the copy bandwidth), backward 66 (0.93), the gain sums
// 5.  4999 rows of 12 + 3 heads of 80 at an odd stride: 14 and 21 us (0.5 of it), bound by instructions: ten of sixteen lanes
// work, with single floats (whole pairs side by side in the lanes, so that neighbours load neighbours, took 17 and 26).
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int MAX_PARTS = FML_QK_NORM_ROPE_PARTS;   // CTAs of a backward launch, one partial sum each
constexpr int MAX_D = 256;
// CTAs an SM: 64 registers a thread forward, 80 backward.  Measured on 16384 rows of 16 + 16 heads of 64, both passes: 122 us,
// 127 with two backward, 129 with five forward; 131 with two items read ahead (three and one CTAs), 129 with CTAs of 16 warps.
// At 80 registers the backward kernels spill 4 to 28 bytes.
constexpr int CTAS_FWD = 4, CTAS_BWD = 3;

struct Side {          // queries or keys
  const float* x;
  const float* dy;     // backward
  float* out;          // y, or dx
  long long ldx, ldy, ldo;
  const float* gain;
  int heads;
  uint32_t per_head;   // ceil(2^32 / heads): divides by multiplying
  int wide;            // which of x (1), dy (2), out (4) can be read or written four floats at a time
};
struct Params {
  Side s[2];
  const int* pos;
  float* parts;        // [CTA][2][d], or NULL when no gain gradient is wanted
  long long rows, each;  // each: rows of a CTA, one more in the first `more` CTAs
  int more;
  int seq_len, d, rot, interleaved, accumulate;
  int rows_cta;        // rows whose angles a CTA forms at once
  double kexp;         // -2 log2(base) / rot
  float eps;
};

// Turns a position of the pairs, in double: once a CTA (the power costs as much as ten sines)
__device__ __forceinline__ void frequencies(const Params& p, double* freq) {
  for (int j = threadIdx.x; j < p.rot >> 1; j += THREADS) freq[j] = exp2(p.kexp * j) * 0.15915494309189533577;
}
// cosines and sines of rows [r0, r0 + n), rot / 2 each a row
__device__ __forceinline__ void angles(const Params& p, const double* freq, long long r0, int n, float* cosv, float* sinv) {
  const int half = p.rot >> 1;
  const long long first = p.seq_len > 0 ? r0 % p.seq_len : r0;
  for (int i = threadIdx.x; i < n * half; i += THREADS) {
    const int r = (int)((unsigned)i / (unsigned)half), j = i - r * half;
    const double pos = p.pos ? (double)p.pos[r0 + r] : p.seq_len > 0 ? (double)((unsigned)(first + r) % (unsigned)p.seq_len) : (double)(first + r);
    const double turns = pos * freq[j];
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cosv[i] = c;
    sinv[i] = s;
  }
}

// first row of CTA b's share: neighbouring rows, the shares equal to a row
__device__ __forceinline__ long long share(const Params& p, unsigned b) { return p.each * b + min(b, (unsigned)p.more); }

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float inv_root(float v) {   // two units in the last place; eps keeps v a normal number
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void load4(float* v, const float* p, bool wide) {
  if (wide) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
  else
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = p[i];
}
__device__ __forceinline__ void store4(float* p, const float* v, bool wide) {
  if (wide) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
  else
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = v[i];
}

// A lane's place in a head: four elements from e0 on and four from e1 on; in the rotated part the two hold each other's
// partners (pairs apart) or two pairs each (neighbouring pairs).
struct Place {
  int e0, e1, half, u;
  bool active, turned;
};

// z turned by +angle (sign = 1) or back (sign = -1)
template <bool INTER>
__device__ __forceinline__ void turn8(float* z, const float* cosr, const float* sinr, const Place& at, float sign) {
  float c[4], s[4];
  if (INTER) {
    *reinterpret_cast<float2*>(c) = *reinterpret_cast<const float2*>(cosr + 2 * at.u);
    *reinterpret_cast<float2*>(c + 2) = *reinterpret_cast<const float2*>(cosr + (at.half >> 1) + 2 * at.u);
    *reinterpret_cast<float2*>(s) = *reinterpret_cast<const float2*>(sinr + 2 * at.u);
    *reinterpret_cast<float2*>(s + 2) = *reinterpret_cast<const float2*>(sinr + (at.half >> 1) + 2 * at.u);
  } else {
    *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cosr + 4 * at.u);
    *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sinr + 4 * at.u);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : i + 4;
    const float a = z[ia], b = z[ib], sn = sign * s[i];
    z[ia] = a * c[i] - b * sn;
    z[ib] = a * sn + b * c[i];
  }
}

// A lane's share of a head, read ahead: eight elements, and where they are (row of the CTA's rows, column).
template <bool BWD>
struct Item {
  float x[8], dy[BWD ? 8 : 1];
  int row, col;
};
// Heads it .. it + 32 / LPH - 1 of the side, its heads in rows [r0, r0 + n) counted through.
template <int LPH, bool BWD>
__device__ __forceinline__ void load_item(const Params& p, const Side& s, long long r0, int n, int it, const Place& at, Item<BWD>& v) {
  const int head = it + (threadIdx.x & 31) / LPH;
  v.row = s.heads == 1 ? head : (int)__umulhi((uint32_t)head, s.per_head);
  v.col = (head - v.row * s.heads) * p.d;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    v.x[i] = 0.f;
    if (BWD) v.dy[i] = 0.f;
  }
  if (!at.active || head >= n * s.heads) return;
  const bool wx = s.wide & 1, wy = s.wide & 2;
  const float* src = s.x + r0 * s.ldx + v.row * s.ldx + v.col;
  load4(v.x, src + at.e0, wx);
  load4(v.x + 4, src + at.e1, wx);
  if (BWD) {
    src = s.dy + r0 * s.ldy + v.row * s.ldy + v.col;
    load4(v.dy, src + at.e0, wy);
    load4(v.dy + 4, src + at.e1, wy);
  }
}

// The heads of one side (queries or keys) in rows [r0, r0 + n), 32 / LPH of them a warp's item; the warp's first item is in
// `ahead`, and afterwards its first of `then`, the other side, if there is one.
template <int LPH, bool BWD, bool INTER>
__device__ __forceinline__ void side_heads(const Params& p, const Side& s, const Side* then, long long r0, int n, const float* cosv,
                                           const float* sinv, const Place& at, float* dg, Item<BWD>& ahead) {
  constexpr int STEP = WARPS * (32 / LPH);
  const int sub = (threadIdx.x & 31) / LPH, start = (threadIdx.x >> 5) * (32 / LPH);
  const int total = n * s.heads;
  const bool wo = s.wide & 4;
  const float inv_d = 1.f / (float)p.d;
  float* o0 = s.out + r0 * s.ldo;
  float gain[8];
#pragma unroll
  for (int i = 0; i < 8; i++) gain[i] = at.active && s.gain ? s.gain[(i < 4 ? at.e0 : at.e1) + (i & 3)] : 1.f;
  if (start >= total && then) load_item<LPH, BWD>(p, *then, r0, n, start, at, ahead);
  for (int it = start; it < total; it += STEP) {
    Item<BWD> v = ahead;
    if (it + STEP < total) load_item<LPH, BWD>(p, s, r0, n, it + STEP, at, ahead);
    else if (then) load_item<LPH, BWD>(p, *then, r0, n, start, at, ahead);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(v.x[i], v.x[i], ss);
    const float rstd = inv_root(fmaf(head_sum<LPH>(ss), inv_d, p.eps));
    const int table = min(v.row, n - 1) * at.half;
    float z[8];
    if (!BWD) {
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] = v.x[i] * rstd * gain[i];
      if (at.turned) turn8<INTER>(z, cosv + table, sinv + table, at, 1.f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] = v.dy[i];
      if (at.turned) turn8<INTER>(z, cosv + table, sinv + table, at, -1.f);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        v.x[i] *= rstd;
        dg[i] = fmaf(z[i], v.x[i], dg[i]);
        z[i] *= gain[i];
        dot = fmaf(z[i], v.x[i], dot);
      }
      dot = head_sum<LPH>(dot) * inv_d;
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] = rstd * (z[i] - v.x[i] * dot);
    }
    if (!at.active || it + sub >= total) continue;
    float* dst = o0 + v.row * s.ldo + v.col;
    if (BWD && p.accumulate) {
      float old[8];
      load4(old, dst + at.e0, wo);
      load4(old + 4, dst + at.e1, wo);
#pragma unroll
      for (int i = 0; i < 8; i++) z[i] += old[i];
    }
    store4(dst + at.e0, z, wo);
    store4(dst + at.e1, z + 4, wo);
  }
}

template <int LPH, bool BWD, bool INTER>
__global__ void __launch_bounds__(THREADS, BWD ? CTAS_BWD : CTAS_FWD) qk_vec_kernel(const Params p) {
  extern __shared__ __align__(16) float sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPH;
  const int d = p.d;
  Place at;
  at.u = lane % LPH;
  at.half = p.rot >> 1;
  at.active = at.u < (d >> 3);
  at.turned = at.u < (p.rot >> 3);
  at.e0 = at.turned ? 4 * at.u : p.rot + 4 * (at.u - (p.rot >> 3));
  at.e1 = at.turned ? 4 * at.u + at.half : at.e0 + ((d - p.rot) >> 1);
  __shared__ double freq[MAX_D / 2];
  fml_chain_next();
  frequencies(p, freq);
  fml_chain_wait();
  float* cosv = sm;
  float* sinv = sm + p.rows_cta * at.half;
  float dg[2][8];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 8; i++) dg[t][i] = 0.f;
  const long long last = share(p, blockIdx.x + 1);
  for (long long r0 = share(p, blockIdx.x); r0 < last; r0 += p.rows_cta) {
    const int n = (int)min((long long)p.rows_cta, last - r0);
    Item<BWD> ahead;                                  // under way while the angles are formed
    load_item<LPH, BWD>(p, p.s[0], r0, n, warp * (32 / LPH), at, ahead);
    __syncthreads();                                  // the table of the step before has been read
    angles(p, freq, r0, n, cosv, sinv);
    __syncthreads();
    side_heads<LPH, BWD, INTER>(p, p.s[0], &p.s[1], r0, n, cosv, sinv, at, dg[0], ahead);
    side_heads<LPH, BWD, INTER>(p, p.s[1], nullptr, r0, n, cosv, sinv, at, dg[1], ahead);
  }
  if (!BWD || !p.parts) return;
  // the CTA's sums: over the warp's heads, then over the warps, in a fixed order
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float v = dg[t][i];
#pragma unroll
      for (int o = LPH; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (sub == 0 && at.active) sm[(warp * 2 + t) * d + (i < 4 ? at.e0 : at.e1) + (i & 3)] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) v += sm[w * 2 * d + i];
    p.parts[(long long)blockIdx.x * 2 * d + i] = v;
  }
}

// One warp a head, its elements as pairs: the rotated ones, then neighbours of the rest (the last may be half a pair).
template <bool BWD>
__global__ void __launch_bounds__(THREADS) qk_pair_kernel(const Params p) {
  extern __shared__ float sm[];
  constexpr int SLOTS = MAX_D / 64;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = p.rot >> 1, d = p.d;
  __shared__ double freq[MAX_D / 2];
  fml_chain_next();
  frequencies(p, freq);
  fml_chain_wait();
  float* cosv = sm;
  float* sinv = sm + p.rows_cta * half;
  const int total = p.s[0].heads + p.s[1].heads;
  int ea[SLOTS], eb[SLOTS];                            // elements of the lane's pairs, -1: none
  float dg[2][SLOTS][2];
#pragma unroll
  for (int j = 0; j < SLOTS; j++) {
    const int q = lane + 32 * j;
    if (q < half) {
      ea[j] = p.interleaved ? 2 * q : q;
      eb[j] = p.interleaved ? 2 * q + 1 : q + half;
    } else {
      const int e = p.rot + 2 * (q - half);
      ea[j] = e < d ? e : -1;
      eb[j] = e + 1 < d ? e + 1 : -1;
    }
    dg[0][j][0] = dg[0][j][1] = dg[1][j][0] = dg[1][j][1] = 0.f;
  }
  const float inv_d = 1.f / (float)d;
  const long long last = share(p, blockIdx.x + 1);
  for (long long r0 = share(p, blockIdx.x); r0 < last; r0 += p.rows_cta) {
    const int n = (int)min((long long)p.rows_cta, last - r0);
    __syncthreads();
    angles(p, freq, r0, n, cosv, sinv);
    __syncthreads();
    for (int it = warp; it < n * total; it += WARPS) {
      const int r = it / total, head = it - r * total;
      const int key = head >= p.s[0].heads;
      const Side& s = p.s[key];
      const long long h0 = (long long)(key ? head - p.s[0].heads : head) * d;
      const float* src = s.x + (r0 + r) * s.ldx + h0;
      float xa[SLOTS], xb[SLOTS], ya[SLOTS], yb[SLOTS];
#pragma unroll
      for (int j = 0; j < SLOTS; j++) {
        xa[j] = ea[j] >= 0 ? src[ea[j]] : 0.f;
        xb[j] = eb[j] >= 0 ? src[eb[j]] : 0.f;
      }
      if (BWD) {
        const float* dsrc = s.dy + (r0 + r) * s.ldy + h0;
#pragma unroll
        for (int j = 0; j < SLOTS; j++) {
          ya[j] = ea[j] >= 0 ? dsrc[ea[j]] : 0.f;
          yb[j] = eb[j] >= 0 ? dsrc[eb[j]] : 0.f;
        }
      }
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < SLOTS; j++) ss = fmaf(xa[j], xa[j], fmaf(xb[j], xb[j], ss));
      const float rstd = inv_root(fmaf(head_sum<32>(ss), inv_d, p.eps));
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < SLOTS; j++) {
        const int q = lane + 32 * j;
        const float c = q < half ? cosv[r * half + q] : 1.f, sn = q < half ? sinv[r * half + q] : 0.f;
        const float ga = s.gain && ea[j] >= 0 ? s.gain[ea[j]] : 1.f, gb = s.gain && eb[j] >= 0 ? s.gain[eb[j]] : 1.f;
        xa[j] *= rstd;
        xb[j] *= rstd;
        if (!BWD) {
          const float za = xa[j] * ga, zb = xb[j] * gb;
          ya[j] = q < half ? za * c - zb * sn : za;
          yb[j] = q < half ? za * sn + zb * c : zb;
        } else {
          float za = q < half ? ya[j] * c + yb[j] * sn : ya[j], zb = q < half ? yb[j] * c - ya[j] * sn : yb[j];
          dg[0][j][0] += key ? 0.f : za * xa[j];
          dg[0][j][1] += key ? 0.f : zb * xb[j];
          dg[1][j][0] += key ? za * xa[j] : 0.f;
          dg[1][j][1] += key ? zb * xb[j] : 0.f;
          za *= ga;
          zb *= gb;
          dot = fmaf(za, xa[j], fmaf(zb, xb[j], dot));
          ya[j] = za;
          yb[j] = zb;
        }
      }
      if (BWD) {
        dot = head_sum<32>(dot) * inv_d;
#pragma unroll
        for (int j = 0; j < SLOTS; j++) {
          ya[j] = rstd * (ya[j] - xa[j] * dot);
          yb[j] = rstd * (yb[j] - xb[j] * dot);
        }
      }
      float* dst = s.out + (r0 + r) * s.ldo + h0;
#pragma unroll
      for (int j = 0; j < SLOTS; j++) {
        if (ea[j] >= 0) dst[ea[j]] = BWD && p.accumulate ? dst[ea[j]] + ya[j] : ya[j];
        if (eb[j] >= 0) dst[eb[j]] = BWD && p.accumulate ? dst[eb[j]] + yb[j] : yb[j];
      }
    }
  }
  if (!BWD || !p.parts) return;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int j = 0; j < SLOTS; j++) {
      if (ea[j] >= 0) sm[(warp * 2 + t) * d + ea[j]] = dg[t][j][0];
      if (eb[j] >= 0) sm[(warp * 2 + t) * d + eb[j]] = dg[t][j][1];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) v += sm[w * 2 * d + i];
    p.parts[(long long)blockIdx.x * 2 * d + i] = v;
  }
}

// dgain += the CTAs' sums, 32 columns a block, in a fixed order.  32 warps, so that a thread's loads are one trip to memory:
// with eight it took 10 us.
__global__ void __launch_bounds__(1024) qk_gain_kernel(const float* parts, int n_parts, int d, float* dgain_q, float* dgain_k) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  fml_chain_next();
  fml_chain_wait();
  const int col = blockIdx.x * 32 + warp;
  float* dst = col < d ? dgain_q : dgain_k;
  if (dst) dst += col < d ? col : col - d;
  const bool mine = lane == 0 && col < 2 * d && dst;
  const float old = mine ? *dst : 0.f;
  constexpr int PER = (MAX_PARTS + 31) / 32;
  float v[PER], sum = 0.f;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int c = warp + 32 * k;
    v[k] = i < 2 * d && c < n_parts ? parts[(long long)c * 2 * d + i] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < PER; k++) sum += v[k];
  red[lane][warp] = sum;
  __syncthreads();
  sum = red[warp][lane];                              // column `warp` of the block, the warps' sums across the lanes
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (mine) *dst = old + sum;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether two row-strided slices share an element.  Slices of one row stride are compared column by column, so the
// parts of a fused projection are told apart; others by their ranges.
bool clash(const float* a, long long lda, long long wa, const float* b, long long ldb, long long wb, long long rows) {
  if (!a || !b || rows == 0 || wa == 0 || wb == 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  if (pa + 4 * ((rows - 1) * lda + wa) <= pb || pb + 4 * ((rows - 1) * ldb + wb) <= pa) return false;
  if (rows == 1 || lda != ldb || (pa & 3) != (pb & 3)) return true;
  const long long off = ((long long)(pb - pa) / 4 % lda + lda) % lda;   // b's first column, counted from a's
  return off < wa || off + wb > lda;
}
bool same(const float* a, long long lda, const float* b, long long ldb) { return a == b && lda == ldb; }

int32_t check(fml_ctx* ctx, const Params& p, double base) {
  FML_REQUIRE(ctx, p.rows >= 0 && p.d >= 1 && p.d <= MAX_D, "fml_qk_norm_rope: d_head must be 1 .. 256");
  FML_REQUIRE(ctx, p.s[0].heads >= 1 && p.s[1].heads >= 0 && p.s[0].heads <= 32768 && p.s[1].heads <= 32768, "fml_qk_norm_rope: bad number of heads");
  FML_REQUIRE(ctx, p.rot >= 0 && p.rot <= p.d && p.rot % 2 == 0, "fml_qk_norm_rope: rot_dim must be even, 0 .. d_head");
  FML_REQUIRE(ctx, p.rot == 0 || (base > 0 && isfinite(base)), "fml_qk_norm_rope: base must be positive");
  FML_REQUIRE(ctx, p.eps >= 1e-37f && isfinite(p.eps), "fml_qk_norm_rope: eps must be 1e-37 or more");
  FML_REQUIRE(ctx, p.seq_len >= 0, "fml_qk_norm_rope: bad seq_len");
  FML_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(p.s[0].gain) | reinterpret_cast<uintptr_t>(p.s[1].gain) | reinterpret_cast<uintptr_t>(p.pos)) & 3) == 0,
              "fml_qk_norm_rope: misaligned gains or positions");
  for (int t = 0; t < 2; t++) {
    const Side& s = p.s[t];
    if (s.heads == 0) continue;
    FML_REQUIRE(ctx, s.x && s.out && ((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.out) | reinterpret_cast<uintptr_t>(s.dy)) & 3) == 0,
                "fml_qk_norm_rope: missing or misaligned buffer");
    const long long w = (long long)s.heads * p.d;
    FML_REQUIRE(ctx, s.ldx >= w && s.ldo >= w && (!s.dy || s.ldy >= w), "fml_qk_norm_rope: a row stride is shorter than the heads");
  }
  // an output may take the place of its own input; anything else that it shares with another buffer would be read after
  // it was overwritten
  for (int t = 0; t < 2; t++) {
    const Side& s = p.s[t];
    const long long w = (long long)s.heads * p.d;
    for (int o = 0; o < 2; o++) {
      const Side& q = p.s[o];
      const long long wq = (long long)q.heads * p.d;
      const bool x_ok = o == t && same(s.out, s.ldo, q.x, q.ldx), dy_ok = o == t && same(s.out, s.ldo, q.dy, q.ldy) && !p.accumulate;
      FML_REQUIRE(ctx, x_ok || !clash(s.out, s.ldo, w, q.x, q.ldx, wq, p.rows), "fml_qk_norm_rope: an output overlaps an input");
      FML_REQUIRE(ctx, dy_ok || !clash(s.out, s.ldo, w, q.dy, q.ldy, wq, p.rows), "fml_qk_norm_rope: an output overlaps an input");
    }
  }
  FML_REQUIRE(ctx, !clash(p.s[0].out, p.s[0].ldo, (long long)p.s[0].heads * p.d, p.s[1].out, p.s[1].ldo, (long long)p.s[1].heads * p.d, p.rows),
              "fml_qk_norm_rope: the outputs overlap");
  return FML_OK;
}

// Whether heads can be shared out by eights; and what the lanes need to know for that
bool can_vec(Params& p) {
  if (p.d % 8 || p.rot % 8) return false;   // the rest of the head is a multiple of 8 then too
  for (Side& s : p.s) {
    s.per_head = s.heads > 1 ? (uint32_t)(((1ull << 32) + s.heads - 1) / s.heads) : 0;   // exact for numbers below 2^32 / heads
    s.wide = (al16(s.x) && s.ldx % 4 == 0 ? 1 : 0) | (al16(s.dy) && s.ldy % 4 == 0 ? 2 : 0) | (al16(s.out) && s.ldo % 4 == 0 ? 4 : 0);
  }
  return true;
}

template <int LPH, bool BWD>
cudaError_t launch_vec(const Params& p, int grid, size_t smem, cudaStream_t s) {
  return fml_launch_chained(p.interleaved ? qk_vec_kernel<LPH, BWD, true> : qk_vec_kernel<LPH, BWD, false>, dim3(grid), dim3(THREADS), smem, s, p);
}

template <bool BWD>
int32_t launch(fml_ctx* ctx, Params& p, int* grid_out) {
  const bool vec = can_vec(p);
  const int lph = p.d <= 32 ? 4 : p.d <= 64 ? 8 : p.d <= 128 ? 16 : 32;
  const int fit = ctx->sm_count * (BWD ? CTAS_BWD : CTAS_FWD);
  const int grid = (int)std::min<long long>({p.rows, fit, BWD ? MAX_PARTS : fit});
  p.each = p.rows / grid;
  p.more = (int)(p.rows % grid);
  // rows whose angles are formed at once: a table of 32 KB at most, no more than the CTA has, and the heads of all of them
  // times the heads of one below 2^32, where dividing by multiplying is exact
  const long long heads = std::max(p.s[0].heads, p.s[1].heads);
  p.rows_cta = (int)std::min<long long>({32, 8192 / std::max(p.rot, 1), (p.rows + grid - 1) / grid, std::max(1ll, (1ll << 31) / (heads * heads))});
  const int rc = p.rows_cta;
  const size_t smem = std::max<size_t>((size_t)rc * p.rot * 4, BWD ? (size_t)WARPS * 2 * p.d * 4 : 0);   // at most 32 KB
  const cudaError_t e = !vec        ? fml_launch_chained(qk_pair_kernel<BWD>, dim3(grid), dim3(THREADS), smem, ctx->stream, p)
                        : lph == 4  ? launch_vec<4, BWD>(p, grid, smem, ctx->stream)
                        : lph == 8  ? launch_vec<8, BWD>(p, grid, smem, ctx->stream)
                        : lph == 16 ? launch_vec<16, BWD>(p, grid, smem, ctx->stream)
                                    : launch_vec<32, BWD>(p, grid, smem, ctx->stream);
  if (e != cudaSuccess) return fml_fail(ctx, FML_ERR_CUDA, std::string("qk_norm_rope kernel: ") + cudaGetErrorString(e));
  *grid_out = grid;
  return FML_OK;
}

}  // namespace

extern "C" {

int32_t fml_qk_norm_rope_fwd(fml_ctx* ctx, const float* q, int64_t ld_q, float* q_out, int64_t ld_q_out, int32_t heads_q, const float* k,
                             int64_t ld_k, float* k_out, int64_t ld_k_out, int32_t heads_k, int64_t rows, int32_t d_head,
                             const float* gain_q, const float* gain_k, const int32_t* positions, int32_t seq_len, int32_t rot_dim,
                             int32_t interleaved, double base, float eps) {
  FML_REQUIRE(ctx, ctx, "fml_qk_norm_rope_fwd: no context");
  FML_ENTER(ctx);
  Params p = {};
  p.s[0] = {q, nullptr, q_out, ld_q, 0, ld_q_out, gain_q, heads_q};
  p.s[1] = {k, nullptr, k_out, ld_k, 0, ld_k_out, gain_k, heads_k};
  p.pos = positions; p.rows = rows; p.seq_len = seq_len; p.d = d_head; p.rot = rot_dim; p.interleaved = interleaved != 0; p.eps = eps;
  int32_t rc = check(ctx, p, base);
  if (rc || rows == 0) return rc;
  p.kexp = rot_dim ? -2.0 * log2(base) / rot_dim : 0.0;
  int grid;
  return launch<false>(ctx, p, &grid);
}

int32_t fml_qk_norm_rope_bwd(fml_ctx* ctx, const float* q, int64_t ld_q, const float* dq_out, int64_t ld_dq_out, float* dq, int64_t ld_dq,
                             int32_t heads_q, const float* k, int64_t ld_k, const float* dk_out, int64_t ld_dk_out, float* dk,
                             int64_t ld_dk, int32_t heads_k, int64_t rows, int32_t d_head, const float* gain_q, const float* gain_k,
                             float* dgain_q, float* dgain_k, const int32_t* positions, int32_t seq_len, int32_t rot_dim,
                             int32_t interleaved, double base, float eps, int32_t accumulate, float* scratch) {
  FML_REQUIRE(ctx, ctx, "fml_qk_norm_rope_bwd: no context");
  FML_ENTER(ctx);
  Params p = {};
  p.s[0] = {q, dq_out, dq, ld_q, ld_dq_out, ld_dq, gain_q, heads_q};
  p.s[1] = {k, dk_out, dk, ld_k, ld_dk_out, ld_dk, gain_k, heads_k};
  p.pos = positions; p.rows = rows; p.seq_len = seq_len; p.d = d_head; p.rot = rot_dim; p.interleaved = interleaved != 0; p.eps = eps;
  p.accumulate = accumulate != 0;
  int32_t rc = check(ctx, p, base);
  if (rc) return rc;
  FML_REQUIRE(ctx, dq_out && (heads_k == 0 || dk_out), "fml_qk_norm_rope_bwd: missing gradient");
  FML_REQUIRE(ctx, (!dgain_q || gain_q) && (!dgain_k || (gain_k && heads_k)), "fml_qk_norm_rope_bwd: the gradient of a gain that is not there");
  FML_REQUIRE(ctx, !(dgain_q || dgain_k) || scratch, "fml_qk_norm_rope_bwd: gain gradients need the scratch buffer");
  FML_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(dgain_q) | reinterpret_cast<uintptr_t>(dgain_k) | reinterpret_cast<uintptr_t>(scratch)) & 3) == 0,
              "fml_qk_norm_rope_bwd: misaligned gain gradients or scratch buffer");
  const long long sw = (long long)MAX_PARTS * 2 * d_head;
  FML_REQUIRE(ctx, !clash(dgain_q, d_head, d_head, dgain_k, d_head, d_head, 1) && !clash(dgain_q, d_head, d_head, scratch, sw, sw, 1) &&
                       !clash(dgain_k, d_head, d_head, scratch, sw, sw, 1),
              "fml_qk_norm_rope_bwd: the gain gradients and the scratch buffer must not overlap");
  if (rows == 0) return FML_OK;
  p.kexp = rot_dim ? -2.0 * log2(base) / rot_dim : 0.0;
  p.parts = dgain_q || dgain_k ? scratch : nullptr;
  int grid;
  rc = launch<true>(ctx, p, &grid);
  if (rc || !p.parts) return rc;
  FML_CUDA(ctx, fml_launch_chained(qk_gain_kernel, dim3((unsigned)(2 * d_head + 31) / 32), dim3(1024), 0, ctx->stream, scratch, grid, d_head, dgain_q, dgain_k));
  return FML_OK;
}

}  // extern "C"
