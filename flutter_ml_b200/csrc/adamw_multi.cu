// AdamW (lib/optimizers/adamw.dart:82-89) over a list of tensors in one launch, first and second moments in 32 or 8 bits.
//
// For every element, with g' = grad_scale g, c1 = 1 - beta1^t, c2 = 1 - beta2^t:
//   m <- beta1 m + (1 - beta1) g'      v <- beta2 v + (1 - beta2) g'^2
//   w <- w - lr (m / c1) / (sqrt(v / c2) + eps)        w <- w - lr weight_decay w
//
// Bound: memory, 28 bytes an element with 32-bit states (w, m, v read and written, g read), 16 with 8-bit ones.
//
// Layout: every tensor is cut into blocks of 256 elements, one warp a block, eight elements a lane (two float4: elements
// 4 l .. 4 l + 3 and 128 + 4 l ..), all loads issued before the first use.  The states of all tensors lie in ONE buffer by
// block, so they are aligned whatever the tensors' own addresses; parameters and gradients may start anywhere.  The list
// becomes a table of work items on the device once, when the plan is made: a step is one launch whatever their number.
//
// 8-bit states.  m and r = sqrt(v) (v itself has twice the exponent range) are held as sign, four exponent and three
// fraction bits times a power of two for each block, the smallest that brings the block's largest finite value to 448 at
// most.  With a power of two every scaling is exact: the only rounding is that to three fraction bits, and a block's scale
// changing does not move the values that it holds.  Values down to 2^-18 of the block's largest keep their precision or
// part of it, smaller ones become zero; a positive r is held at 2^-9 of the scale at least, because m over a root that was
// rounded to zero would be a step of any size.  beta2 = 0.999 changes v by a thousandth a step, far less than the half step
// of 1/16 that rounding to the nearest takes away, so a v rounded that way stands still until a gradient beats it by an
// order of magnitude: rounding up with the probability of the dropped bits (16 of them) keeps m and the root right on average
// (v, the square of the root, is high by the variance of the rounding: 4 % in a simulation with normal gradients).
// The bits come from a counter (seed, step, block, element), so a run can be repeated exactly.  An element that is not
// finite is held as NaN and left out of the block's scale: it damages nothing but itself.
//
// The moments are formed with one rounding an operation (no contraction), so a restatement in any IEEE float32 arithmetic
// reproduces the codes bit for bit; the root is the rounded one.
//
// Measured on 141 M parameters: 32 bits 566 us, 7.0 TB/s; 8 bits 382 us (5.9 TB/s) at the full clock, 403 to 418 where the
// power cap lowers it: about 64 instructions an element, 0.8 of the issue slots, 4 to 20 bytes spilled at 48 registers.  The
// first form, codes taken apart by shifts and selections, took 549.  Persistent CTAs with the next block in registers: 460
// (two CTAs an SM).
#include <math.h>

#include <algorithm>
#include <new>
#include <stdexcept>

#include "common.cuh"

namespace {

constexpr int BLOCK = 256;                 // elements that share a scale, and a warp's work
constexpr int WARPS = 8;
constexpr int ITEM = BLOCK * WARPS;        // elements of a work item: one CTA

struct Item {
  float* w;
  float* g;
  uint32_t block;   // first block in the state buffers
  uint32_t count;   // elements, 1 .. ITEM
};

struct Hyper {
  float b1, omb1, b2, omb2;
  float step;       // lr / (1 - beta1^t)
  float rc2;        // 1 / sqrt(1 - beta2^t)
  float eps, decay; // decay = lr * weight_decay
  float gs;
  uint32_t key;     // of the random bits
};

// Hyper-parameters before the step count enters; with them a device-side counter can be the step count.
struct HyperIn {
  double lr, beta1, beta2, eps, decay, gs;
  int64_t seed;
};

__host__ __device__ inline uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x85EBCA77u;
  return x ^ (x >> 13);
}

__host__ __device__ inline Hyper hyper_at(const HyperIn& p, int t) {
  Hyper h;
  h.b1 = (float)p.beta1; h.omb1 = (float)(1.0 - p.beta1);
  h.b2 = (float)p.beta2; h.omb2 = (float)(1.0 - p.beta2);
  h.step = (float)(p.lr / (1.0 - pow(p.beta1, (double)t)));
  h.rc2 = (float)(1.0 / sqrt(1.0 - pow(p.beta2, (double)t)));
  h.eps = (float)p.eps; h.decay = (float)(p.lr * p.decay); h.gs = (float)p.gs;
  const uint64_t s = (uint64_t)p.seed;
  h.key = mix32(mix32(mix32((uint32_t)s) ^ (uint32_t)(s >> 32)) ^ (uint32_t)t);
  return h;
}

struct DeviceStep { Hyper h; int t; };   // the plan's own step counter, advanced on the device (captured launches included)
__global__ void advance_kernel(DeviceStep* d, const HyperIn p) {
  fml_chain_next();
  fml_chain_wait();
  if (d->t < 0x7fffffff) d->t++;
  d->h = hyper_at(p, d->t);
}

__device__ __forceinline__ bool finite_bits(uint32_t b) { return (b & 0x7fffffffu) < 0x7f800000u; }

// four codes in units of their scale
__device__ __forceinline__ void decode8(uint32_t codes, float* out) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)(codes >> (16 * i))));
    asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(out[2 * i]), "=f"(out[2 * i + 1]) : "r"(h2));
  }
}

// exponent of the block's scale from the bits of its largest finite absolute value
__device__ __forceinline__ int scale_exponent(uint32_t amax) { return max((int)((amax + 0x1FFFFFu) >> 23) - 135, -126); }

// Scales whose power of two, brought down by 2^-120, is still a float: larger ones take the rare way (see encode8)
constexpr int BIG_SCALE = 29;
__device__ __forceinline__ float power_of_two(int e) {   // -149 .. 127
  return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << (e + 149));
}

// `down` brings x to x / scale * 2^-120: then 2^-6, the format's smallest normal number, is float's smallest normal number, and
// the float's bits from the twentieth on ARE the code, subnormal or not, and those below are what is rounded away.  Returns
// them with the rounding added, moved up by four: the code in the upper byte.  `up16` is the random number in bits 8 .. 23.
template <bool NEAREST, bool SIGNED>
__device__ __forceinline__ uint32_t encode8(float x, float down, uint32_t up16) {
  const uint32_t z = __float_as_uint(__fmul_rn(x, down));
  const uint32_t t = NEAREST ? (z + 0x7FFFFu + ((z >> 20) & 1u)) * 16u : z * 16u + up16;
  return SIGNED ? t | (z & 0x80000000u) : t;
}
// the upper bytes of four numbers
__device__ __forceinline__ uint32_t pack8(const uint32_t* z) {
  return __byte_perm(__byte_perm(z[0], z[1], 0x0073), __byte_perm(z[2], z[3], 0x0073), 0x5410);
}

// A warp's block on its way through the registers: eight elements a lane, 4 l .. 4 l + 3 and 128 + 4 l ..
template <bool EIGHT>
struct Block {
  float* w;
  float* g;
  long long b;                  // block in the state buffers
  int n;                        // elements from the block's first to the work item's last; none: no block
  bool vec;                     // a whole block at addresses that float4 can take
  float wv[8], gv[8];
  float mv[EIGHT ? 1 : 8], vv[EIGHT ? 1 : 8];
  uint32_t mc[EIGHT ? 2 : 1], rc[EIGHT ? 2 : 1];
  float ms, rs;
};

template <bool EIGHT>
__device__ __forceinline__ void load_block(Block<EIGHT>& k, const Item& it, const float* mbuf, const float* vbuf, long long n_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k.n = (int)it.count - warp * BLOCK;
  if (k.n <= 0) return;
  k.b = (long long)it.block + warp;
  k.w = it.w + warp * BLOCK;
  k.g = it.g + warp * BLOCK;
  k.vec = k.n >= BLOCK && ((reinterpret_cast<uintptr_t>(k.w) | reinterpret_cast<uintptr_t>(k.g)) & 15) == 0;
  if (k.vec) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      reinterpret_cast<float4*>(k.wv)[q] = reinterpret_cast<const float4*>(k.w)[lane + 32 * q];
      reinterpret_cast<float4*>(k.gv)[q] = reinterpret_cast<const float4*>(k.g)[lane + 32 * q];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = (j >> 2) * 128 + 4 * lane + (j & 3);
      k.wv[j] = i < k.n ? k.w[i] : 0.f;
      k.gv[j] = i < k.n ? k.g[i] : 0.f;
    }
  }
  if (EIGHT) {
    const uint32_t* mw = reinterpret_cast<const uint32_t*>(mbuf) + k.b * (BLOCK / 4);
    const uint32_t* rw = reinterpret_cast<const uint32_t*>(vbuf) + k.b * (BLOCK / 4);
#pragma unroll
    for (int q = 0; q < 2; q++) { k.mc[q] = mw[lane + 32 * q]; k.rc[q] = rw[lane + 32 * q]; }
    k.ms = mbuf[n_blocks * (BLOCK / 4) + k.b];
    k.rs = vbuf[n_blocks * (BLOCK / 4) + k.b];
  } else {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      reinterpret_cast<float4*>(k.mv)[q] = reinterpret_cast<const float4*>(mbuf + k.b * BLOCK)[lane + 32 * q];
      reinterpret_cast<float4*>(k.vv)[q] = reinterpret_cast<const float4*>(vbuf + k.b * BLOCK)[lane + 32 * q];
    }
  }
}

template <bool EIGHT, bool NEAREST, bool ZERO>
__device__ __forceinline__ void update_block(Block<EIGHT>& k, float* mbuf, float* vbuf, long long n_blocks, const Hyper& h) {
  if (k.n <= 0) return;
  const int lane = threadIdx.x & 31;
  float m8[8], v8[8];
  if (EIGHT) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      decode8(k.mc[q], m8 + 4 * q);
      decode8(k.rc[q], v8 + 4 * q);
    }
  }
  float* mv = EIGHT ? m8 : k.mv;
  float* vv = EIGHT ? v8 : k.vv;
  if (h.gs != 1.f) {
#pragma unroll
    for (int j = 0; j < 8; j++) k.gv[j] = __fmul_rn(k.gv[j], h.gs);
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    float m = mv[j], v = vv[j];
    if (EIGHT) {
      m = __fmul_rn(m, k.ms);
      v = __fmul_rn(v, k.rs);
      v = __fmul_rn(v, v);
    }
    const float gj = k.gv[j];
    mv[j] = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(gj, h.omb1));
    vv[j] = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(gj, gj), h.omb2));
  }
  float root[8], mmax = 0.f, rmax = 0.f, all = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float m = mv[j];
    root[j] = __fsqrt_rn(vv[j]);
    // the hardware's reciprocal, good to one unit in the last place: it moves w by lr times that
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(root[j], h.rc2, h.eps)));
    k.wv[j] -= h.step * m * inv;
    k.wv[j] -= h.decay * k.wv[j];
    if (EIGHT) {
      mmax = fmaxf(mmax, fabsf(m));
      rmax = fmaxf(rmax, root[j]);
      all += k.wv[j];   // NaN if m or the root is
    }
  }
  if (k.vec) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      reinterpret_cast<float4*>(k.w)[lane + 32 * q] = reinterpret_cast<float4*>(k.wv)[q];
      if (ZERO) reinterpret_cast<float4*>(k.g)[lane + 32 * q] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = (j >> 2) * 128 + 4 * lane + (j & 3);
      if (i < k.n) {
        k.w[i] = k.wv[j];
        if (ZERO) k.g[i] = 0.f;
      }
    }
  }
  if (!EIGHT) {   // places behind a tensor's last element in its last block: m = v = 0 stays so
#pragma unroll
    for (int q = 0; q < 2; q++) {
      reinterpret_cast<float4*>(mbuf + k.b * BLOCK)[lane + 32 * q] = reinterpret_cast<float4*>(mv)[q];
      reinterpret_cast<float4*>(vbuf + k.b * BLOCK)[lane + 32 * q] = reinterpret_cast<float4*>(vv)[q];
    }
    return;
  }
  // A block with a number that is not finite leaves it out of its scale and makes its code NaN (fmaxf has passed over NaN).
  const bool odd = __any_sync(0xffffffffu, !(fabsf(all) < INFINITY) || mmax == INFINITY || rmax == INFINITY);
  if (odd) {
    mmax = rmax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (finite_bits(__float_as_uint(mv[j]))) mmax = fmaxf(mmax, fabsf(mv[j]));
      if (finite_bits(__float_as_uint(root[j]))) rmax = fmaxf(rmax, root[j]);
    }
  }
  const int me = scale_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(mmax)));
  const int re = scale_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(rmax)));
  // the rare way of scales above 2^29: the numbers brought down first (those that this takes below float's range have a code of 0)
  if (me > BIG_SCALE)
#pragma unroll
    for (int j = 0; j < 8; j++) mv[j] = finite_bits(__float_as_uint(mv[j])) ? mv[j] * 0x1p-120f : mv[j];
  if (re > BIG_SCALE)
#pragma unroll
    for (int j = 0; j < 8; j++) root[j] = finite_bits(__float_as_uint(root[j])) ? root[j] * 0x1p-120f : root[j];
  const float md = power_of_two(me > BIG_SCALE ? -me : -120 - me), rd = power_of_two(re > BIG_SCALE ? -re : -120 - re);
  const uint32_t key = NEAREST ? 0u : mix32(h.key + (uint32_t)k.b * 0x9E3779B1u) + 4 * lane;
  uint32_t mo[2], ro[2];
#pragma unroll
  for (int q = 0; q < 2; q++) {
    uint32_t zm[4], zr[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t word = NEAREST ? 0u : mix32(key + (q * 128 + i));
      zm[i] = encode8<NEAREST, true>(mv[4 * q + i], md, __byte_perm(word, 0, 0x4324));    // the upper half
      zr[i] = encode8<NEAREST, false>(root[4 * q + i], rd, __byte_perm(word, 0, 0x4104));  // the lower half
    }
    mo[q] = pack8(zm);
    ro[q] = pack8(zr);
    if ((ro[q] - 0x01010101u) & 0x80808080u) {        // some code is 0: a positive root keeps the smallest one
#pragma unroll
      for (int i = 0; i < 4; i++)
        if ((ro[q] >> (8 * i) & 0xffu) == 0 && vv[4 * q + i] > 0.f) ro[q] |= 1u << (8 * i);
    }
    if (odd) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t b = __float_as_uint(mv[4 * q + i]);
        if (!finite_bits(b)) mo[q] = (mo[q] & ~(0xffu << (8 * i))) | (b == 0xff800000u ? 0xffu : 0x7fu) << (8 * i);
        if (!finite_bits(__float_as_uint(root[4 * q + i]))) ro[q] = (ro[q] & ~(0xffu << (8 * i))) | 0x7fu << (8 * i);
      }
    }
  }
  uint32_t* mw = reinterpret_cast<uint32_t*>(mbuf) + k.b * (BLOCK / 4);
  uint32_t* rw = reinterpret_cast<uint32_t*>(vbuf) + k.b * (BLOCK / 4);
#pragma unroll
  for (int q = 0; q < 2; q++) { mw[lane + 32 * q] = mo[q]; rw[lane + 32 * q] = ro[q]; }
  if (lane == 0) {
    mbuf[n_blocks * (BLOCK / 4) + k.b] = __int_as_float((me + 127) << 23);
    vbuf[n_blocks * (BLOCK / 4) + k.b] = __int_as_float((re + 127) << 23);
  }
}

// One work item a CTA: the loads of the other CTAs of the SM run beside its arithmetic.
template <bool EIGHT, bool NEAREST, bool ZERO>
__global__ void __launch_bounds__(32 * WARPS, EIGHT ? 5 : 1)
adamw_kernel(const Item* __restrict__ items, float* mbuf, float* vbuf, long long n_blocks, Hyper h, const DeviceStep* dev) {
  fml_chain_next();
  const Item it = items[blockIdx.x];                  // the plan's own table: written before any step
  fml_chain_wait();
  Block<EIGHT> k;
  load_block(k, it, mbuf, vbuf, n_blocks);
  if (dev) h = dev->h;
  update_block<EIGHT, NEAREST, ZERO>(k, mbuf, vbuf, n_blocks, h);
}

int64_t blocks_of(int64_t n) { return (n + BLOCK - 1) / BLOCK; }

// Total number of blocks, or -1 (bad arguments) / -2 (more than the 32-bit block counter holds)
int64_t total_blocks(int32_t n, const int64_t* sizes) {
  if (n < 1 || !sizes) return -1;
  int64_t total = 0;
  for (int32_t i = 0; i < n; i++) {
    if (sizes[i] < 0) return -1;
    if (sizes[i] > ((int64_t)1 << 39)) return -2;
    total += blocks_of(sizes[i]);
    if (total > 0x7fffffff) return -2;
  }
  return total;
}

}  // namespace

struct fml_adamw_plan {
  Item* items = nullptr;
  DeviceStep* step = nullptr;
  float *m = nullptr, *v = nullptr;
  int64_t n_blocks = 0;
  uint32_t n_items = 0;
  int bits = 32;
  bool recorded = false;   // a graph refers to the table and the counter: they are kept until the context goes
  bool gone = false;
};

static fml_adamw_plan* find_plan(fml_ctx* ctx, int32_t id) {
  if (id < 0 || id >= (int32_t)ctx->adamw_plans.size()) return nullptr;
  fml_adamw_plan* p = ctx->adamw_plans[id];
  return p && !p->gone ? p : nullptr;
}

static void free_plan(fml_adamw_plan* p) {
  if (p->items) cudaFree(p->items);
  if (p->step) cudaFree(p->step);
  delete p;
}
void fml_adamw_release(fml_ctx* ctx) {
  for (fml_adamw_plan* p : ctx->adamw_plans)
    if (p) free_plan(p);
  ctx->adamw_plans.clear();
}

extern "C" {

int32_t fml_adamw_state_floats(int32_t n, const int64_t* sizes, int32_t state_bits, int64_t* floats) {
  if (!floats || (state_bits != 8 && state_bits != 32)) return fml_fail(nullptr, FML_ERR_INVALID, "fml_adamw_state_floats: bad arguments");
  const int64_t nb = total_blocks(n, sizes);
  if (nb < 0) return fml_fail(nullptr, nb == -1 ? FML_ERR_INVALID : FML_ERR_OOM, "fml_adamw_state_floats: bad tensor sizes");
  *floats = state_bits == 32 ? nb * BLOCK : nb * (BLOCK / 4 + 1);
  return FML_OK;
}

int32_t fml_adamw_plan_create(fml_ctx* ctx, int32_t n, float* const* w, float* const* g, const int64_t* sizes, float* m, float* v,
                              int32_t state_bits, int32_t* plan_id) {
  if (plan_id) *plan_id = -1;
  FML_REQUIRE(ctx, ctx && w && g && plan_id, "fml_adamw_plan_create: bad arguments");
  FML_REQUIRE(ctx, state_bits == 8 || state_bits == 32, "fml_adamw_plan_create: states are held in 8 or 32 bits");
  FML_REQUIRE(ctx, !ctx->capturing, "fml_adamw_plan_create: make the plan before the recording starts");
  FML_ENTER(ctx);
  const int64_t nb = total_blocks(n, sizes);
  FML_REQUIRE(ctx, nb != -1, "fml_adamw_plan_create: bad tensor sizes");
  if (nb == -2) return fml_fail(ctx, FML_ERR_OOM, "fml_adamw_plan_create: too many elements for one plan");
  FML_REQUIRE(ctx, nb == 0 || (m && v), "fml_adamw_plan_create: missing state buffer");
  FML_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
              "fml_adamw_plan_create: state buffers must be 16-byte aligned");
  fml_adamw_plan* p = nullptr;
  try {
    struct Range { uintptr_t a, e; };
    std::vector<Range> used;
    std::vector<Item> items;
    const uintptr_t sb = (uintptr_t)(state_bits == 32 ? nb * BLOCK : nb * (BLOCK / 4 + 1)) * 4;
    if (nb) {
      used.push_back({reinterpret_cast<uintptr_t>(m), reinterpret_cast<uintptr_t>(m) + sb});
      used.push_back({reinterpret_cast<uintptr_t>(v), reinterpret_cast<uintptr_t>(v) + sb});
    }
    uint32_t block = 0;
    for (int32_t i = 0; i < n; i++) {
      if (sizes[i] == 0) continue;
      FML_REQUIRE(ctx, w[i] && g[i], "fml_adamw_plan_create: missing tensor or gradient");
      FML_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(w[i]) | reinterpret_cast<uintptr_t>(g[i])) & 3) == 0,
                  "fml_adamw_plan_create: misaligned tensor or gradient");
      for (const float* q : {w[i], g[i]}) used.push_back({reinterpret_cast<uintptr_t>(q), reinterpret_cast<uintptr_t>(q + sizes[i])});
      for (int64_t o = 0; o < sizes[i]; o += ITEM, block += WARPS)
        items.push_back({w[i] + o, g[i] + o, block, (uint32_t)std::min<int64_t>(ITEM, sizes[i] - o)});
      block -= (uint32_t)((WARPS - blocks_of(sizes[i]) % WARPS) % WARPS);   // the last item's missing blocks
    }
    for (const Range& r : used) {
      cudaPointerAttributes a;
      FML_CUDA(ctx, cudaPointerGetAttributes(&a, reinterpret_cast<const void*>(r.a)));
      FML_REQUIRE(ctx, (a.type == cudaMemoryTypeDevice && a.device == ctx->device) || a.type == cudaMemoryTypeManaged,
                  "fml_adamw_plan_create: a buffer is not in the memory of the context's device");
    }
    std::sort(used.begin(), used.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
    for (size_t i = 1; i < used.size(); i++)
      FML_REQUIRE(ctx, used[i - 1].e <= used[i].a, "fml_adamw_plan_create: tensors, gradients and states must not overlap");
    p = new fml_adamw_plan();
    p->m = m; p->v = v; p->n_blocks = nb; p->n_items = (uint32_t)items.size(); p->bits = state_bits;
    cudaError_t e = cudaMalloc(&p->step, sizeof(DeviceStep));
    if (e == cudaSuccess) e = cudaMemset(p->step, 0, sizeof(DeviceStep));
    if (e == cudaSuccess && !items.empty()) e = cudaMalloc(&p->items, items.size() * sizeof(Item));
    if (e == cudaSuccess && !items.empty()) e = cudaMemcpy(p->items, items.data(), items.size() * sizeof(Item), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();   // the table is there whatever stream the first step runs on
    if (e != cudaSuccess) {
      free_plan(p);
      return fml_fail(ctx, e == cudaErrorMemoryAllocation ? FML_ERR_OOM : FML_ERR_CUDA, std::string("fml_adamw_plan_create: ") + cudaGetErrorString(e));
    }
    ctx->adamw_plans.push_back(p);
  } catch (const std::exception&) {
    if (p) free_plan(p);
    return fml_fail(ctx, FML_ERR_OOM, "fml_adamw_plan_create: out of host memory");
  }
  *plan_id = (int32_t)ctx->adamw_plans.size() - 1;
  return FML_OK;
}

int32_t fml_adamw_plan_step(fml_ctx* ctx, int32_t plan_id, int32_t lane, double lr, double beta1, double beta2, double eps,
                            double weight_decay, int32_t t, double grad_scale, int32_t zero_grad, int64_t seed) {
  FML_REQUIRE(ctx, ctx, "fml_adamw_plan_step: no context");
  FML_ENTER(ctx);
  fml_adamw_plan* p = find_plan(ctx, plan_id);
  FML_REQUIRE(ctx, p, "fml_adamw_plan_step: unknown plan");
  FML_REQUIRE(ctx, beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "fml_adamw_plan_step: betas must be in [0, 1)");
  FML_REQUIRE(ctx, eps >= 1e-37 && isfinite(eps) && isfinite(lr) && isfinite(weight_decay) && isfinite(grad_scale),
              "fml_adamw_plan_step: hyper-parameters must be finite, eps at least 1e-37");
  FML_REQUIRE(ctx, t >= 0, "fml_adamw_plan_step: t must be >= 1, or 0 for the plan's own counter");
  cudaStream_t s;
  const int32_t rc = fml_any_stream(ctx, lane, &s);
  if (rc) return rc;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;   // also of a stream that the caller records
  FML_CUDA(ctx, cudaStreamIsCapturing(s, &capture));
  p->recorded |= capture != cudaStreamCaptureStatusNone;
  const HyperIn in = {lr, beta1, beta2, eps, weight_decay, grad_scale, seed};
  const DeviceStep* dev = nullptr;
  if (t == 0) {
    FML_CUDA(ctx, fml_launch_chained(advance_kernel, dim3(1), dim3(1), 0, s, p->step, in));
    dev = p->step;
  }
  if (p->n_items == 0) return FML_OK;
  const Hyper h = hyper_at(in, t ? t : 1);
  const bool nearest = seed < 0, zero = zero_grad != 0;
  auto* k = p->bits == 32 ? (zero ? adamw_kernel<false, true, true> : adamw_kernel<false, true, false>)
            : nearest     ? (zero ? adamw_kernel<true, true, true> : adamw_kernel<true, true, false>)
                          : (zero ? adamw_kernel<true, false, true> : adamw_kernel<true, false, false>);
  FML_CUDA(ctx, fml_launch_chained(k, dim3(p->n_items), dim3(32 * WARPS), 0, s, p->items, p->m, p->v, p->n_blocks, h, dev));
  return FML_OK;
}

// The plan's own counter, once every step enqueued so far has run, on whatever stream
static int32_t counter(fml_ctx* ctx, int32_t plan_id, int* t, bool set) {
  FML_ENTER(ctx);
  fml_adamw_plan* p = find_plan(ctx, plan_id);
  FML_REQUIRE(ctx, p, "fml_adamw_plan_count: unknown plan");
  FML_REQUIRE(ctx, !ctx->capturing, "fml_adamw_plan_count: not while a graph is being recorded");
  FML_CUDA(ctx, cudaDeviceSynchronize());
  int* at = &p->step->t;
  FML_CUDA(ctx, set ? cudaMemcpy(at, t, sizeof(int), cudaMemcpyHostToDevice) : cudaMemcpy(t, at, sizeof(int), cudaMemcpyDeviceToHost));
  if (set) FML_CUDA(ctx, cudaDeviceSynchronize());
  return FML_OK;
}

int32_t fml_adamw_plan_count(fml_ctx* ctx, int32_t plan_id, int32_t* t) {
  FML_REQUIRE(ctx, ctx && t, "fml_adamw_plan_count: bad arguments");
  return counter(ctx, plan_id, t, false);
}

int32_t fml_adamw_plan_set_count(fml_ctx* ctx, int32_t plan_id, int32_t t) {
  FML_REQUIRE(ctx, ctx && t >= 0, "fml_adamw_plan_set_count: the number of steps must not be negative");
  return counter(ctx, plan_id, &t, true);
}

int32_t fml_adamw_plan_destroy(fml_ctx* ctx, int32_t plan_id) {
  FML_REQUIRE(ctx, ctx, "fml_adamw_plan_destroy: no context");
  FML_ENTER(ctx);
  fml_adamw_plan* p = find_plan(ctx, plan_id);
  FML_REQUIRE(ctx, p, "fml_adamw_plan_destroy: unknown plan");
  FML_REQUIRE(ctx, !ctx->capturing, "fml_adamw_plan_destroy: not while a graph is being recorded");
  FML_CUDA(ctx, cudaDeviceSynchronize());   // steps may still run on the main stream or on any lane
  if (p->recorded) {
    p->gone = true;
    return FML_OK;
  }
  free_plan(p);
  ctx->adamw_plans[plan_id] = nullptr;
  return FML_OK;
}

}  // extern "C"
