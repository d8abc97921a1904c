// AdamW over the FLAT fp32 parameter storage, states in 32 or in 8 bits.
//
//   t += 1;  m = b1 m + (1-b1) g;  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd on) - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)
//
// `on` is a byte per 64 elements (the flat storage's alignment, so it never
// covers two parameters): 0 leaves weight decay out there.
//
// 8-bit states: e4m3 of m and of u = sqrt(v), one fp32 scale per 64 elements
// taking the largest to 448. The square root halves v's range in octaves, so
// both fit e4m3's 2^-9..448. m is rounded to the nearest: it moves by
// 1-b1 = 10% a step, above e4m3's half step of 2^-4. u moves by less than
// (1-b2)/2 = 0.05% a step, which nearest rounding would swallow for good, so
// it goes up or down at random with the value as its mean; and never to
// zero, since m / (0 + eps) would be a step of any size. The update itself
// uses the unrounded m and v. The random bits are a mix of element pair,
// step and seed, so a step can be repeated.
//
// HBM-bound: 28 B an element with fp32 states, 16.25 B with 8-bit ones. 89.4
// million elements take 508 us (4.9 TB/s) and 299 us (4.9 TB/s); a large copy
// reaches 4.7 TB/s. 4 elements a lane: 16-byte accesses of p and g, and a
// block's 64 elements are one 16-lane row, whose maximum never leaves the
// VALU. Step number and bias corrections are a launch of one wave before, as
// every block reads them.
#include "common.h"

namespace {

constexpr int TPB = 256;
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100: a block below is 0

struct Hyper {
  float lr_bc1;   // lr / (1 - b1^t)
  float rs_bc2;   // 1 / sqrt(1 - b2^t)
  float decay;    // lr * wd
  unsigned t;     // this step's number, for the random bits
};

// Step number and learning rate live on the device: a captured step replays
// with the next number and the schedule's rate. Powers in 64 bits: 1 - b2^t
// is near 1 - b2 = 1e-3 in the first steps.
__global__ void adamw_begin_k(long* __restrict__ step, float lr,
                              const float* __restrict__ lr_dev, double b1,
                              double b2, float wd, Hyper* __restrict__ hy) {
  if (threadIdx.x) return;
  long t = step[0] + 1;
  step[0] = t;
  if (lr_dev) lr = *lr_dev;
  hy->lr_bc1 = (float)(lr / (1.0 - pow(b1, (double)t)));
  hy->rs_bc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  hy->decay = lr * wd;
  hy->t = (unsigned)t;
}

// No contraction: products and sums round as the plain operations of the CPU
// path do, so that both paths store the same 8-bit states.
DEV_INLINE void moments(float g, float& m, float& v, float b1, float c1,
                        float b2, float c2) {
#pragma clang fp contract(off)
  m = m * b1 + g * c1;
  v = v * b2 + (g * g) * c2;
}

__global__ __launch_bounds__(TPB) void adamw_k(
    float* __restrict__ p, const float* __restrict__ g,
    float* __restrict__ m, float* __restrict__ v, long n4,
    const Hyper* __restrict__ hyp, const unsigned char* __restrict__ on,
    float b1, float c1, float b2, float c2, float eps, float gs) {
  Hyper hy = *hyp;
  long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  long stride = (long)gridDim.x * blockDim.x;
  for (; i < n4; i += stride) {
    float4 pv = reinterpret_cast<float4*>(p)[i];
    float4 gv = reinterpret_cast<const float4*>(g)[i];
    float4 mv = reinterpret_cast<float4*>(m)[i];
    float4 vv = reinterpret_cast<float4*>(v)[i];
    float keep = 1.f - hy.decay * (on ? (float)on[i >> 4] : 1.f);
    float* pp = &pv.x;
    const float* gp = &gv.x;
    float *mp = &mv.x, *vp = &vv.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      moments(gp[j] * gs, mp[j], vp[j], b1, c1, b2, c2);
      pp[j] = pp[j] * keep -
              hy.lr_bc1 * mp[j] / (sqrtf(vp[j]) * hy.rs_bc2 + eps);
    }
    reinterpret_cast<float4*>(p)[i] = pv;
    reinterpret_cast<float4*>(m)[i] = mv;
    reinterpret_cast<float4*>(v)[i] = vv;
  }
}

// largest of a 16-lane row (one block of 64 elements at 4 a lane): DPP row
// rotations stay in the VALU. On the bit pattern of |x| as an integer, which
// orders like the value and keeps a NaN on top.
template <int CTRL>
DEV_INLINE unsigned row_max_step(unsigned x) {
  unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf,
                                                     0xf, true);
  return x > o ? x : o;
}
DEV_INLINE float row_absmax(const float* x) {
  unsigned a = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned b = __float_as_uint(x[j]) & 0x7fffffffu;
    a = a > b ? a : b;
  }
  a = row_max_step<0x128>(a);  // row_ror:8
  a = row_max_step<0x124>(a);
  a = row_max_step<0x122>(a);
  a = row_max_step<0x121>(a);
  return __uint_as_float(a);
}

DEV_INLINE void scale_of(float top, float* scale, float* inv) {
  bool live = !(top < kTiny);  // a NaN stays one, for its whole block
  *scale = live ? top * (1.f / 448.f) : 0.f;
  *inv = live ? (1.f / top) * 448.f : 0.f;
}

// 32 random bits for the element pair `i` of step t; the multipliers are
// fractions of the golden ratio and of the roots of 2, 3, 5 and 7
DEV_INLINE unsigned mix32(unsigned i, unsigned t, unsigned seed) {
  unsigned x = i * 0x9E3779B1u + t * 0x6A09E667u + seed * 0x3B67AE85u;
  x = (x ^ (x >> 16)) * 0x3C6EF373u;
  x = (x ^ (x >> 15)) * 0x254FF53Bu;
  return x ^ (x >> 16);
}

// e4m3 of y >= 0, up with the chance of its remainder: adding r below the
// kept bits carries into them. y above 0 stays above 0.
DEV_INLINE unsigned e4m3_random(float y, unsigned r16) {
  y = fminf(y, 448.f);
  int nrm = (int)((__float_as_uint(y) + (r16 << 4)) >> 20) - (120 << 3);
  int sub = (int)(y * 512.f + (float)r16 * (1.f / 65536.f));
  int c = y >= 0.015625f ? nrm : sub;
  c = c > 126 ? 126 : c;
  return (unsigned)(y > 0.f && c < 1 ? 1 : c) & 0xff;
}

__global__ __launch_bounds__(TPB) void adamw8_k(
    float* __restrict__ p, const float* __restrict__ g,
    unsigned* __restrict__ m8, float* __restrict__ msc,
    unsigned* __restrict__ u8, float* __restrict__ usc, long n4,
    const Hyper* __restrict__ hyp, const unsigned char* __restrict__ on,
    float b1, float c1, float b2, float c2, float eps, float gs,
    unsigned seed) {
  Hyper hy = *hyp;
  // n4 is a multiple of 16, so the 16 lanes of a row come and go together
  long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  long stride = (long)gridDim.x * blockDim.x;
  for (; i < n4; i += stride) {
    float4 pv = reinterpret_cast<float4*>(p)[i];
    float4 gv = reinterpret_cast<const float4*>(g)[i];
    unsigned mc = m8[i], uc = u8[i];
    long blk = i >> 4;
    float ms = msc[blk], us = usc[blk];
    float keep = 1.f - hy.decay * (on ? (float)on[blk] : 1.f);
    auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, false);
    auto m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, true);
    auto u01 = __builtin_amdgcn_cvt_pk_f32_fp8(uc, false);
    auto u23 = __builtin_amdgcn_cvt_pk_f32_fp8(uc, true);
    float m[4] = {m01[0] * ms, m01[1] * ms, m23[0] * ms, m23[1] * ms};
    float u[4] = {u01[0] * us, u01[1] * us, u23[0] * us, u23[1] * us};
    float* pp = &pv.x;
    const float* gp = &gv.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v = u[j] * u[j];
      moments(gp[j] * gs, m[j], v, b1, c1, b2, c2);
      u[j] = sqrtf(v);
      pp[j] = pp[j] * keep - hy.lr_bc1 * m[j] / (u[j] * hy.rs_bc2 + eps);
    }
    reinterpret_cast<float4*>(p)[i] = pv;
    float inv;
    scale_of(row_absmax(m), &ms, &inv);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m[j] = fminf(fmaxf(m[j] * inv, -448.f), 448.f);
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(m[0], m[1], 0, false);
    m8[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[2], m[3], q, true);
    scale_of(row_absmax(u), &us, &inv);
    unsigned r0 = mix32((unsigned)(2 * i), hy.t, seed);
    unsigned r1 = mix32((unsigned)(2 * i + 1), hy.t, seed);
    u8[i] = e4m3_random(u[0] * inv, r0 & 0xffff) |
            e4m3_random(u[1] * inv, r0 >> 16) << 8 |
            e4m3_random(u[2] * inv, r1 & 0xffff) << 16 |
            e4m3_random(u[3] * inv, r1 >> 16) << 24;
    if ((threadIdx.x & 15) == 0) {
      msc[blk] = ms;
      usc[blk] = us;
    }
  }
}

}  // namespace

extern "C" {

// n must be a multiple of 64 (the flat storage's alignment); msc null: m and
// v are fp32. hyp: 16 bytes of workspace.
void pdta_adamw(float* p, const float* g, void* m, void* v, float* msc,
                float* vsc, long n, long* step, float lr,
                const float* lr_dev, double b1, double b2, float eps,
                float wd, const unsigned char* on, float gs, unsigned seed,
                void* hyp, hipStream_t s) {
  Hyper* hy = (Hyper*)hyp;
  adamw_begin_k<<<1, 64, 0, s>>>(step, lr, lr_dev, b1, b2, wd, hy);
  if (n == 0) return;
  long n4 = n / 4;
  int grid = ew_grid(n4, TPB, 1);
  float f1 = (float)b1, f2 = (float)b2;
  float c1 = (float)(1.0 - b1), c2 = (float)(1.0 - b2);
  if (msc)
    adamw8_k<<<grid, TPB, 0, s>>>(p, g, (unsigned*)m, msc, (unsigned*)v, vsc,
                                  n4, hy, on, f1, c1, f2, c2, eps, gs, seed);
  else
    adamw_k<<<grid, TPB, 0, s>>>(p, g, (float*)m, (float*)v, n4, hy, on, f1,
                                 c1, f2, c2, eps, gs);
}

}  // extern "C"
