// RMS norm of each query and key head with the position rotation in the same
// pass, and its backward.
//
//   r = rsqrt(mean(x^2) + eps);  y = w x r           (no weights: y = x)
//   pairs (a, b) of the first `rot` elements turn by the position's angle:
//   (a, b) -> (a cos - b sin, b cos + a sin); a pair is (i, i + rot/2), or
//   (2i, 2i + 1) when INTER
// backward, g the gradient turned back (cos, -sin):
//   dw = sum g x r;   dx = r (w g - x r^2 mean(w g x))
//
// HBM-bound: x in, y out (and dy in, dx out). A wave takes one token: its
// cos and sin stay in registers over the token's heads. G lanes of 8
// elements (16 bytes of a 16-bit type) hold a head, so the sums are G-lane
// shuffles and one reduction serves both of backward's. x is read again in
// backward rather than 1/r kept: it is needed for dw in any case.
// dw: each lane sums its 8 columns over the tokens of its wave, blocks write
// one row each and a second kernel adds the rows in a fixed order.
// Measured: 25216 tokens of 24 heads of 64 (bf16) 27 us forward (5.8 TB/s)
// and 54 us backward (4.3 TB/s), 32768 tokens of 40 heads of 128 124 us (5.4)
// and 228 us (4.4); a large copy reaches 4.7.
#include "common.h"

namespace {

struct HeadsIn {  // one tensor [b, s, heads, hd], strides in elements
  const void* x;
  long sb, ss, sh;
  const void* dy;  // backward: gradient of y, same kind of strides
  long gb, gs, gh;
  const float* w;  // [hd] or null
  void* y;         // y forward, dx backward
  long yb, ys, yh;
  int heads;
};

struct Args {
  HeadsIn t[2];  // queries, keys
  const float *cos, *sin;  // [npos, rot/2]
  const void* pos;         // [b, s] int64 / int32, null: the row's index
  int pos32;
  int npos, rot, hd, s;
  int tokens;  // b * s, below 2^31 less the grid's stride
  float eps;
  int slices;  // waves that share a token's heads (forward)
};

// Where the 8 elements of token (b, srow), head j (queries, then keys), chunk
// lie: the token is the wave's, so its parts are scalars and a lane only
// chooses between the two tensors.
enum Which { X, DY, Y };
template <typename T, Which W>
DEV_INLINE T* at_head(const Args& a, long b, int srow, int j, int chunk) {
  auto base = [&](const HeadsIn& t) {
    if (W == X)
      return const_cast<T*>(reinterpret_cast<const T*>(t.x)) + b * t.sb +
             srow * t.ss;
    if (W == DY)
      return const_cast<T*>(reinterpret_cast<const T*>(t.dy)) + b * t.gb +
             srow * t.gs;
    return reinterpret_cast<T*>(t.y) + b * t.yb + srow * t.ys;
  };
  auto stride = [](const HeadsIn& t) {
    return W == X ? t.sh : W == DY ? t.gh : t.yh;
  };
  T *q = base(a.t[0]), *k = base(a.t[1]) - a.t[0].heads * stride(a.t[1]);
  long sq = stride(a.t[0]), sk = stride(a.t[1]);
  bool isk = j >= a.t[0].heads;
  return (isk ? k : q) + j * (isk ? sk : sq) + chunk * 8;
}

// a position outside the tables turns by NaN: the result shows it
DEV_INLINE int position(const Args& a, long tok, int srow) {
  long p = srow;
  if (a.pos)
    p = a.pos32 ? (long)reinterpret_cast<const int*>(a.pos)[tok]
                : reinterpret_cast<const long*>(a.pos)[tok];
  return p >= 0 && p < a.npos ? (int)p : -1;
}

template <int G>
DEV_INLINE float group_sum(float x) {
#pragma unroll
  for (int m = 1; m < G; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// this lane's cos and sin for its 8 elements (halves) or 4 pairs (INTER);
// for halves the sign of the partner's term is in sin
template <bool INTER>
struct Turn {
  float c[8], s[8];
  int partner;  // lane of the other half
  DEV_INLINE void load(const Args& a, int pos, int chunk, int lane) {
    int e0 = chunk * 8;
    partner = lane;
    bool on = e0 < a.rot;
    constexpr int N = INTER ? 4 : 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (!on) return;
    int half = a.rot / 2;
    int a0 = INTER ? e0 / 2 : (e0 < half ? e0 : e0 - half);
    if (!INTER) partner = e0 < half ? lane + half / 8 : lane - half / 8;
    if (pos < 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = s[i] = __uint_as_float(0x7fc00000u);
      return;
    }
    const float* cp = a.cos + (long)pos * half + a0;
    const float* sp = a.sin + (long)pos * half + a0;
    float sg = !INTER && e0 < half ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      float4 c4 = *reinterpret_cast<const float4*>(cp + i);
      float4 s4 = *reinterpret_cast<const float4*>(sp + i);
      c[i] = c4.x, c[i + 1] = c4.y, c[i + 2] = c4.z, c[i + 3] = c4.w;
      s[i] = sg * s4.x, s[i + 1] = sg * s4.y, s[i + 2] = sg * s4.z,
      s[i + 3] = sg * s4.w;
    }
  }
  // BACK turns by the opposite angle
  template <bool BACK>
  DEV_INLINE void apply(float* v) const {
    if (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = v[2 * i], y = v[2 * i + 1], sn = BACK ? -s[i] : s[i];
        v[2 * i] = x * c[i] - y * sn;
        v[2 * i + 1] = y * c[i] + x * sn;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float o = __shfl(v[i], partner, 64);
        v[i] = v[i] * c[i] + o * (BACK ? -s[i] : s[i]);
      }
    }
  }
};

template <typename T, int G, bool INTER>
__global__ __launch_bounds__(256) void qknorm_fwd_k(Args a) {
  int lane = threadIdx.x & 63;
  unsigned wv = blockIdx.x * 4 +
                __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tok = wv / (unsigned)a.slices;
  if (tok >= a.tokens) return;
  int slice = wv - tok * a.slices;
  int chunk = lane & (G - 1), grp = lane / G;
  bool act = chunk * 8 < a.hd;
  int b = __builtin_amdgcn_readfirstlane(tok / a.s);
  int srow = tok - b * a.s;
  Turn<INTER> turn;
  if (a.rot) turn.load(a, position(a, tok, srow), chunk, lane);
  float w[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) w[k][i] = 1.f;
  bool norm = a.t[0].w != nullptr;
  if (norm && act)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      Vec8<float> v = load8(a.t[k].w + chunk * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[k][i] = v.v[i];
    }
  float inv_hd = 1.f / (float)a.hd;
  int nv = a.t[0].heads + a.t[1].heads;
  // all lanes run the same number of turns: the shuffles need them
  for (int j0 = slice * (64 / G); j0 < nv; j0 += a.slices * (64 / G)) {
    int j = j0 + grp;
    bool isk = j >= a.t[0].heads;
    bool live = act && j < nv;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (live) {
      Vec8<T> v = load8(at_head<T, X>(a, b, srow, j, chunk));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = to_f32(v.v[i]);
    }
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      float r = rsqrtf(group_sum<G>(ss) * inv_hd + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= r * (isk ? w[1][i] : w[0][i]);
    }
    if (a.rot) turn.template apply<false>(x);
    if (live) {
      Vec8<T> v;
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = from_f32<T>(x[i]);
      store8(at_head<T, Y>(a, b, srow, j, chunk), v);
    }
  }
}

// part: [gridDim.x][2][hd] partial dw
template <typename T, int G, bool INTER>
__global__ __launch_bounds__(256, 4) void qknorm_bwd_k(Args a,
                                                    float* __restrict__ part) {
  __shared__ float red[4][2][G * 8];
  // weights in LDS: with them in registers too few waves fit
  __shared__ __attribute__((aligned(16))) float wl[2][G * 8];
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int chunk = lane & (G - 1), grp = lane / G;
  bool act = chunk * 8 < a.hd;
  bool norm = a.t[0].w != nullptr;
  float acc[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[k][i] = 0.f;
  for (int e = threadIdx.x; e < 2 * G * 8; e += 256) {
    int k = e / (G * 8), col = e % (G * 8);
    wl[k][col] = norm && col < a.hd ? a.t[k].w[col] : 1.f;
  }
  __syncthreads();
  float inv_hd = 1.f / (float)a.hd;
  int nv = a.t[0].heads + a.t[1].heads;
  // One step ahead: the loads of the next heads (and of the next token's
  // angles) are out while these are worked on; without that, 16 waves a CU
  // keep too few bytes in flight.
  struct Raw {
    Vec8<T> x, d;
  };
  struct Token {
    int at, b, row;
  };
  auto token = [&](int at) {
    int b = __builtin_amdgcn_readfirstlane(at / a.s);
    return Token{at, b, at - b * a.s};
  };
  if ((int)blockIdx.x * 4 + wave < a.tokens) {
    auto fetch = [&](const Token& t, int j0, Raw& r) {
      int j = j0 + grp;
      if (!act || j >= nv) return;
      r.d = load8(at_head<T, DY>(a, t.b, t.row, j, chunk));
      if (norm) r.x = load8(at_head<T, X>(a, t.b, t.row, j, chunk));
    };
    auto angles = [&](const Token& t, Turn<INTER>& turn) {
      if (a.rot) turn.load(a, position(a, t.at, t.row), chunk, lane);
    };
    Raw raw;
    Turn<INTER> turn;
    Token tok = token(blockIdx.x * 4 + wave);
    angles(tok, turn);
    fetch(tok, 0, raw);
    for (int j0 = 0;;) {
      int nj = j0 + 64 / G;
      Token nt = tok;
      if (nj >= nv) {
        nj = 0;
        nt = token(tok.at + gridDim.x * 4);
      }
      bool more = nt.at < a.tokens;
      Raw next;
      if (more) fetch(nt, nj, next);
      int j = j0 + grp;
      bool isk = j >= a.t[0].heads;
      bool live = act && j < nv;
      float x[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = live && norm ? to_f32(raw.x.v[i]) : 0.f;
        g[i] = live ? to_f32(raw.d.v[i]) : 0.f;
      }
      if (a.rot) turn.template apply<true>(g);
      if (more && nj == 0) angles(nt, turn);
      if (norm) {
        float ss = 0.f, dot = 0.f;
        Vec8<float> w = load8(&wl[isk ? 1 : 0][chunk * 8]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss += x[i] * x[i];
          dot += x[i] * g[i] * w.v[i];
        }
        ss = group_sum<G>(ss);
        dot = group_sum<G>(dot);
        float r = rsqrtf(ss * inv_hd + a.eps);
        float f = r * r * dot * inv_hd;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float gx = g[i] * (x[i] * r);
          acc[0][i] += isk ? 0.f : gx;
          acc[1][i] += isk ? gx : 0.f;
          g[i] = r * (g[i] * w.v[i] - x[i] * f);
        }
      }
      if (live) {
        Vec8<T> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = from_f32<T>(g[i]);
        store8(at_head<T, Y>(a, tok.b, tok.row, j, chunk), v);
      }
      if (!more) break;
      raw = next;
      tok = nt;
      j0 = nj;
    }
  }
  if (!norm) return;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = acc[k][i];
#pragma unroll
      for (int m = G; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
      if (grp == 0) red[wave][k][chunk * 8 + i] = s;
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.hd; e += 256) {
    int k = e >= a.hd, col = e - k * a.hd;
    part[(long)blockIdx.x * 2 * a.hd + e] =
        (red[0][k][col] + red[1][k][col]) + (red[2][k][col] + red[3][k][col]);
  }
}

// Any head size up to 256, any even rot, any strides and alignment: a wave
// per head, a lane per element (and the 64th after it), partners exchanged
// through LDS. For what the 8-element lanes cannot load.
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void qknorm_any_k(Args a, int inter,
                                                    float* __restrict__ part) {
  __shared__ float buf[4][256];
  __shared__ float red[4][2][256];
  int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  bool norm = a.t[0].w != nullptr;
  int half = a.rot / 2;
  int nv = a.t[0].heads + a.t[1].heads;
  float acc[2][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[0][k] = acc[1][k] = 0.f;
  float inv_hd = 1.f / (float)a.hd;
  long total = (long)a.tokens * nv;
  for (long u = (long)blockIdx.x * 4 + wave; u < total;
       u += (long)gridDim.x * 4) {
    long tok = u / nv;
    int j = (int)(u - tok * nv);
    bool isk = j >= a.t[0].heads;
    const HeadsIn& t = a.t[isk ? 1 : 0];
    int head = isk ? j - a.t[0].heads : j;
    long b = tok / a.s;
    int srow = (int)(tok - b * a.s);
    const T* xp = reinterpret_cast<const T*>(t.x) + b * t.sb + srow * t.ss +
                  head * t.sh;
    const T* gp = reinterpret_cast<const T*>(t.dy) + b * t.gb + srow * t.gs +
                  head * t.gh;
    T* yp = reinterpret_cast<T*>(t.y) + b * t.yb + srow * t.ys + head * t.yh;
    int pos = a.rot ? position(a, tok, srow) : 0;
    float x[4], v[4], w[4], ss = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int e = lane + 64 * k;
      bool in = e < a.hd;
      x[k] = in && (norm || !BWD) ? to_f32(xp[e]) : 0.f;
      w[k] = in && norm ? t.w[e] : 1.f;
      v[k] = BWD ? (in ? to_f32(gp[e]) : 0.f) : x[k];
      ss += x[k] * x[k];
    }
    float r = 1.f;
    if (norm) r = rsqrtf(wave_reduce_sum(ss) * inv_hd + a.eps);
    if (!BWD && norm)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= r * w[k];
    if (a.rot) {
#pragma unroll
      for (int k = 0; k < 4; ++k) buf[wave][lane + 64 * k] = v[k];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        int e = lane + 64 * k;
        if (e < a.rot) {
          bool first = inter ? !(e & 1) : e < half;
          int ang = inter ? e / 2 : (first ? e : e - half);
          int o = inter ? e ^ 1 : (first ? e + half : e - half);
          float c = __uint_as_float(0x7fc00000u), s = c;
          if (pos >= 0) {
            c = a.cos[(long)pos * half + ang];
            s = a.sin[(long)pos * half + ang];
          }
          v[k] = v[k] * c + buf[wave][o] * (first != BWD ? -s : s);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (BWD && norm) {
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) dot += x[k] * v[k] * w[k];
      float f = r * r * wave_reduce_sum(dot) * inv_hd;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float gx = v[k] * (x[k] * r);
        acc[0][k] += isk ? 0.f : gx;
        acc[1][k] += isk ? gx : 0.f;
        v[k] = r * (v[k] * w[k] - x[k] * f);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int e = lane + 64 * k;
      if (e < a.hd) yp[e] = from_f32<T>(v[k]);
    }
  }
  if (!BWD || !norm) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    red[wave][0][lane + 64 * k] = acc[0][k];
    red[wave][1][lane + 64 * k] = acc[1][k];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.hd; e += 256) {
    int k = e >= a.hd, col = e - k * a.hd;
    part[(long)blockIdx.x * 2 * a.hd + e] =
        (red[0][k][col] + red[1][k][col]) + (red[2][k][col] + red[3][k][col]);
  }
}

// dw[e] = sum over rows of part[row][e]; 16 columns x 16 row slices a block
__global__ __launch_bounds__(256) void qknorm_dw_k(
    const float* __restrict__ part, int rows, int cols, int hd,
    float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float red[16][17];
  int c = threadIdx.x & 15, sl = threadIdx.x >> 4;
  int e = blockIdx.x * 16 + c;
  float s = 0.f;
  if (e < cols) {
#pragma unroll 16
    for (int r = sl; r < rows; r += 16) s += part[(long)r * cols + e];
  }
  red[sl][c] = s;
  __syncthreads();
  if (sl == 0 && e < cols) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][c];
    if (e < hd)
      dwq[e] = s;
    else
      dwk[e - hd] = s;
  }
}

constexpr int kBwdBlocks = 1024;  // 4 a CU, what the registers let run

template <typename T, int G>
void launch_vec(const Args& a, int inter, int bwd, float* part, int blocks,
                hipStream_t s) {
  if (bwd) {
    if (inter)
      qknorm_bwd_k<T, G, true><<<blocks, 256, 0, s>>>(a, part);
    else
      qknorm_bwd_k<T, G, false><<<blocks, 256, 0, s>>>(a, part);
  } else {
    if (inter)
      qknorm_fwd_k<T, G, true><<<blocks, 256, 0, s>>>(a);
    else
      qknorm_fwd_k<T, G, false><<<blocks, 256, 0, s>>>(a);
  }
}

}  // namespace

extern "C" {

// rows of `part` that backward needs (each 2*hd floats)
int pdta_qknorm_rows(long tokens, int nv, int vec) {
  long units = vec ? tokens : tokens * nv;
  long blocks = (units + 3) / 4;
  return (int)(blocks < kBwdBlocks ? blocks : kBwdBlocks);
}

// Two tensors (queries, keys): x, dy and y pointers and element strides (b,
// s, head). vec: hd a multiple of 8 up to 256, rot a
// multiple of 8 (16 for halves), strides multiples of 8 and all pointers
// 16-byte aligned; else hd up to 256 and rot even. bwd: y is dx, part holds
// pdta_qknorm_rows rows and dwq, dwk [hd] are written (norm only).
void pdta_qknorm(const void* const* x, const long* xs, const void* const* dy,
                 const long* gs, const float* const* w, void* const* y,
                 const long* ys, const int* heads, const float* cos, const float* sin,
                 const void* pos, int pos32, int npos, int rot, int hd,
                 long b, long s_len, float eps, int inter, int vec, int bwd,
                 float* part, float* dwq, float* dwk, int dt, hipStream_t s) {
  Args a;
  for (int k = 0; k < 2; ++k)
    a.t[k] = {x[k], xs[3 * k], xs[3 * k + 1], xs[3 * k + 2],
              dy[k], gs[3 * k], gs[3 * k + 1], gs[3 * k + 2],
              w[k], y[k], ys[3 * k], ys[3 * k + 1], ys[3 * k + 2],
              heads[k]};
  a.cos = cos, a.sin = sin, a.pos = pos, a.pos32 = pos32, a.npos = npos;
  a.rot = rot, a.hd = hd, a.s = (int)s_len, a.tokens = (int)(b * s_len);
  a.eps = eps, a.slices = 1;
  int nv = heads[0] + heads[1];
  if (a.tokens == 0 || nv == 0) return;
  int blocks = pdta_qknorm_rows(a.tokens, nv, vec);
  if (vec) {
    int G = 4;
    while (G * 8 < hd) G *= 2;
    if (!bwd) {
      // a wave a token; where that leaves the chip empty, its heads are
      // shared out
      int most = (nv + 64 / G - 1) / (64 / G);
      long want = (2048 + a.tokens - 1) / a.tokens;
      a.slices = (int)(want < most ? want : most);
      blocks = (int)(((long)a.tokens * a.slices + 3) / 4);
    }
    PDTA_DISPATCH_DTYPE(dt, T, {
      if (G == 4)
        launch_vec<T, 4>(a, inter, bwd, part, blocks, s);
      else if (G == 8)
        launch_vec<T, 8>(a, inter, bwd, part, blocks, s);
      else if (G == 16)
        launch_vec<T, 16>(a, inter, bwd, part, blocks, s);
      else
        launch_vec<T, 32>(a, inter, bwd, part, blocks, s);
    });
  } else {
    PDTA_DISPATCH_DTYPE(dt, T, {
      if (bwd)
        qknorm_any_k<T, true><<<blocks, 256, 0, s>>>(a, inter, part);
      else
        qknorm_any_k<T, false><<<blocks, 256, 0, s>>>(a, inter, part);
    });
  }
  if (bwd && w[0])
    qknorm_dw_k<<<(2 * hd + 15) / 16, 256, 0, s>>>(part, blocks, 2 * hd, hd,
                                                   dwq, dwk);
}

}  // extern "C"
