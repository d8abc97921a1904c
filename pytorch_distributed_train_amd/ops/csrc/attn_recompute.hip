// Attention whose backward recomputes the probabilities: nothing of size
// sq x sk is ever written.
//
//   S = scale Q K^T;  P = exp(S - lse);  O = P V
//   D = rowsum(dO * O);  dV = P^T dO;  dP = dO V^T;  dS = P * (dP - D)
//   dQ = scale dS K;  dK = scale dS^T Q
// Query i of a sequence sees key j if i < q_len, j < kv_len and, when causal,
// j <= i + kv_len - q_len (the last query sees the last key). A row that sees
// no key gives 0 and takes no gradient (its lse is +inf, so P is 0).
//
// Heads: the g = h / hk query heads of one key head are g rows a position,
// row r = position * g + head. Every kernel works on those packed rows, so a
// key head's tiles serve all of its query heads and dK, dV sum over them in
// registers, in a fixed order.
//
// Layout: 32x32x16 MFMA. Each wave keeps 32 rows (or keys) on the lanes: the
// product that makes S is taken with the kept side as the B operand, so a
// lane holds one row's scores in its accumulators, 16 of every 32 keys, and
// the other half sits 32 lanes away. Row maxima and sums are then loops over
// a lane's registers. Packed to 16 bits, the same registers ARE the B operand
// of the next product (its k index runs over the keys in the order that the
// accumulators hold them, and the A operand is fetched from LDS in that
// order): P and dS never pass through LDS. The other operands stream through
// LDS tiles of 64 rows, two buffers deep, filled by global-to-LDS loads;
// lanes outside a sequence or past the head's end fetch zeros, so nothing
// behind a sequence is ever read.
//
// LDS rows are 128 or 256 bytes; 16-byte chunk c of row r lies at
// c ^ perm(r), perm(r) = r's bits (1,0,2): 8 neighbouring rows spread over
// all banks both for row fragments (16 bytes of one row a lane) and for the
// transposing reads, whose 4 rows x 32 bytes need different chunk pairs.
#include "common.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int TILE = 64;  // streamed rows a step

template <typename T> struct Op;
template <> struct Op<__hip_bfloat16> {
  static DEV_INLINE f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
  }
  static DEV_INLINE unsigned pack(float a, float b) {
    f32x2 f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, bf16x2));
  }
};
template <> struct Op<__half> {
  static DEV_INLINE f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
        0);
  }
  static DEV_INLINE unsigned pack(float a, float b) {
    f32x2 f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, f16x2));
  }
};

struct View {  // [b, s, heads, hd] of a 16-bit type, strides in elements
  const void* p;
  long sb, ss, sh;
  bool quick;  // see Stream
};

struct Args {
  View q, k, v, dout;
  void *out, *dq, *dk, *dv;    // contiguous; out is read by backward
  float *lse, *delta;          // [b, hk, sq*g]; lse in base 2 of scaled scores
  const void *q_lens, *kv_lens;  // [b] int32 / int64, or null
  int lens64;
  int b, sq, sk, hk, g, hd, causal;
  unsigned g_mul;
  int g_shift;
  float scale;
};

__device__ const uint4 kZeros = {0, 0, 0, 0};
__device__ const float kInf = INFINITY;

DEV_INLINE int length_of(const void* lens, int wide, int b, int most) {
  if (!lens) return most;
  long n = wide ? reinterpret_cast<const long*>(lens)[b]
                : (long)reinterpret_cast<const int*>(lens)[b];
  return n < 0 ? 0 : n > most ? most : (int)n;
}

// one block's sequence and key head
struct Seq {
  int batch, kvh, qlen, klen, off;  // off = klen - qlen
  int rows;                         // qlen * g
  DEV_INLINE Seq(const Args& a, int bh) {
    batch = bh / a.hk;
    kvh = bh - batch * a.hk;
    qlen = length_of(a.q_lens, a.lens64, batch, a.sq);
    klen = length_of(a.kv_lens, a.lens64, batch, a.sk);
    off = klen - qlen;
    rows = qlen * a.g;
  }
};

// Block index -> sequence and head, block of it, and part. Causal: all heads'
// longest blocks first (LAST: high indexes are long). Else 8 heads at a time.
// Either way a head's blocks are 8 (or bh) apart, and as the hardware deals
// blocks out to its 8 dies in turn, they meet in one die's L2.
DEV_INLINE void place(const Args& a, int nblk, bool last, int* bh, int* blk) {
  int heads = a.b * a.hk, i = blockIdx.x;
  if (a.causal) {
    *blk = i / heads;
    *bh = i - *blk * heads;
    if (last) *blk = nblk - 1 - *blk;
  } else {
    int grp = i / (8 * nblk), w = i - grp * 8 * nblk;
    int n = heads - grp * 8;
    n = n < 8 ? n : 8;
    *blk = w / n;
    *bh = grp * 8 + w - *blk * n;
  }
}

template <int HDT> struct Geo {
  static constexpr int NCH = HDT == 64 ? 8 : 16;  // chunks of an LDS row
  static constexpr int PITCH = NCH * 16;
  static constexpr int KS = HDT / 16;  // k steps of a product over the head
  static constexpr int DT = HDT / 32;  // 32-column tiles of the head
};

DEV_INLINE int perm(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

// A or B operand whose k runs along the row: rows r0 + (lane & 31), elements
// 16*ks + 8*(lane >> 5) + 0..7
template <int HDT>
DEV_INLINE s16x8 frag_row(const char* lds, int r0, int ks, int lane) {
  return *reinterpret_cast<const s16x8*>(
      lds + (r0 + (lane & 31)) * Geo<HDT>::PITCH +
      (((2 * ks + (lane >> 5)) ^ perm(lane)) << 4));
}

// A operand whose k runs down the rows, in the accumulators' order: column
// 32*dt + (lane & 31), rows r0 + 4*h + 0..3 and r0 + 8 + 4*h + 0..3 with
// h = lane >> 5. The transposing read hands each lane of 16 one column of
// the 4 x 16 block that the 16 lanes fetch in 8-byte pieces.
template <int HDT>
DEV_INLINE s16x8 frag_col(const char* lds, int r0, int dt, int lane) {
  int row = 4 * (lane >> 5) + ((lane >> 2) & 3);
  int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1);
  const char* p = lds + (r0 + row) * Geo<HDT>::PITCH +
                  ((chunk ^ perm(row)) << 4) + (lane & 1) * 8;
  typedef __attribute__((address_space(3))) s16x4* tp_t;
  s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tp_t)p);
  s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (tp_t)(p + 8 * Geo<HDT>::PITCH));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Global to LDS: lane l's 16 (4) bytes land at dst + 16 (4) * l. In assembly
// and not by the builtin, since the compiler would make LDS reads of the other
// buffer wait for these loads; staged() waits for them. They have no output
// register, and an uncounted load in flight only makes the compiler's own
// waits longer.
DEV_INLINE unsigned lds_base(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
DEV_INLINE void to_lds16(const void* src, void* dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
      :
      : "v"(src), "s"(lds_base(dst))
      : "memory", "m0");
}
// from the wave's `base` plus the lane's 32-bit offset
DEV_INLINE void to_lds16(const void* base, unsigned off, void* dst) {
  asm volatile(
      "s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
      :
      : "v"(off), "s"(base), "s"(lds_base(dst))
      : "memory", "m0");
}
DEV_INLINE void to_lds4(const void* src, void* dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
      :
      : "v"(src), "s"(lds_base(dst))
      : "memory", "m0");
}

// A streamed operand: rows r0.. below `end` of one sequence and head go to
// LDS in tiles of R rows, by 4 waves. PACKED: row r is position r / g of head
// r % g, else position r. A wave's load moves RPI = 4 or 8 rows. In a whole
// tile their addresses are a scalar base and a lane's offset that never
// changes (`quick`: RPI rows must not straddle positions unevenly, so g
// divides RPI or RPI g); lanes past the head's end fetch its first chunk,
// whose partner in the product is 0 or whose result is not stored. The last
// tile works out each lane's row and fetches zeros beyond the end.
template <int HDT, int R, bool PACKED>
struct Stream {
  static constexpr int NCH = Geo<HDT>::NCH, RPI = 64 / NCH, N = R / RPI / 4;
  static_assert(N > 0 && (NCH == 8 || N % 2 == 0), "pieces a wave");
  const char* base;
  long ss, sh;
  unsigned off[2];  // even and odd pieces (their rows' perm differs)
  bool quick;

  DEV_INLINE Stream(const Args& a, const View& v, const Seq& s, int lane) {
    ss = v.ss, sh = v.sh;
    base = reinterpret_cast<const char*>(v.p) +
           2 * (s.batch * v.sb + (long)s.kvh * (PACKED ? a.g : 1) * sh);
    quick = v.quick;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int l = lane / NCH;
      int chunk = (lane % NCH) ^ perm(NCH == 8 ? l : l + 4 * k);
      if (chunk * 8 >= a.hd) chunk = 0;
      long at = PACKED ? (l / a.g) * ss + (l % a.g) * sh : l * ss;
      off[k] = (unsigned)(2 * at) + chunk * 16;
    }
  }

  DEV_INLINE void load(const Args& a, int r0, int end, char* lds, int wave,
                       int lane) const {
    if (quick && r0 + R <= end) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int idx = wave * N + i, x = r0 + idx * RPI;
        long at;
        if (PACKED) {
          int pos = (int)mdiv(x, a.g_mul, a.g_shift);
          at = pos * ss + (x - pos * a.g) * sh;
        } else {
          at = x * ss;
        }
        to_lds16(base + 2 * at, off[NCH == 8 ? 0 : i & 1], lds + idx * 1024);
      }
      return;
    }
    asm volatile("" : "+v"(lane));  // keeps this out of the loop's registers
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int idx = wave * N + i;
      int row = idx * RPI + lane / NCH;
      int chunk = (lane % NCH) ^ perm(row);
      int r = r0 + row;
      long at;
      if (PACKED) {
        int pos = (int)mdiv(r, a.g_mul, a.g_shift);
        at = pos * ss + (r - pos * a.g) * sh;
      } else {
        at = r * ss;
      }
      const char* src = base + 2 * at + chunk * 16;
      if (r >= end || chunk * 8 >= a.hd)
        src = reinterpret_cast<const char*>(&kZeros);
      to_lds16(src, lds + idx * 1024);
    }
  }
};

// the lane's row of a kept operand, in registers
template <int HDT>
DEV_INLINE void keep(const Args& a, const char* row, bool valid, int lane,
                     s16x8* f) {
#pragma unroll
  for (int ks = 0; ks < Geo<HDT>::KS; ++ks) {
    int e = ks * 16 + (lane >> 5) * 8;
    s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
    f[ks] = valid && e < a.hd
                ? *reinterpret_cast<const s16x8*>(row + 2 * e)
                : z;
  }
}

// accumulators acc[DT] (lane: one row, d = 32*dt + 8*j + 4*h + 0..3) times m
// to the row's memory, 8 bytes a piece
template <typename T, int DT>
DEV_INLINE void put_row(T* row, const f32x16* acc, float m, int hd, int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int d = dt * 32 + j * 8 + (lane >> 5) * 4;
      if (d < hd) {
        uint2 v = {Op<T>::pack(acc[dt][4 * j] * m, acc[dt][4 * j + 1] * m),
                   Op<T>::pack(acc[dt][4 * j + 2] * m,
                               acc[dt][4 * j + 3] * m)};
        *reinterpret_cast<uint2*>(row + d) = v;
      }
    }
}

DEV_INLINE float other_half(float x) { return __shfl_xor(x, 32, 64); }

DEV_INLINE s16x8 pack8(const unsigned* p) {
  uint4 v = {p[0], p[1], p[2], p[3]};
  return __builtin_bit_cast(s16x8, v);
}

// Buffers are arrays of their own and steps come in pairs that name them: a
// read of one buffer then provably does not wait for the loads in flight to
// the other (as one array indexed by step & 1, every step waited for the next
// one's loads).
#define LDS_BUFFER(name, bytes) \
  __shared__ __attribute__((aligned(16))) char name[bytes]

DEV_INLINE void staged() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

DEV_INLINE int wave_min(int x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    int o = __shfl_xor(x, m, 64);
    x = x < o ? x : o;
  }
  return __builtin_amdgcn_readfirstlane(x);
}
DEV_INLINE int wave_max(int x) { return -wave_min(-x); }

constexpr f32x16 kNone = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

// a lane's row of the packed rows and how many keys it sees
struct Row {
  int r, pos, head, lim;
  bool valid, stored;
  DEV_INLINE Row(const Args& a, const Seq& s, int row) {
    r = row;
    pos = (int)mdiv(r, a.g_mul, a.g_shift);
    head = s.kvh * a.g + (r - pos * a.g);
    stored = pos < a.sq;
    valid = pos < s.qlen;
    lim = s.klen;
    if (a.causal && valid) {
      lim = pos + s.off + 1;
      lim = lim < 0 ? 0 : lim;  // pos < qlen keeps it <= klen
    }
  }
};

// ---- forward: a block has 128 packed rows, a wave 32 ----------------------
template <typename T, int HDT>
__global__ __launch_bounds__(256, 2) void attn_rc_fwd_k(Args a, int nblk) {
  using G = Geo<HDT>;
  LDS_BUFFER(k0, TILE * G::PITCH);
  LDS_BUFFER(k1, TILE * G::PITCH);
  LDS_BUFFER(v0, TILE * G::PITCH);
  LDS_BUFFER(v1, TILE * G::PITCH);
  int lane = threadIdx.x & 63, h = lane >> 5;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk;
  place(a, nblk, true, &bh, &blk);
  Seq s(a, bh);
  Row row(a, s, blk * 128 + wave * 32 + (lane & 31));
  Stream<HDT, TILE, false> kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  s16x8 qf[G::KS];
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.q.p) +
                2 * (s.batch * a.q.sb + row.pos * a.q.ss + row.head * a.q.sh),
            row.valid, lane, qf);
  // keys that any row of the block sees: the last row's, or none
  int last = (blk * 128 + 127) / a.g;
  last = last < s.qlen ? last : s.qlen - 1;
  int end = blk * 128 < s.rows ? s.klen : 0;
  if (a.causal && last + s.off + 1 < end) end = last + s.off + 1;
  int ntile = end > 0 ? (end + TILE - 1) / TILE : 0;
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);

  float c = a.scale * kLog2e, far = 8.f / c;
  float top = -INFINITY, sum = 0.f;
  f32x16 acc[G::DT];
#pragma unroll
  for (int i = 0; i < G::DT; ++i) acc[i] = kNone;

  auto load = [&](int t, char* kd, char* vd) {
    kin.load(a, t * TILE, s.klen, kd, wave, lane);
    vin.load(a, t * TILE, s.klen, vd, wave, lane);
  };
  auto step = [&](int t, const char* kt, const char* vt) {
    int key0 = t * TILE;
    if (key0 >= whi) return;
    f32x16 sc[2] = {kNone, kNone};
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        sc[u] = Op<T>::mfma(frag_row<HDT>(kt, u * 32, ks, lane), qf[ks],
                            sc[u]);
    if (key0 + TILE > wlo) {
      int rel = row.lim - key0 - h * 4;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if ((i >> 2) * 8 + (i & 3) >= rel) sc[i >> 4][i & 15] = -INFINITY;
    }
    float m = sc[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) m = fmaxf(m, sc[i >> 4][i & 15]);
    m = fmaxf(m, other_half(m));
    // P is taken relative to `top`, which follows the running maximum only
    // when that is 2^8 past it: P stays below 2^8, which neither 16-bit type
    // minds, and most steps rescale nothing
    bool up = m > top + far;
    if (__any(up)) {
      float f = up ? __builtin_amdgcn_exp2f((top - m) * c) : 1.f;
      top = up ? m : top;
      sum *= f;
#pragma unroll
      for (int i = 0; i < G::DT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] *= f;
    }
    float base = top == -INFINITY ? 0.f : -top * c;
    unsigned p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = __builtin_amdgcn_exp2f(
          fmaf(sc[i >> 3][(2 * i) & 15], c, base));
      float y = __builtin_amdgcn_exp2f(
          fmaf(sc[i >> 3][(2 * i + 1) & 15], c, base));
      sum += x + y;
      p[i] = Op<T>::pack(x, y);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < G::DT; ++i)
        acc[i] = Op<T>::mfma(frag_col<HDT>(vt, k * 16, i, lane),
                             pack8(p + 4 * k), acc[i]);
  };
  if (ntile) load(0, k0, v0);
  staged();
  for (int t = 0; t < ntile; t += 2) {
    if (t + 1 < ntile) load(t + 1, k1, v1);
    step(t, k0, v0);
    staged();
    if (t + 1 >= ntile) break;
    if (t + 2 < ntile) load(t + 2, k0, v0);
    step(t + 1, k1, v1);
    staged();
  }
  sum += other_half(sum);
  if (!row.stored) return;
  bool some = row.valid && row.lim > 0;
  T* o = reinterpret_cast<T*>(a.out) +
         (((long)s.batch * a.sq + row.pos) * a.hk * a.g + row.head) * a.hd;
  if (!some)
#pragma unroll
    for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  put_row<T, G::DT>(o, acc, some ? 1.f / sum : 0.f, a.hd, lane);
  if (h == 0 && a.lse)
    a.lse[(long)bh * a.sq * a.g + row.r] =
        some ? top * c + __builtin_amdgcn_logf(sum) : INFINITY;
}

// ---- backward 1: D, and dQ of 128 packed rows -----------------------------
template <typename T, int HDT>
__global__ __launch_bounds__(256, 2) void attn_rc_dq_k(Args a, int nblk) {
  using G = Geo<HDT>;
  LDS_BUFFER(k0, TILE * G::PITCH);
  LDS_BUFFER(k1, TILE * G::PITCH);
  LDS_BUFFER(v0, TILE * G::PITCH);
  LDS_BUFFER(v1, TILE * G::PITCH);
  int lane = threadIdx.x & 63, h = lane >> 5;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk;
  place(a, nblk, true, &bh, &blk);
  Seq s(a, bh);
  Row row(a, s, blk * 128 + wave * 32 + (lane & 31));
  Stream<HDT, TILE, false> kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  int last = (blk * 128 + 127) / a.g;
  last = last < s.qlen ? last : s.qlen - 1;
  int end = blk * 128 < s.rows ? s.klen : 0;
  if (a.causal && last + s.off + 1 < end) end = last + s.off + 1;
  int ntile = end > 0 ? (end + TILE - 1) / TILE : 0;
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);
  auto load = [&](int t, char* kd, char* vd) {
    kin.load(a, t * TILE, s.klen, kd, wave, lane);
    vin.load(a, t * TILE, s.klen, vd, wave, lane);
  };
  if (ntile) load(0, k0, v0);
  s16x8 qf[G::KS], df[G::KS];
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.dout.p) +
                2 * (s.batch * a.dout.sb + row.pos * a.dout.ss +
                     row.head * a.dout.sh),
            row.valid, lane, df);
  long oat = (((long)s.batch * a.sq + row.pos) * a.hk * a.g + row.head) *
             a.hd;
  // D from the stored output: its rounding moves dS by P times a sum of
  // random half steps, below dS's own rounding
  keep<HDT>(a, reinterpret_cast<const char*>(a.out) + 2 * oat, row.valid,
            lane, qf);
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      T x = __builtin_bit_cast(T, (short)qf[ks][i]);
      T y = __builtin_bit_cast(T, (short)df[ks][i]);
      delta += to_f32(x) * to_f32(y);
    }
  delta += other_half(delta);
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.q.p) +
                2 * (s.batch * a.q.sb + row.pos * a.q.ss + row.head * a.q.sh),
            row.valid, lane, qf);
  float lse = INFINITY;
  long lat = (long)bh * a.sq * a.g + row.r;
  if (row.valid) lse = a.lse[lat];
  if (row.stored && h == 0) a.delta[lat] = delta;

  float c = a.scale * kLog2e;
  f32x16 acc[G::DT];
#pragma unroll
  for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  auto step = [&](int t, const char* kt, const char* vt) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int key0 = t * TILE + u * 32;
      if (key0 >= whi) return;
      f32x16 sc = kNone, dp = kNone;
#pragma unroll
      for (int ks = 0; ks < G::KS; ++ks) {
        sc = Op<T>::mfma(frag_row<HDT>(kt, u * 32, ks, lane), qf[ks], sc);
        dp = Op<T>::mfma(frag_row<HDT>(vt, u * 32, ks, lane), df[ks], dp);
      }
      if (key0 + 32 > wlo) {
        int rel = row.lim - key0 - h * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((i >> 2) * 8 + (i & 3) >= rel) sc[i] = -INFINITY;
      }
      unsigned p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = __builtin_amdgcn_exp2f(fmaf(sc[2 * i], c, -lse)) *
                  (dp[2 * i] - delta);
        float y = __builtin_amdgcn_exp2f(fmaf(sc[2 * i + 1], c, -lse)) *
                  (dp[2 * i + 1] - delta);
        p[i] = Op<T>::pack(x, y);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < G::DT; ++i)
          acc[i] = Op<T>::mfma(frag_col<HDT>(kt, u * 32 + k * 16, i, lane),
                               pack8(p + 4 * k), acc[i]);
    }
  };
  staged();
  for (int t = 0; t < ntile; t += 2) {
    if (t + 1 < ntile) load(t + 1, k1, v1);
    step(t, k0, v0);
    staged();
    if (t + 1 >= ntile) break;
    if (t + 2 < ntile) load(t + 2, k0, v0);
    step(t + 1, k1, v1);
    staged();
  }
  if (!row.stored) return;
  bool some = row.valid && row.lim > 0;
  if (!some)
#pragma unroll
    for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  put_row<T, G::DT>(reinterpret_cast<T*>(a.dq) + oat, acc, a.scale, a.hd,
                    lane);
}

// ---- backward 2: dK, dV of 128 keys, over all packed rows -----------------
// Kept in registers: the wave's 32 keys' K, and dK, dV (64 each at a head of
// 128). V as well would spill there, so from heads of 96 on it stays in LDS
// and rows stream 32 at a time to leave room for two blocks a CU.
// With few key blocks the rows are dealt out to `nsplit` blocks in turn
// (tile t to block t % nsplit), whose fp32 sums a last kernel adds.
template <typename T, int HDT>
__global__ __launch_bounds__(256, 2) void attn_rc_dkv_k(Args a, int nblk,
                                                        int nsplit,
                                                        float* part) {
  using G = Geo<HDT>;
  constexpr bool VLDS = HDT > 64;
  constexpr int RT = VLDS ? 32 : 64;
  LDS_BUFFER(q0, RT * G::PITCH);
  LDS_BUFFER(q1, RT * G::PITCH);
  LDS_BUFFER(d0, RT * G::PITCH);
  LDS_BUFFER(d1, RT * G::PITCH);
  LDS_BUFFER(stat0, 512);  // 64 rows' lse and D
  LDS_BUFFER(stat1, 512);
  LDS_BUFFER(vkeep, VLDS ? 128 * G::PITCH : 16);
  int lane = threadIdx.x & 63, h = lane >> 5;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk;
  place(a, nblk * nsplit, false, &bh, &blk);
  int split = blk % nsplit;
  blk /= nsplit;
  Seq s(a, bh);
  int key = blk * 128 + wave * 32 + (lane & 31);
  bool valid = key < s.klen;
  Stream<HDT, RT, true> qin(a, a.q, s, lane), din(a, a.dout, s, lane);
  const char* kb = reinterpret_cast<const char*>(a.k.p) +
                   2 * (s.batch * a.k.sb + s.kvh * a.k.sh);
  const char* vb = reinterpret_cast<const char*>(a.v.p) +
                   2 * (s.batch * a.v.sb + s.kvh * a.v.sh);
  const float* lse = a.lse + (long)bh * a.sq * a.g;
  const float* del = a.delta + (long)bh * a.sq * a.g;
  // rows from `lo` on see this lane's key
  int lo = 0;
  if (a.causal) lo = key > s.off ? (key - s.off) * a.g : 0;
  int first = 0;
  if (a.causal && blk * 128 > s.off) first = (blk * 128 - s.off) * a.g;
  first &= ~(RT - 1);
  int ntile = 0;
  if (blk * 128 < s.klen && first < s.rows)
    ntile = (s.rows - first + RT - 1) / RT;
  int wlo = wave_min(lo), whi = wave_max(valid ? lo : 0);
  bool wlive = wave_max(valid) != 0;

  auto load = [&](int t, char* qd, char* dd, char* sd) {
    int r0 = first + t * RT;
    qin.load(a, r0, s.rows, qd, wave, lane);
    din.load(a, r0, s.rows, dd, wave, lane);
    if (wave < 2) {
      bool in = r0 + lane < s.rows;
      const float* src = wave ? (in ? del + r0 + lane
                                    : reinterpret_cast<const float*>(&kZeros))
                              : (in ? lse + r0 + lane : &kInf);
      to_lds4(src, sd + wave * 256);
    }
  };
  s16x8 kf[G::KS], vf[VLDS ? 1 : G::KS];
  if (split < ntile) {
    load(split, q0, d0, stat0);
    if (VLDS) {
      Stream<HDT, 128, false> vin(a, a.v, s, lane);
      vin.quick = false;  // zeros past the head's end: dO has none there
      vin.load(a, blk * 128, s.klen, vkeep, wave, lane);
    }
  }
  keep<HDT>(a, kb + 2 * (key * a.k.ss), valid, lane, kf);
  if (!VLDS) keep<HDT>(a, vb + 2 * (key * a.v.ss), valid, lane, vf);
  float c = a.scale * kLog2e;
  f32x16 dk[G::DT], dv[G::DT];
#pragma unroll
  for (int i = 0; i < G::DT; ++i) dk[i] = dv[i] = kNone;
  auto step = [&](int t, const char* qt, const char* dt, const char* sd) {
    const float* ls = reinterpret_cast<const float*>(sd);
    const float* ds = ls + 64;
#pragma unroll
    for (int u = 0; u < RT / 32; ++u) {
      int r0 = first + t * RT + u * 32;
      if (!wlive || r0 + 32 <= wlo || r0 >= s.rows) continue;
      f32x16 sc = kNone, dp = kNone;
#pragma unroll
      for (int ks = 0; ks < G::KS; ++ks) {
        sc = Op<T>::mfma(frag_row<HDT>(qt, u * 32, ks, lane), kf[ks], sc);
        dp = Op<T>::mfma(frag_row<HDT>(dt, u * 32, ks, lane),
                         VLDS ? frag_row<HDT>(vkeep, wave * 32, ks, lane)
                              : vf[VLDS ? 0 : ks],
                         dp);
      }
      if (r0 < whi) {
        int rel = lo - r0 - h * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((i >> 2) * 8 + (i & 3) < rel) sc[i] = -INFINITY;
      }
      unsigned p[8], d[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 l4 =
            *reinterpret_cast<const float4*>(ls + u * 32 + j * 8 + h * 4);
        float4 d4 =
            *reinterpret_cast<const float4*>(ds + u * 32 + j * 8 + h * 4);
        const float *lp = &l4.x, *dl = &d4.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i], c, -lp[2 * i]));
          float y = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i + 1], c, -lp[2 * i + 1]));
          p[2 * j + i] = Op<T>::pack(x, y);
          d[2 * j + i] =
              Op<T>::pack(x * (dp[4 * j + 2 * i] - dl[2 * i]),
                          y * (dp[4 * j + 2 * i + 1] - dl[2 * i + 1]));
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < G::DT; ++i) {
          dv[i] = Op<T>::mfma(frag_col<HDT>(dt, u * 32 + k * 16, i, lane),
                              pack8(p + 4 * k), dv[i]);
          dk[i] = Op<T>::mfma(frag_col<HDT>(qt, u * 32 + k * 16, i, lane),
                              pack8(d + 4 * k), dk[i]);
        }
    }
  };
  staged();
  for (int t = split; t < ntile; t += 2 * nsplit) {
    int t1 = t + nsplit, t2 = t1 + nsplit;
    if (t1 < ntile) load(t1, q1, d1, stat1);
    step(t, q0, d0, stat0);
    staged();
    if (t1 >= ntile) break;
    if (t2 < ntile) load(t2, q0, d0, stat0);
    step(t1, q1, d1, stat1);
    staged();
  }
  if (key >= a.sk) return;
  if (!valid)
#pragma unroll
    for (int i = 0; i < G::DT; ++i) dk[i] = dv[i] = kNone;
  long at = (((long)s.batch * a.sk + key) * a.hk + s.kvh) * a.hd;
  if (nsplit == 1) {
    put_row<T, G::DT>(reinterpret_cast<T*>(a.dv) + at, dv, 1.f, a.hd, lane);
    put_row<T, G::DT>(reinterpret_cast<T*>(a.dk) + at, dk, a.scale, a.hd,
                      lane);
    return;
  }
  long n = (long)a.b * a.sk * a.hk * a.hd;
  float* out = part + 2 * split * n + at;
#pragma unroll
  for (int i = 0; i < G::DT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int e = i * 32 + j * 8 + h * 4;
      if (e < a.hd) {
        *reinterpret_cast<float4*>(out + e) = {dk[i][4 * j], dk[i][4 * j + 1],
                                               dk[i][4 * j + 2],
                                               dk[i][4 * j + 3]};
        *reinterpret_cast<float4*>(out + n + e) = {
            dv[i][4 * j], dv[i][4 * j + 1], dv[i][4 * j + 2],
            dv[i][4 * j + 3]};
      }
    }
}

// dk, dv = sums over the splits' part[split][2][n], 4 elements a thread
template <typename T>
__global__ __launch_bounds__(256) void attn_rc_join_k(
    const float* __restrict__ part, long n, int nsplit, float scale,
    T* __restrict__ dk, T* __restrict__ dv) {
  long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= 2 * n) return;
  float4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < nsplit; ++k) {
    float4 x = *reinterpret_cast<const float4*>(part + 2 * k * n + i);
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  float m = i < n ? scale : 1.f;
  uint2 v = {Op<T>::pack(sum.x * m, sum.y * m),
             Op<T>::pack(sum.z * m, sum.w * m)};
  *reinterpret_cast<uint2*>(i < n ? dk + i : dv + (i - n)) = v;
}

// Blocks that share a key block's rows. Two blocks run on each of 256 CUs;
// below four rounds of them (a causal mask's blocks differ in length) rows
// are dealt out, 512 at least to each.
int dkv_splits(long b, long sq, long sk, long hk, long g) {
  long blocks = b * hk * ((sk + 127) / 128), rows = sq * g;
  if (blocks == 0) return 1;
  long n = (2048 + blocks - 1) / blocks;
  if (n > rows / 512) n = rows / 512;
  if (n > 16) n = 16;
  return n < 1 ? 1 : (int)n;
}

template <typename T, int HDT>
void launch(const Args& a, int bwd, float* part, hipStream_t s) {
  int rblk = (a.sq * a.g + 127) / 128, kblk = (a.sk + 127) / 128;
  int bh = a.b * a.hk;
  if (!bwd) {
    if (rblk) attn_rc_fwd_k<T, HDT><<<bh * rblk, 256, 0, s>>>(a, rblk);
    return;
  }
  if (rblk) attn_rc_dq_k<T, HDT><<<bh * rblk, 256, 0, s>>>(a, rblk);
  if (!kblk) return;
  int nsplit = dkv_splits(a.b, a.sq, a.sk, a.hk, a.g);
  attn_rc_dkv_k<T, HDT><<<bh * kblk * nsplit, 256, 0, s>>>(a, kblk, nsplit,
                                                           part);
  if (nsplit > 1) {
    long n = (long)a.b * a.sk * a.hk * a.hd;
    attn_rc_join_k<T><<<(n / 2 + 255) / 256, 256, 0, s>>>(
        part, n, nsplit, a.scale, (T*)a.dk, (T*)a.dv);
  }
}

}  // namespace

extern "C" {

// floats of workspace that backward needs
long pdta_attn_recompute_ws(long b, long sq, long sk, long hk, long g,
                            long hd) {
  int n = dkv_splits(b, sq, sk, hk, g);
  return n > 1 ? 2 * n * b * sk * hk * hd : 0;
}

// strides: q, k, v, dout, each (b, s, head) in elements; multiples of 8, all
// pointers 16-byte aligned, hd a multiple of 8 up to 128. lens null or [b].
// Forward writes out and, unless null, lse; backward reads both and writes
// delta, dq, dk, dv, with pdta_attn_recompute_ws floats in ws. Grids must stay below 2^31 blocks and sq*g below 2^31.
void pdta_attn_recompute(const void* q, const void* k, const void* v,
                         const void* dout, const long* st, void* out,
                         float* lse, float* delta, void* dq, void* dk,
                         void* dv, const void* q_lens, const void* kv_lens,
                         int lens64, int b, int sq, int sk, int hk, int g,
                         int hd, float scale, int causal, int bwd,
                         float* ws, int dt, hipStream_t s) {
  Args a;
  int rpi = hd <= 64 ? 8 : 4;  // rows a load moves
  bool even = rpi % g == 0 || g % rpi == 0;
  auto view = [&](const void* x, const long* n, bool packed) {
    long far = 8 * (n[1] + n[2]) + hd;  // a lane's offset, in elements
    return View{x, n[0], n[1], n[2],
                far < (1l << 31) && (!packed || even)};
  };
  a.q = view(q, st, true);
  a.k = view(k, st + 3, false);
  a.v = view(v, st + 6, false);
  a.dout = view(dout, st + 9, true);
  a.out = out, a.dq = dq, a.dk = dk, a.dv = dv, a.lse = lse, a.delta = delta;
  a.q_lens = q_lens, a.kv_lens = kv_lens, a.lens64 = lens64;
  a.b = b, a.sq = sq, a.sk = sk, a.hk = hk, a.g = g, a.hd = hd;
  a.scale = scale, a.causal = causal;
  MagicDiv m = magic_div((unsigned)g);
  a.g_mul = m.mul, a.g_shift = m.shift;
  if (b == 0 || hk == 0) return;
  PDTA_DISPATCH_DTYPE16(dt, T, {
    if (hd <= 64)
      launch<T, 64>(a, bwd, ws, s);
    else if (hd <= 96)
      launch<T, 96>(a, bwd, ws, s);
    else
      launch<T, 128>(a, bwd, ws, s);
  });
}

}  // extern "C"
