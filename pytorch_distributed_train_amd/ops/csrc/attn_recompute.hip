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
// LDS tiles of 64 or 32 rows, two buffers deep, filled by global-to-LDS
// loads; lanes outside a sequence fetch zeros, so nothing behind it is read.
//
// Roundings: scores, softmax statistics, D and all sums are fp32. P and dS
// are rounded to the tensors' type as operands of the second products, half
// a step relative each; summed over keys with random sign that is as much as
// the results' own rounding, and 32-bit operands would leave the matrix
// units. Backward computes P from fp32 scores and lse again, unrounded for
// dS.
//
// What bounds it: 9 products of 2*hd flops a visible pair, where two (S and
// dP again for dK, dV) are the price of no atomics. On long sequences with
// heads of 128 dQ reaches 1150 to 1250 TFLOP/s, dK/dV 1020 to 1100, the
// forward 1030; a large matrix product reaches 1250. Heads of 64 have half
// the products an exponential: 800 to 1000. Splitting differently was slower:
// scores one tile ahead of the softmax (more registers, fewer waves: 0 to
// -25%), 32-key tiles with three blocks a CU (+4% long, -6% short).
//
// LDS rows are 128 or 256 bytes, in groups of 1024 bytes (what one load
// brings) that lie 1056 or 1040 apart; 16-byte chunk c of row r lies at
// c ^ perm(r). The banks span 256 bytes, and a row fragment's read (16 bytes
// of a row a lane) is served 16 lanes at a time, lanes 0-3, 12-15, 20-27 and
// the rest: these rows need 16 different 16-byte places. The transposing
// reads take 64 bytes of 4 neighbouring rows at a time: these need 4
// different 64-byte places. perm puts a row's low bits into the place's high
// bits for the latter, the bytes between groups set the others apart for the
// former, and the way from row to row + 16 stays a constant. Conflicts took
// 16 to 20% of all cycles at heads of 128 when perm alone did this.
#include <cfloat>

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
  long vb, vs, vh;             // but dv has strides of its own
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

DEV_INLINE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

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
    batch = uniform(bh / a.hk);
    kvh = bh - batch * a.hk;
    set(a, length_of(a.q_lens, a.lens64, batch, a.sq),
        length_of(a.kv_lens, a.lens64, batch, a.sk));
  }
  DEV_INLINE Seq(const Args& a, int batch_, int kvh_, int q, int k)
      : batch(batch_), kvh(kvh_) {
    set(a, q, k);
  }
  DEV_INLINE void set(const Args& a, int q, int k) {
    qlen = q, klen = k;
    off = klen - qlen;
    rows = qlen * a.g;
  }
};

template <int CTRL, int ROWS>
DEV_INLINE int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
// running sum over the wave's lanes
DEV_INLINE int wave_scan(int x) {
  x = dpp_add<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes before, in rows of 16
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // a row's last lane to the odd rows
  return dpp_add<0x143, 0xc>(x);  // lane 31 to the upper half
}

// Blocks of sequences with lengths, longest first: block index -> block of
// its head, sequence and head. KEYS: blocks of keys that run over the rows;
// else of rows over the keys. Only the blocks in front of the sequence's end
// have work; the others come last. Blocks go to the 8 dies in turn and there
// to one CU after the other, two each; so a head's blocks stay on a die, and
// the first 32 go there from short to long, so that the long ones share their
// CU with the shortest of the next 32. 16 sequences of 0 to 777 tokens, 10
// heads of 80: forward 34 us, dQ 41, dK/dV 51; in the order of the batch each
// took 6 to 13 us more. A block spends 1.4 us here, the longest 21 on its run.
// Lane l ranks sequence l (b <= 64) and then places head die + 8 l; heads are
// a multiple of 8 up to 512.
template <bool KEYS, int BLOCK>
DEV_INLINE Seq by_length(const Args& a, int nblk, int nsplit, int* bh,
                         int* blk) {
  int lane = threadIdx.x & 63, die = blockIdx.x & 7, at = blockIdx.x >> 3;
  bool in = lane < a.b;
  int ql = in ? length_of(a.q_lens, a.lens64, lane, a.sq) : -1;
  int kl = in ? length_of(a.kv_lens, a.lens64, lane, a.sk) : -1;
  int n = KEYS ? ql : kl, rank = 0;
  // lanes from a.b on hold -1: they are not counted
  for (int j = 0; j < a.b; j += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      rank += __builtin_amdgcn_readlane(n, j + i) >= n + (j + i >= lane);
  int live = ((KEYS ? kl : ql * a.g) + BLOCK - 1) / BLOCK * nsplit;
  live = n > 0 ? live : 0;
  // by rank, then by head
  int x = __builtin_amdgcn_ds_permute((in ? rank : lane) * 4,
                                      live << 6 | lane);
  int j = (die + 8 * lane) / a.hk;
  x = __builtin_amdgcn_ds_bpermute((j & 63) * 4, x);
  int seq = x & 63;
  live = j < a.b ? x >> 6 : 0;
  int upto = wave_scan(live);
  int total = __builtin_amdgcn_readlane(upto, 63);
  if (at < total) {
    int first = total < 32 ? total : 32;
    if (at < first) at = first - 1 - at;
  } else {
    // past the live ones: head by head the blocks behind them
    at -= total;
    upto = nblk * (lane + 1) - upto;
    live = nblk;
  }
  int to = __builtin_ctzll(__ballot(upto > at));
  *blk = at - __builtin_amdgcn_readlane(upto - live, to);
  seq = __builtin_amdgcn_readlane(seq, to);
  int kvh = die + 8 * to - __builtin_amdgcn_readlane(j, to) * a.hk;
  *bh = seq * a.hk + kvh;
  return Seq(a, seq, kvh, __builtin_amdgcn_readlane(ql, seq),
             __builtin_amdgcn_readlane(kl, seq));
}

// Block index -> block and part, sequence and head. Causal: all heads' longest
// blocks first. With lengths: by_length. Else 8 heads at a time. In each case
// a head's blocks are a multiple of 8 (or bh) apart, and as the hardware deals
// blocks out to its 8 dies in turn, they meet in one die's L2.
template <bool KEYS, int BLOCK = 128>
DEV_INLINE Seq place(const Args& a, int nblk, int nsplit, int* bh, int* blk,
                     int* split) {
  int heads = a.b * a.hk, i = blockIdx.x;
  nblk *= nsplit;
  auto parted = [&] {
    int x = *blk;
    *blk = uniform(x / nsplit);
    *split = x - *blk * nsplit;
  };
  if (!a.causal && (KEYS ? a.q_lens : a.kv_lens) && a.b <= 64 &&
      heads <= 512 && heads % 8 == 0) {
    Seq s = by_length<KEYS, BLOCK>(a, nblk, nsplit, bh, blk);
    parted();
    return s;
  }
  if (a.causal) {
    *blk = uniform(i / heads);
    *bh = i - *blk * heads;
    if (!KEYS) *blk = nblk - 1 - *blk;
  } else {
    int grp = uniform(i / (8 * nblk)), w = i - grp * 8 * nblk;
    int n = heads - grp * 8;
    n = n < 8 ? n : 8;
    *blk = uniform(w / n);
    *bh = grp * 8 + w - *blk * n;
  }
  parted();
  return Seq(a, *bh);
}

// zeros to n pieces of 16 * chunks bytes, 32 chunks at most
template <typename F>
DEV_INLINE void clear(int n, int chunks, F piece) {
  int c = threadIdx.x & 31;
  if (c >= chunks) return;
  for (int i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5)
    reinterpret_cast<uint4*>(piece(i))[c] = {0, 0, 0, 0};
}

template <int HDT> struct Geo {
  static constexpr int NCH = HDT == 64 ? 8 : 16;  // chunks of an LDS row
  static constexpr int GROUP = 64 / NCH;          // rows of a group
  static constexpr int SPAN = HDT == 64 ? 1056 : 1040;
  static constexpr int bytes(int rows) { return rows / GROUP * SPAN; }
  static constexpr int KS = HDT / 16;  // k steps of a product over the head
  static constexpr int DT = HDT / 32;  // 32-column tiles of the head
};

template <int HDT>
DEV_INLINE int perm(int row) {
  return HDT == 64 ? ((row & 2) << 1) | ((row & 4) >> 2) : (row & 3) << 2;
}
template <int HDT>
DEV_INLINE int lds_at(int row, int chunk) {
  using G = Geo<HDT>;
  return row / G::GROUP * G::SPAN + row % G::GROUP * (G::NCH * 16) +
         ((chunk ^ perm<HDT>(row)) << 4);
}

// A or B operand whose k runs along the row: rows r0 + (lane & 31), elements
// 16*ks + 8*(lane >> 5) + 0..7; r0 a multiple of 16
template <int HDT>
DEV_INLINE s16x8 frag_row(const char* lds, int r0, int ks, int lane) {
  // chunk bit 1 is in no perm: it stays out of the lane's part
  return *reinterpret_cast<const s16x8*>(
      lds + Geo<HDT>::bytes(r0) + (ks & 1) * 32 +
      lds_at<HDT>(lane & 31, 2 * (ks & ~1) + (lane >> 5)));
}

DEV_INLINE s16x8 read_tr2(const char* lo, const char* hi) {
  typedef __attribute__((address_space(3))) s16x4* tp_t;
  s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tp_t)lo);
  s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tp_t)hi);
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
// A operand whose k runs down the rows, in the accumulators' order: column
// 32*dt + (lane & 31), rows r0 + 4*h + 0..3 and r0 + 8 + 4*h + 0..3 with
// h = lane >> 5; r0 a multiple of 16. The transposing read hands each lane of
// 16 one column of the 4 x 16 block that the 16 lanes fetch in 8-byte pieces.
template <int HDT>
DEV_INLINE s16x8 frag_col(const char* lds, int r0, int dt, int lane) {
  int row = 4 * (lane >> 5) + ((lane >> 2) & 3);
  int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1);
  const char* p = lds + Geo<HDT>::bytes(r0) + lds_at<HDT>(row, chunk) +
                  (lane & 1) * 8;
  return read_tr2(p, p + Geo<HDT>::bytes(8));
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
  uintptr_t b = (uintptr_t)base;
  b = (uintptr_t)(unsigned)uniform((int)(b >> 32)) << 32 |
      (unsigned)uniform((int)b);
  base = reinterpret_cast<const void*>(b);
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
// LDS in tiles of R rows, by W waves. PACKED: row r is position r / g of head
// r % g, else position r. A wave's load moves RPI = 4 or 8 rows. In a whole
// tile their addresses are a scalar base and a lane's offset that never
// changes (`quick`: RPI rows must not straddle positions unevenly, so g
// divides RPI or RPI g); lanes past the head's end fetch its first chunk,
// whose partner in the product is 0 or whose result is not stored. The last
// tile works out each lane's row and fetches zeros beyond the end.
template <int HDT, int R, bool PACKED, int W = 4>
struct Stream {
  static constexpr int NCH = Geo<HDT>::NCH, RPI = 64 / NCH, N = R / RPI / W;
  static_assert(N > 0, "pieces a wave");
  static constexpr int SPAN = Geo<HDT>::SPAN;
  const char* base;
  long ss, sh;
  unsigned off;
  bool quick;

  DEV_INLINE Stream(const Args& a, const View& v, const Seq& s, int lane) {
    ss = v.ss, sh = v.sh;
    base = reinterpret_cast<const char*>(v.p) +
           2 * (s.batch * v.sb + (long)s.kvh * (PACKED ? a.g : 1) * sh);
    quick = v.quick;
    int l = lane / NCH;
    int chunk = (lane % NCH) ^ perm<HDT>(l);
    if (chunk * 8 >= a.hd) chunk = 0;
    long at = PACKED ? (l / a.g) * ss + (l % a.g) * sh : l * ss;
    off = (unsigned)(2 * at) + chunk * 16;
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
        to_lds16(base + 2 * at, off, lds + idx * SPAN);
      }
      return;
    }
    asm volatile("" : "+v"(lane));  // keeps this out of the loop's registers
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int idx = wave * N + i;
      int row = idx * RPI + lane / NCH;
      int chunk = (lane % NCH) ^ perm<HDT>(row);
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
      to_lds16(src, lds + idx * SPAN);
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
// to the row's memory. A row's two lanes swap every second piece, so that each
// stores 16 bytes.
template <typename T, int DT>
DEV_INLINE void put_row(T* row, const f32x16* acc, float m, int hd, int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      unsigned v[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int x = 4 * j + 2 * i, y = x + 4;
        auto p = __builtin_amdgcn_permlane32_swap(
            Op<T>::pack(acc[dt][x] * m, acc[dt][x + 1] * m),
            Op<T>::pack(acc[dt][y] * m, acc[dt][y + 1] * m), false, false);
        v[i] = p[0], v[i + 2] = p[1];
      }
      int d = dt * 32 + (j + (lane >> 5)) * 8;
      if (d < hd)
        *reinterpret_cast<uint4*>(row + d) = {v[0], v[1], v[2], v[3]};
    }
}

// the same as fp32, 16 bytes a piece
template <int DT>
DEV_INLINE void put_part(float* row, const f32x16* acc, int hd, int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int d = dt * 32 + j * 8 + (lane >> 5) * 4;
      if (d < hd)
        *reinterpret_cast<float4*>(row + d) = {
            acc[dt][4 * j], acc[dt][4 * j + 1], acc[dt][4 * j + 2],
            acc[dt][4 * j + 3]};
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

// what a lane carries of its row over the keys: P's reference, its sum and
// O^T (lane: row, d = 32*i + 8*j + 4*h + 0..3)
template <typename T, int HDT>
struct Running {
  using G = Geo<HDT>;
  float top = -INFINITY, sum = 0.f;
  f32x16 acc[G::DT];
  float c, far;
  DEV_INLINE explicit Running(float scale) : c(scale * kLog2e) {
    far = fminf(8.f / c, FLT_MAX);  // top + far starts at -inf, not NaN
#pragma unroll
    for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  }
  // keys key0 .. key0 + 32*U - 1; the lane's row sees those below `lim`,
  // none of the wave's rows is cut short when they end below `wlo`
  template <int U>
  DEV_INLINE void step(const char* kt, const char* vt, const s16x8* qf,
                       int key0, int lim, int wlo, int lane) {
    f32x16 sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sc[u] = kNone;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
      for (int u = 0; u < U; ++u)
        sc[u] = Op<T>::mfma(frag_row<HDT>(kt, u * 32, ks, lane), qf[ks],
                            sc[u]);
    if (key0 + U * 32 > wlo) {
      int rel = lim - key0 - (lane >> 5) * 4;
#pragma unroll
      for (int i = 0; i < U * 16; ++i)
        if ((i >> 2) * 8 + (i & 3) >= rel) sc[i >> 4][i & 15] = -INFINITY;
    }
    float m = sc[0][0];
#pragma unroll
    for (int i = 1; i < U * 16; ++i) m = fmaxf(m, sc[i >> 4][i & 15]);
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
    unsigned p[U * 8];
#pragma unroll
    for (int i = 0; i < U * 8; ++i) {
      float x = __builtin_amdgcn_exp2f(
          fmaf(sc[i >> 3][(2 * i) & 15], c, base));
      float y = __builtin_amdgcn_exp2f(
          fmaf(sc[i >> 3][(2 * i + 1) & 15], c, base));
      sum += x + y;
      p[i] = Op<T>::pack(x, y);
    }
#pragma unroll
    for (int k = 0; k < U * 2; ++k)
#pragma unroll
      for (int i = 0; i < G::DT; ++i)
        acc[i] = Op<T>::mfma(frag_col<HDT>(vt, k * 16, i, lane),
                             pack8(p + 4 * k), acc[i]);
  }
  // The row's output and lse; or, as part `at` of several (part: [parts]
  // [rows][hd] of outputs, then [parts][rows] of lse, rows = b*hk*sq*g), its
  // share of them for attn_rc_join_rows_k
  DEV_INLINE void put(const Args& a, const Seq& s, const Row& row, int bh,
                      int parts, int at, float* part, int lane) {
    sum += other_half(sum);
    if (!row.stored) return;
    bool some = row.valid && row.lim > 0 && top != -INFINITY;
    // a NaN has to come out: it fails the comparisons that raise `top`
    some = some || (row.valid && sum != sum);
    float lse = some ? top * c + __builtin_amdgcn_logf(sum) : INFINITY;
    float m = some ? 1.f / sum : 0.f;
    if (!some)
#pragma unroll
      for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
    long r = (long)bh * a.sq * a.g + row.r;
    if (parts == 1) {
      T* o = reinterpret_cast<T*>(a.out) +
             (((long)s.batch * a.sq + row.pos) * a.hk * a.g + row.head) *
                 a.hd;
      put_row<T, G::DT>(o, acc, m, a.hd, lane);
      if (lane < 32 && a.lse) a.lse[r] = lse;
      return;
    }
    long rows = (long)a.b * a.hk * a.sq * a.g;
    if (lane < 32) part[parts * rows * a.hd + at * rows + r] = lse;
    if (!some) return;  // not read then
#pragma unroll
    for (int i = 0; i < G::DT; ++i) acc[i] *= m;
    put_part<G::DT>(part + (at * rows + r) * a.hd, acc, a.hd, lane);
  }
};

// forward of a block of n packed rows from r0 on that see no key, or none of
// part `at`'s
DEV_INLINE void no_keys(const Args& a, const Seq& s, int bh, int r0, int n,
                        int parts, int at, float* part) {
  int all = a.sq * a.g;
  n = all - r0 < n ? all - r0 : n;
  long r = (long)bh * all + r0, rows = (long)a.b * a.hk * all;
  float* lse = parts == 1 ? a.lse + r : part + parts * rows * a.hd +
                                            at * rows + r;
  if ((parts > 1 || a.lse) && (int)threadIdx.x < n)
    lse[threadIdx.x] = INFINITY;
  if (parts > 1) return;  // no output is read then
  clear(n, a.hd / 8, [&](int i) {
    int pos = (int)mdiv(r0 + i, a.g_mul, a.g_shift);
    return reinterpret_cast<short*>(a.out) +
           (((long)s.batch * a.sq + pos) * a.hk * a.g + s.kvh * a.g + r0 + i -
            pos * a.g) *
               a.hd;
  });
}

// ---- forward: a block has 128 packed rows, a wave 32 ----------------------
// nsplit > 1: the keys' tiles go to that many blocks in turn, whose results a
// last kernel joins (in runs, causal blocks were done at different times: 268
// against 161 us for 16384 tokens of 2 heads of 128). 4 x 4096 tokens x 12 heads: 250 us at heads of
// 64, 435 at 128; 16384 causal tokens, 16/2 heads of 128: 1.07 ms.
template <typename T, int HDT>
__global__ __launch_bounds__(256, 2) void attn_rc_fwd_k(Args a, int nblk,
                                                        int nsplit,
                                                        float* part) {
  using G = Geo<HDT>;
  LDS_BUFFER(k0, G::bytes(TILE));
  LDS_BUFFER(k1, G::bytes(TILE));
  LDS_BUFFER(v0, G::bytes(TILE));
  LDS_BUFFER(v1, G::bytes(TILE));
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk, split;
  Seq s = place<false>(a, nblk, nsplit, &bh, &blk, &split);
  // keys that any row of the block sees: the last row's, or none
  int last = (blk * 128 + 127) / a.g;
  last = last < s.qlen ? last : s.qlen - 1;
  int end = blk * 128 < s.rows ? s.klen : 0;
  if (a.causal && last + s.off + 1 < end) end = last + s.off + 1;
  int ntile = end > 0 ? (end + TILE - 1) / TILE : 0;
  if (split >= ntile) {
    no_keys(a, s, bh, blk * 128, 128, nsplit, split, part);
    return;
  }
  Row row(a, s, blk * 128 + wave * 32 + (lane & 31));
  Stream<HDT, TILE, false> kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  s16x8 qf[G::KS];
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.q.p) +
                2 * (s.batch * a.q.sb + row.pos * a.q.ss + row.head * a.q.sh),
            row.valid, lane, qf);
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);
  Running<T, HDT> run(a.scale);
  auto load = [&](int t, char* kd, char* vd) {
    kin.load(a, t * TILE, s.klen, kd, wave, lane);
    vin.load(a, t * TILE, s.klen, vd, wave, lane);
  };
  auto step = [&](int t, const char* kt, const char* vt) {
    if (t * TILE < whi)
      run.template step<2>(kt, vt, qf, t * TILE, row.lim, wlo, lane);
  };
  load(split, k0, v0);
  staged();
  for (int t = split; t < ntile; t += 2 * nsplit) {
    int t1 = t + nsplit, t2 = t1 + nsplit;
    if (t1 < ntile) load(t1, k1, v1);
    step(t, k0, v0);
    staged();
    if (t1 >= ntile) break;
    if (t2 < ntile) load(t2, k0, v0);
    step(t1, k1, v1);
    staged();
  }
  run.put(a, s, row, bh, nsplit, split, part, lane);
}

// ---- forward of short sequences: 256 keys at most, heads up to 64 ---------
// All of K and V is loaded at once and 8 waves take 256 packed rows: a step is
// shorter than a load's latency, which is paid once instead of once a tile.
// Two blocks a CU: 1536 heads of 197 tokens 45 us; one block that fetches the
// next head's tiles into the other half of its LDS meanwhile took 70.
template <typename T>
__global__ __launch_bounds__(512, 4) void attn_rc_fwd_short_k(Args a,
                                                              int nblk) {
  using G = Geo<64>;
  LDS_BUFFER(kall, G::bytes(256));
  LDS_BUFFER(vall, G::bytes(256));
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk, split;
  Seq s = place<false, 256>(a, nblk, 1, &bh, &blk, &split);
  Stream<64, 64, false, 8> kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  int end = blk * 256 < s.rows ? s.klen : 0;
  if (end == 0) {
    no_keys(a, s, bh, blk * 256, 256, 1, 0, nullptr);
    return;
  }
  int ntile = (end + 63) / 64;
  for (int t = 0; t < ntile; ++t) {
    kin.load(a, t * 64, s.klen, kall + G::bytes(64) * t, wave, lane);
    vin.load(a, t * 64, s.klen, vall + G::bytes(64) * t, wave, lane);
  }
  Row row(a, s, blk * 256 + wave * 32 + (lane & 31));
  s16x8 qf[4];
  keep<64>(a,
           reinterpret_cast<const char*>(a.q.p) +
               2 * (s.batch * a.q.sb + row.pos * a.q.ss + row.head * a.q.sh),
           row.valid, lane, qf);
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);
  Running<T, 64> run(a.scale);
  staged();
  for (int t = 0; t < ntile; ++t) {
    if (t * 64 >= whi) break;
    run.template step<2>(kall + G::bytes(64) * t, vall + G::bytes(64) * t, qf,
                         t * 64, row.lim, wlo, lane);
  }
  run.put(a, s, row, bh, 1, 0, nullptr, lane);
}

// ---- forward of few rows (32 at most: single tokens) ----------------------
// The keys' bytes are all there is to it, so every wave streams its own run
// of them, 32 at a time, through its own two buffers, with no barrier: a
// block's two waves share nothing but the launch. parts = 2 * gridDim / bh.
// 32 caches of 8191 keys, 4 key heads of 128: 131 us, 4.1 TB/s (a large copy
// reaches 4.7); by blocks of 128 rows it took 270.
template <typename T, int HDT>
__global__ __launch_bounds__(128, 2) void attn_rc_few_k(Args a, int parts,
                                                        int per,
                                                        float* part) {
  using G = Geo<HDT>;
  using In = Stream<HDT, 32, false, 1>;
  __shared__ __attribute__((aligned(16))) char lds[2][4][G::bytes(32)];
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int heads = a.b * a.hk;
  int at = uniform(blockIdx.x / heads), bh = blockIdx.x - at * heads;
  at = at * 2 + wave;
  Seq s(a, bh);
  Row row(a, s, lane & 31);
  char *k0 = lds[wave][0], *v0 = lds[wave][1];
  char *k1 = lds[wave][2], *v1 = lds[wave][3];
  In kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  s16x8 qf[G::KS];
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.q.p) +
                2 * (s.batch * a.q.sb + row.pos * a.q.ss + row.head * a.q.sh),
            row.valid, lane, qf);
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);
  int t = at * per, end = (whi + 31) / 32;
  end = end < t + per ? end : t + per;
  Running<T, HDT> run(a.scale);
  auto load = [&](int i, char* kd, char* vd) {
    kin.load(a, i * 32, s.klen, kd, 0, lane);
    vin.load(a, i * 32, s.klen, vd, 0, lane);
  };
  // all but the newest tile's loads have landed
  auto landed = [&](bool newest) {
    if (newest)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * In::N) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  auto step = [&](int i, const char* kt, const char* vt) {
    run.template step<1>(kt, vt, qf, i * 32, row.lim, wlo, lane);
    // the buffer's reads are done before it is loaded again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  if (t < end) load(t, k0, v0);
  for (; t < end; t += 2) {
    if (t + 1 < end) load(t + 1, k1, v1);
    landed(t + 1 < end);
    step(t, k0, v0);
    if (t + 1 >= end) break;
    if (t + 2 < end) load(t + 2, k0, v0);
    landed(t + 2 < end);
    step(t + 1, k1, v1);
  }
  run.put(a, s, row, bh, parts, at, part, lane);
}

// out = sum over parts of exp2(lse_p - lse) out_p, lse = log2 sum exp2(lse_p).
// Groups of 32 lanes, GPR of the block's 8 a row: with many parts a row has
// all 8, which take the parts in turn, so that all of its loads are out at
// once; with 8 parts or fewer each group has a row. Parts that saw no key have
// lse +inf and no output; they come last, as parts take the keys in turn.
template <typename T, int GPR>
__global__ __launch_bounds__(256) void attn_rc_join_rows_k(Args a, int parts,
                                                           const float* part) {
  __shared__ float4 accs[8][32];
  __shared__ float sums[8];
  long rows = (long)a.b * a.hk * a.sq * a.g;
  int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, d = lane * 4;
  long r = (long)blockIdx.x * (8 / GPR) + grp / GPR;
  grp %= GPR;
  if (GPR < 8 && r >= rows) return;
  const float* ls = part + parts * rows * a.hd + r;
  float top = -INFINITY;
  int used = 0;
  for (int p = lane; p < parts; p += 32) {
    float l = ls[p * rows];
    if (l != INFINITY) {
      top = fmaxf(top, l);
      used = p + 1;
    }
  }
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    top = fmaxf(top, __shfl_xor(top, m, 64));
    int o = __shfl_xor(used, m, 64);
    used = o > used ? o : used;
  }
  float sum = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  int at = d < a.hd ? d : 0;  // lanes past the head load and drop its start
#pragma unroll 4
  for (int p = grp; p < used; p += GPR) {
    float4 x =
        *reinterpret_cast<const float4*>(part + (p * rows + r) * a.hd + at);
    // a part whose scores are all -inf has no output either
    bool none = ls[p * rows] == INFINITY;
    float w = none ? 0.f : __builtin_amdgcn_exp2f(ls[p * rows] - top);
    x.x = none ? 0.f : x.x, x.y = none ? 0.f : x.y;
    x.z = none ? 0.f : x.z, x.w = none ? 0.f : x.w;
    sum += w;
    acc.x += w * x.x, acc.y += w * x.y, acc.z += w * x.z, acc.w += w * x.w;
  }
  if (GPR == 8) {
    accs[grp][lane] = acc;
    if (lane == 0) sums[grp] = sum;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      float4 x = accs[k][lane];
      sum += sums[k];
      acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
    }
  }
  float m = sum != 0.f ? 1.f / sum : 0.f;
  int n = a.sq * a.g;
  int bh = (int)(r / n), pr = (int)(r - (long)bh * n);
  int batch = bh / a.hk, pos = (int)mdiv(pr, a.g_mul, a.g_shift);
  int head = (bh - batch * a.hk) * a.g + pr - pos * a.g;
  if (d < a.hd) {
    uint2 v = {Op<T>::pack(acc.x * m, acc.y * m),
               Op<T>::pack(acc.z * m, acc.w * m)};
    *reinterpret_cast<uint2*>(
        reinterpret_cast<T*>(a.out) +
        (((long)batch * a.sq + pos) * a.hk * a.g + head) * a.hd + d) = v;
  }
  if (lane == 0 && a.lse)
    a.lse[r] = sum != 0.f ? top + __builtin_amdgcn_logf(sum) : INFINITY;
}

// ---- backward 1: D, and dQ of 128 packed rows -----------------------------
// nsplit > 1: the keys' tiles go to that many blocks in turn, whose fp32 sums
// a last kernel adds. 4 x 4096 tokens x 12 heads: 308 us at heads of 64, 541
// at 128; 16384 causal tokens, 16/2 heads of 128: 1.3 to 1.4 ms. dP's sums start
// from -D, here and for dK, dV: 1 to 3% less than a subtraction behind them.
template <typename T, int HDT>
__global__ __launch_bounds__(256, 2) void attn_rc_dq_k(Args a, int nblk,
                                                       int nsplit,
                                                       float* part) {
  using G = Geo<HDT>;
  LDS_BUFFER(k0, G::bytes(TILE));
  LDS_BUFFER(k1, G::bytes(TILE));
  LDS_BUFFER(v0, G::bytes(TILE));
  LDS_BUFFER(v1, G::bytes(TILE));
  int lane = threadIdx.x & 63, h = lane >> 5;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk, split;
  Seq s = place<false>(a, nblk, nsplit, &bh, &blk, &split);
  int last = (blk * 128 + 127) / a.g;
  last = last < s.qlen ? last : s.qlen - 1;
  int end = blk * 128 < s.rows ? s.klen : 0;
  if (a.causal && last + s.off + 1 < end) end = last + s.off + 1;
  int ntile = end > 0 ? (end + TILE - 1) / TILE : 0;
  if (split >= ntile) {  // nothing to see, or no tile for this part
    int all = a.sq * a.g, n = all - blk * 128 < 128 ? all - blk * 128 : 128;
    if (split == 0 && (int)threadIdx.x < n)
      a.delta[(long)bh * all + blk * 128 + threadIdx.x] = 0.f;
    auto at = [&](int i) {
      int r = blk * 128 + i, pos = (int)mdiv(r, a.g_mul, a.g_shift);
      return (((long)s.batch * a.sq + pos) * a.hk * a.g + s.kvh * a.g + r -
              pos * a.g) *
             a.hd;
    };
    if (nsplit == 1)
      clear(n, a.hd / 8,
            [&](int i) { return reinterpret_cast<T*>(a.dq) + at(i); });
    else
      clear(n, a.hd / 4, [&](int i) {
        return part + (long)split * a.b * a.sq * a.hk * a.g * a.hd + at(i);
      });
    return;
  }
  Row row(a, s, blk * 128 + wave * 32 + (lane & 31));
  Stream<HDT, TILE, false> kin(a, a.k, s, lane), vin(a, a.v, s, lane);
  int wlo = wave_min(row.lim), whi = wave_max(row.valid ? row.lim : 0);
  auto load = [&](int t, char* kd, char* vd) {
    kin.load(a, t * TILE, s.klen, kd, wave, lane);
    vin.load(a, t * TILE, s.klen, vd, wave, lane);
  };
  load(split, k0, v0);
  s16x8 qf[G::KS], df[G::KS];
  keep<HDT>(a,
            reinterpret_cast<const char*>(a.dout.p) +
                2 * (s.batch * a.dout.sb + row.pos * a.dout.ss +
                     row.head * a.dout.sh),
            row.valid, lane, df);
  long oat = (((long)s.batch * a.sq + row.pos) * a.hk * a.g + row.head) *
             a.hd;
  // D from the stored output. Its rounding moves dS by P times a sum of
  // random half steps, which is below dS's own rounding where P is spread
  // over many keys; rows of few keys get it from P and dP, below.
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

  float c = a.scale * kLog2e;
  f32x16 acc[G::DT];
#pragma unroll
  for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  // P and dP plus `from` of keys key0.. that lie at rows r0.. of the tiles
  auto probs = [&](const char* kt, const char* vt, int r0, int key0,
                   const f32x16& from, f32x16& sc, f32x16& dp) {
    sc = kNone;
    dp = from;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) {
      sc = Op<T>::mfma(frag_row<HDT>(kt, r0, ks, lane), qf[ks], sc);
      dp = Op<T>::mfma(frag_row<HDT>(vt, r0, ks, lane), df[ks], dp);
    }
    if (key0 + 32 > wlo) {
      int rel = row.lim - key0 - h * 4;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((i >> 2) * 8 + (i & 3) >= rel) sc[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], c, -lse));
  };
  f32x16 less;  // -D: dP's products start from it
  auto step = [&](int t, const char* kt, const char* vt) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int key0 = t * TILE + u * 32;
      if (key0 >= whi) return;
      f32x16 x, dp;
      probs(kt, vt, u * 32, key0, less, x, dp);
      unsigned p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        p[i] = Op<T>::pack(x[2 * i] * dp[2 * i], x[2 * i + 1] * dp[2 * i + 1]);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < G::DT; ++i)
          acc[i] = Op<T>::mfma(frag_col<HDT>(kt, u * 32 + k * 16, i, lane),
                               pack8(p + 4 * k), acc[i]);
    }
  };
  staged();
  if (split == 0 && wlo <= TILE) {
    float d = 0.f;
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
      f32x16 x, dp;
      probs(k0, v0, u * 32, u * 32, kNone, x, dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) d += x[i] * dp[i];
    }
    d += other_half(d);
    if (row.lim <= TILE) delta = row.valid ? d : 0.f;
  }
  if (row.stored && h == 0 && split == 0) a.delta[lat] = -delta;
#pragma unroll
  for (int i = 0; i < 16; ++i) less[i] = -delta;
  for (int t = split; t < ntile; t += 2 * nsplit) {
    int t1 = t + nsplit, t2 = t1 + nsplit;
    if (t1 < ntile) load(t1, k1, v1);
    step(t, k0, v0);
    staged();
    if (t1 >= ntile) break;
    if (t2 < ntile) load(t2, k0, v0);
    step(t1, k1, v1);
    staged();
  }
  if (!row.stored) return;
  bool some = row.valid && row.lim > 0;
  if (!some)
#pragma unroll
    for (int i = 0; i < G::DT; ++i) acc[i] = kNone;
  if (nsplit == 1) {
    put_row<T, G::DT>(reinterpret_cast<T*>(a.dq) + oat, acc, a.scale, a.hd,
                      lane);
    return;
  }
  put_part<G::DT>(part + (long)split * a.b * a.sq * a.hk * a.g * a.hd + oat,
                  acc, a.hd, lane);
}

// ---- backward 2: dK, dV of 128 keys, over all packed rows -----------------
// Kept in registers: the wave's 32 keys' K, and dK, dV (64 each at a head of
// 128). V as well would spill there, so from heads of 96 on it stays in LDS
// and rows stream 32 at a time to leave room for two blocks a CU.
// With few key blocks the rows are dealt out to `nsplit` blocks in turn
// (tile t to block t % nsplit), whose fp32 sums a last kernel adds; runs of
// tiles instead, so that causal blocks are alike in length, took 1.4 to 1.8
// times as long. 4 x 4096 tokens x 12 heads: 427 us at heads of 64 (three
// blocks a CU; two took 6% more), 808 at 128; 16384 causal tokens, 16/2 heads
// of 128: 2.0 to 2.1 ms.
template <typename T, int HDT>
__global__ __launch_bounds__(256, HDT == 64 ? 3 : 2) void attn_rc_dkv_k(
    Args a, int nblk, int nsplit, float* part) {
  using G = Geo<HDT>;
  constexpr bool VLDS = HDT > 64;
  constexpr int RT = VLDS ? 32 : 64;
  LDS_BUFFER(q0, G::bytes(RT));
  LDS_BUFFER(q1, G::bytes(RT));
  LDS_BUFFER(d0, G::bytes(RT));
  LDS_BUFFER(d1, G::bytes(RT));
  LDS_BUFFER(stat0, 512);  // 64 rows' lse and -D
  LDS_BUFFER(stat1, 512);
  LDS_BUFFER(vkeep, VLDS ? G::bytes(128) : 16);
  int lane = threadIdx.x & 63;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bh, blk, split;
  Seq s = place<true>(a, nblk, nsplit, &bh, &blk, &split);
  int first = 0;
  if (a.causal && blk * 128 > s.off) first = (blk * 128 - s.off) * a.g;
  first &= ~(RT - 1);
  int ntile = 0;
  if (blk * 128 < s.klen && first < s.rows)
    ntile = (s.rows - first + RT - 1) / RT;
  if (split >= ntile) {  // no row sees these keys, or no tile for this part
    int n = a.sk - blk * 128 < 128 ? a.sk - blk * 128 : 128;
    auto at = [&](int i) {
      return (((long)s.batch * a.sk + blk * 128 + i) * a.hk + s.kvh) * a.hd;
    };
    if (nsplit == 1) {
      clear(n, a.hd / 8,
            [&](int i) { return reinterpret_cast<T*>(a.dk) + at(i); });
      clear(n, a.hd / 8, [&](int i) {
        return reinterpret_cast<T*>(a.dv) + s.batch * a.vb +
               (blk * 128 + i) * a.vs + s.kvh * a.vh;
      });
    } else {
      long all = (long)a.b * a.sk * a.hk * a.hd;
      float* out = part + 2 * split * all;
      clear(n, a.hd / 4, [&](int i) { return out + at(i); });
      clear(n, a.hd / 4, [&](int i) { return out + all + at(i); });
    }
    return;
  }
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
  load(split, q0, d0, stat0);
  if (VLDS) {
    Stream<HDT, 128, false> vin(a, a.v, s, lane);
    vin.quick = false;  // zeros past the head's end: dO has none there
    vin.load(a, blk * 128, s.klen, vkeep, wave, lane);
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
    int ln = lane;  // some addresses are worked out anew, for registers
    asm volatile("" : "+v"(ln));
    int h = ln >> 5;
#pragma unroll
    for (int u = 0; u < RT / 32; ++u) {
      int r0 = first + t * RT + u * 32;
      if (!wlive || r0 + 32 <= wlo || r0 >= s.rows) continue;
      f32x16 sc = kNone, dp;  // dP - D
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 d4 =
            *reinterpret_cast<const float4*>(ds + u * 32 + j * 8 + h * 4);
        dp[4 * j] = d4.x, dp[4 * j + 1] = d4.y;
        dp[4 * j + 2] = d4.z, dp[4 * j + 3] = d4.w;
      }
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
        const float* lp = &l4.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i], c, -lp[2 * i]));
          float y = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i + 1], c, -lp[2 * i + 1]));
          p[2 * j + i] = Op<T>::pack(x, y);
          d[2 * j + i] = Op<T>::pack(x * dp[4 * j + 2 * i],
                                     y * dp[4 * j + 2 * i + 1]);
        }
      }
      // these products' operands are fetched only now: K or V went to scratch
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < G::DT; ++i) {
          dv[i] = Op<T>::mfma(frag_col<HDT>(dt, u * 32 + k * 16, i, ln),
                              pack8(p + 4 * k), dv[i]);
          dk[i] = Op<T>::mfma(frag_col<HDT>(qt, u * 32 + k * 16, i, ln),
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
  asm volatile("" : "+v"(lane));  // worked out anew, for registers
  key = blk * 128 + wave * 32 + (lane & 31);
  if (key >= a.sk) return;
  if (key >= s.klen)
#pragma unroll
    for (int i = 0; i < G::DT; ++i) dk[i] = dv[i] = kNone;
  long at = (((long)s.batch * a.sk + key) * a.hk + s.kvh) * a.hd;
  if (nsplit == 1) {
    put_row<T, G::DT>(reinterpret_cast<T*>(a.dv) + s.batch * a.vb +
                          key * a.vs + s.kvh * a.vh,
                      dv, 1.f, a.hd, lane);
    put_row<T, G::DT>(reinterpret_cast<T*>(a.dk) + at, dk, a.scale, a.hd,
                      lane);
    return;
  }
  long n = (long)a.b * a.sk * a.hk * a.hd;
  float* out = part + 2 * split * n + at;
  put_part<G::DT>(out, dk, a.hd, lane);
  put_part<G::DT>(out + n, dv, a.hd, lane);
}

// ---- backward of short sequences: all three gradients in one pass ---------
// 65 to 256 keys, as many packed rows, heads up to 64: a block of 4 waves
// holds a key head's keys, a wave one or two groups of 32, and runs over its
// rows 32 at a time, so S, dP and the exponentials are worked out once, and
// q, k, v, out and dout are read once. Two blocks share a CU, so that one's
// loads and barriers pass under the other's products (one block of 8 waves
// took 158 us at 1536 heads of 197 tokens, this one 117; the two kernels above
// 163). dK and dV gather in registers as
// in attn_rc_dkv_k. dQ needs all keys of a row: the waves put dS (16 bits,
// which it has as an operand anyway) to LDS, and after a barrier each takes 16
// columns of dQ's 32 rows over all keys, in 16x16x32 products.
// dS lies by key, 32 rows or 64 bytes each, with its 8-byte pieces moved
// about (ds_at) so that 32 keys' writes and the transposing reads' 8 keys x
// 32 bytes meet distinct banks.
typedef float f32x4v __attribute__((ext_vector_type(4)));
// row r (0..31, a multiple of 4) of a key's dS
DEV_INLINE int ds_at(int key, int r) {
  int f = ((key >> 2) & 2) | ((key >> 2) & 1);
  return key * 64 + (((r >> 3) ^ f) << 4) +
         ((((r >> 2) ^ (key >> 4)) & 1) << 3);
}
template <typename T> DEV_INLINE f32x4v mfma16(s16x8 a, s16x8 b, f32x4v c);
template <>
DEV_INLINE f32x4v mfma16<__hip_bfloat16>(s16x8 a, s16x8 b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
      0);
}
template <>
DEV_INLINE f32x4v mfma16<__half>(s16x8 a, s16x8 b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// NKG: groups of 32 keys there is room for. (A second dS buffer in place of
// the step's second barrier made no difference.)
template <typename T, int NKG>
__global__ __launch_bounds__(256, 2) void attn_rc_bwd_short_k(Args a) {
  using G = Geo<64>;
  constexpr int KG = (NKG + 3) / 4;  // groups of a wave: wave, wave + 4
  LDS_BUFFER(kall, G::bytes(NKG * 32));
  LDS_BUFFER(q0, G::bytes(32));
  LDS_BUFFER(q1, G::bytes(32));
  LDS_BUFFER(d0, G::bytes(32));
  LDS_BUFFER(d1, G::bytes(32));
  LDS_BUFFER(dso, NKG * 32 * 64);
  __shared__ __attribute__((aligned(16))) float lse[256], del[256];
  int lane = threadIdx.x & 63, h = lane >> 5;
  int wave = uniform(threadIdx.x >> 6);
  int bh = blockIdx.x;
  Seq s(a, bh);
  int ntile = (s.rows + 31) / 32;
  Stream<64, NKG * 32, false> kin(a, a.k, s, lane);
  Stream<64, 32, true> qin(a, a.q, s, lane), din(a, a.dout, s, lane);
  kin.load(a, 0, s.klen, kall, wave, lane);
  auto load = [&](int t, char* qd, char* dd) {
    qin.load(a, t * 32, s.rows, qd, wave, lane);
    din.load(a, t * 32, s.rows, dd, wave, lane);
  };
  load(0, q0, d0);
  // D of all rows: 8 elements a thread, 8 threads a row
  {
    int de = (threadIdx.x & 7) * 8;
    const T* ob = reinterpret_cast<const T*>(a.out) +
                  (((long)s.batch * a.sq) * a.hk * a.g + (long)s.kvh * a.g) *
                      a.hd +
                  de;
    const T* db = reinterpret_cast<const T*>(din.base) + de;
    uint4 ov[8], dv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int r = i * 32 + (threadIdx.x >> 3);
      ov[i] = dv[i] = {0, 0, 0, 0};
      if (r < s.rows && de < a.hd) {
        int pos = (int)mdiv(r, a.g_mul, a.g_shift), hd = r - pos * a.g;
        ov[i] = *reinterpret_cast<const uint4*>(
            ob + ((long)pos * a.hk * a.g + hd) * a.hd);
        dv[i] = *reinterpret_cast<const uint4*>(db + pos * a.dout.ss +
                                                hd * a.dout.sh);
      }
    }
    lse[threadIdx.x] = threadIdx.x < s.rows
                           ? a.lse[(long)bh * a.sq * a.g + threadIdx.x]
                           : INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* x = reinterpret_cast<const T*>(&ov[i]);
      const T* y = reinterpret_cast<const T*>(&dv[i]);
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) d += to_f32(x[j]) * to_f32(y[j]);
#pragma unroll
      for (int m = 1; m < 8; m <<= 1) d += __shfl_xor(d, m, 64);
      if ((threadIdx.x & 7) == 0) del[i * 32 + (threadIdx.x >> 3)] = d;
    }
  }
  s16x8 vf[KG][4];
  float bias[KG];
#pragma unroll
  for (int n = 0; n < KG; ++n) {
    int key = (wave + n * 4) * 32 + (lane & 31);
    bias[n] = key < s.klen ? 0.f : -INFINITY;
    keep<64>(a,
             reinterpret_cast<const char*>(a.v.p) +
                 2 * (s.batch * a.v.sb + s.kvh * a.v.sh + key * a.v.ss),
             key < s.klen, lane, vf[n]);
  }
  float c = a.scale * kLog2e;
  f32x16 dk[KG][2], dv[KG][2];
#pragma unroll
  for (int n = 0; n < KG; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) dk[n][i] = dv[n][i] = kNone;
  int nk = (s.klen + 31) / 32;
  staged();

  auto step = [&](int t, const char* qt, const char* dt) {
    const float *ls = lse + t * 32, *dl = del + t * 32;
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int n = 0; n < KG; ++n) {
      int grp = wave + n * 4;
      if (grp >= nk) continue;
      f32x16 sc = kNone, dp = kNone;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        sc = Op<T>::mfma(frag_row<64>(qt, 0, ks, lane),
                         frag_row<64>(kall, grp * 32, ks, lane), sc);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        dp = Op<T>::mfma(frag_row<64>(dt, 0, ks, lane), vf[n][ks], dp);
      // the products' operands leave the registers first: spilled ones would
      // have to wait for the tile's loads
      __builtin_amdgcn_sched_barrier(0);
      unsigned p[8], d[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 l4 = *reinterpret_cast<const float4*>(ls + j * 8 + h * 4);
        float4 d4 = *reinterpret_cast<const float4*>(dl + j * 8 + h * 4);
        const float *lp = &l4.x, *dd = &d4.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // a key that is not there has scores of 0 and a bias of -inf
          float x = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i], c, bias[n] - lp[2 * i]));
          float y = __builtin_amdgcn_exp2f(
              fmaf(sc[4 * j + 2 * i + 1], c, bias[n] - lp[2 * i + 1]));
          p[2 * j + i] = Op<T>::pack(x, y);
          d[2 * j + i] =
              Op<T>::pack(x * (dp[4 * j + 2 * i] - dd[2 * i]),
                          y * (dp[4 * j + 2 * i + 1] - dd[2 * i + 1]));
        }
        uint2 v = {d[2 * j], d[2 * j + 1]};
        *reinterpret_cast<uint2*>(dso + grp * 32 * 64 +
                                  ds_at(ln & 31, j * 8 + (ln >> 5) * 4)) = v;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          dv[n][i] = Op<T>::mfma(frag_col<64>(dt, k * 16, i, lane),
                                 pack8(p + 4 * k), dv[n][i]);
          dk[n][i] = Op<T>::mfma(frag_col<64>(qt, k * 16, i, lane),
                                 pack8(d + 4 * k), dk[n][i]);
        }
    }
  };
  // columns 16 * wave.. of the tile's dQ
  auto put_dq = [&](int t) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // its addresses are worked out anew
    int l4 = (ln & 15) >> 2, seg = ln & 3;
    f32x4v acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    int x = (ln >> 4) * 8 + l4;  // keys x.., x + 4.. of a group
    const char* kc = kall + (seg & 1) * 8;
    int chunk = wave * 2 + (seg >> 1);
#pragma unroll
    for (int k = 0; k < NKG; ++k) {
      if (k >= nk) break;
      s16x8 kt = read_tr2(kc + G::bytes(k * 32) + lds_at<64>(x, chunk),
                          kc + G::bytes(k * 32) + lds_at<64>(x + 4, chunk));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const char* d = dso + k * 32 * 64;
        int r = u * 16 + seg * 4;
        acc[u] = mfma16<T>(
            kt, read_tr2(d + ds_at(x, r), d + ds_at(x + 4, r)), acc[u]);
      }
    }
    int e = wave * 16 + (ln >> 4) * 4;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int r = t * 32 + u * 16 + (ln & 15);
      int pos = (int)mdiv(r, a.g_mul, a.g_shift);
      if (pos < a.sq && e < a.hd) {
        uint2 v = {Op<T>::pack(acc[u][0] * a.scale, acc[u][1] * a.scale),
                   Op<T>::pack(acc[u][2] * a.scale, acc[u][3] * a.scale)};
        *reinterpret_cast<uint2*>(
            reinterpret_cast<T*>(a.dq) +
            (((long)s.batch * a.sq + pos) * a.hk * a.g + s.kvh * a.g + r -
             pos * a.g) *
                a.hd +
            e) = v;
      }
    }
    __syncthreads();  // dS is read
  };
  for (int t = 0; t < ntile; t += 2) {
    if (t + 1 < ntile) load(t + 1, q1, d1);
    step(t, q0, d0);
    staged();
    put_dq(t);
    if (t + 1 >= ntile) break;
    if (t + 2 < ntile) load(t + 2, q0, d0);
    step(t + 1, q1, d1);
    staged();
    put_dq(t + 1);
  }
#pragma unroll
  for (int n = 0; n < KG; ++n) {
    int key = (wave + n * 4) * 32 + (lane & 31);
    if (key >= a.sk) continue;
    if (key >= s.klen)
#pragma unroll
      for (int i = 0; i < 2; ++i) dk[n][i] = dv[n][i] = kNone;
    put_row<T, 2>(reinterpret_cast<T*>(a.dv) + s.batch * a.vb + key * a.vs +
                      s.kvh * a.vh,
                  dv[n], 1.f, a.hd, lane);
    put_row<T, 2>(reinterpret_cast<T*>(a.dk) +
                      (((long)s.batch * a.sk + key) * a.hk + s.kvh) * a.hd,
                  dk[n], a.scale, a.hd, lane);
  }
}

// x = scale * sums over the splits of part[split][nx + ny], then dv the sums
// of the ny behind; 4 elements a thread; nx and ny are multiples of 4
template <typename T>
__global__ __launch_bounds__(256) void attn_rc_join_k(
    const float* __restrict__ part, long nx, long ny, int nsplit, T* x,
    Args a) {
  long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= nx + ny) return;
  float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < nsplit; ++k) {
    float4 v = *reinterpret_cast<const float4*>(part + k * (nx + ny) + i);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  float m = i < nx ? a.scale : 1.f;
  uint2 v = {Op<T>::pack(sum.x * m, sum.y * m),
             Op<T>::pack(sum.z * m, sum.w * m)};
  T* to = x + i;
  if (i >= nx) {
    long row = (i - nx) / a.hd;
    int d = (int)(i - nx - row * a.hd), kvh = (int)(row % a.hk);
    row /= a.hk;
    long batch = row / a.sk;
    to = reinterpret_cast<T*>(a.dv) + batch * a.vb +
         (row - batch * a.sk) * a.vs + kvh * a.vh + d;
  }
  *reinterpret_cast<uint2*>(to) = v;
}

// How work is dealt out where there are few blocks; shapes alone decide. Two
// blocks run on each of 256 CUs.
struct Plan {
  int fwd;       // forward: parts over the keys
  bool few;      // rows fit one wave: attn_rc_few_k, ...
  int per;       // ... tiles of 32 in a part
  int dq, dkv;   // backward: parts over the keys, over the rows
  bool whole;    // backward in one pass: attn_rc_bwd_short_k
  bool whole_fwd;  // all keys at once: attn_rc_fwd_short_k
  Plan(long b, long sq, long sk, long hk, long g, long hd, bool causal,
       bool lens) {
    long bh = b * hk, rows = sq * g;
    // One block a head has to fill the chip, or be short: 4 x 65 tokens of 3
    // heads 10 against 15 us, but 8 x 197 of 12 26 against 24. Sequences of
    // few keys take D from P and dP, which only the two-pass backward does.
    whole = !causal && !lens && hd <= 64 && sk > 64 && sk <= 256 &&
            rows <= 256 && (bh >= 256 || (sk <= 128 && rows <= 128));
    long rblk = bh * ((rows + 127) / 128), kblk = bh * ((sk + 127) / 128);
    // two of its blocks a CU: 45 against 51 us at 1536 heads of 197 tokens,
    // and no gain below
    whole_fwd = hd <= 64 && sk <= 256 && rows > 128 &&
                bh * ((rows + 255) / 256) >= 512;
    fwd = dq = dkv = 1;
    per = 0;
    few = false;
    if (rblk == 0 || kblk == 0) return;
    // Parts to fill the chip once; twice where there is work enough to pay for
    // the join of more parts and one round leaves CUs idle or, for a causal
    // mask, with blocks of different lengths. dQ and its join: 8192 causal
    // tokens of 4 heads of 64 74 against 99 us, 2048 of 16 heads of 128 63
    // against 58; 8192 tokens of 6 heads of 64 170 against 193, 4096 of 8 heads
    // of 128 132 against 118.
    long want = rblk < 512 ? 512 / rblk : 1;
    if (rblk < 512 && sk * rblk >= 3 << 19 && (causal || want * rblk < 480))
      want = 1024 / rblk;
    int part = clamp(want, sk / 512, 64);
    if (rows <= 32 && sk >= 512) {
      // runs of 256 keys (8 tiles) a wave, longer where that makes more
      // than 4096 waves, 128 where it makes fewer than 1024
      few = true;
      long tiles = (sk + 31) / 32, run = 8;
      if (bh * ((tiles + 7) / 8) < 1024) run = 4;
      while (run < tiles && bh * ((tiles + run - 1) / run) > 4096) run *= 2;
      per = (int)run;
      fwd = (int)((tiles + 2 * run - 1) / (2 * run)) * 2;
    } else {
      fwd = part;
    }
    dq = part;
    // A causal mask's blocks differ in length: where there is work enough to
    // pay for the join of more parts, two rounds even them out (512 key blocks
    // of 4096 rows 177 against 195 us, of 2048 rows 119 against 107).
    bool even = causal && kblk <= 512 && rows >= 4096 && rows * kblk >= 1 << 20;
    dkv = clamp(((even ? 1024 : 512) + kblk - 1) / kblk, rows / 512, 16);
  }
  static int clamp(long want, long most, long cap) {
    long n = want < most ? want : most;
    n = n < cap ? n : cap;
    return n < 1 ? 1 : (int)n;
  }
};

// -D of every row at the start of backward's workspace, the parts 16-byte
// aligned behind it
long delta_floats(long rows) { return (rows + 3) / 4 * 4; }

template <typename T, int HDT>
void launch(Args a, int bwd, float* ws, hipStream_t s) {
  int rblk = (a.sq * a.g + 127) / 128, kblk = (a.sk + 127) / 128;
  int bh = a.b * a.hk, rblk256 = (a.sq * a.g + 255) / 256;
  Plan p(a.b, a.sq, a.sk, a.hk, a.g, a.hd, a.causal,
         a.q_lens || a.kv_lens);
  if (!bwd) {
    if (rblk == 0) return;
    if (p.few)
      attn_rc_few_k<T, HDT>
          <<<bh * (p.fwd / 2), 128, 0, s>>>(a, p.fwd, p.per, ws);
    else if (HDT == 64 && p.whole_fwd)
      attn_rc_fwd_short_k<T><<<bh * rblk256, 512, 0, s>>>(a, rblk256);
    else
      attn_rc_fwd_k<T, HDT>
          <<<bh * rblk * p.fwd, 256, 0, s>>>(a, rblk, p.fwd, ws);
    if (p.fwd > 1) {
      long rows = (long)bh * a.sq * a.g;
      if (p.fwd > 8)
        attn_rc_join_rows_k<T, 8><<<rows, 256, 0, s>>>(a, p.fwd, ws);
      else
        attn_rc_join_rows_k<T, 1>
            <<<(rows + 7) / 8, 256, 0, s>>>(a, p.fwd, ws);
    }
    return;
  }
  if constexpr (HDT == 64)
    if (p.whole) {
      if (a.sk <= 128)
        attn_rc_bwd_short_k<T, 4><<<bh, 256, 0, s>>>(a);
      else if (a.sk <= 224)
        attn_rc_bwd_short_k<T, 7><<<bh, 256, 0, s>>>(a);
      else
        attn_rc_bwd_short_k<T, 8><<<bh, 256, 0, s>>>(a);
      return;
    }
  long nq = (long)a.b * a.sq * a.hk * a.g * a.hd;
  long nk = (long)a.b * a.sk * a.hk * a.hd;
  a.delta = ws;
  ws += delta_floats(nq / a.hd);
  if (rblk) {
    attn_rc_dq_k<T, HDT><<<bh * rblk * p.dq, 256, 0, s>>>(a, rblk, p.dq, ws);
    if (p.dq > 1)
      attn_rc_join_k<T><<<(nq / 4 + 255) / 256, 256, 0, s>>>(
          ws, nq, 0, p.dq, (T*)a.dq, a);
  }
  if (kblk) {
    attn_rc_dkv_k<T, HDT>
        <<<bh * kblk * p.dkv, 256, 0, s>>>(a, kblk, p.dkv, ws);
    if (p.dkv > 1)
      attn_rc_join_k<T><<<(nk / 2 + 255) / 256, 256, 0, s>>>(
          ws, nk, nk, p.dkv, (T*)a.dk, a);
  }
}

}  // namespace

extern "C" {

// floats of workspace that forward or backward needs; lens: there are lengths
long pdta_attn_recompute_ws(long b, long sq, long sk, long hk, long g,
                            long hd, int causal, int lens, int bwd) {
  Plan p(b, sq, sk, hk, g, hd, causal, lens);
  long nq = b * sq * hk * g * hd, nk = b * sk * hk * hd;
  if (!bwd) return p.fwd > 1 ? p.fwd * (nq + nq / hd) : 0;
  if (p.whole) return 0;
  long x = p.dq > 1 ? p.dq * nq : 0, y = p.dkv > 1 ? 2 * p.dkv * nk : 0;
  return delta_floats(nq / hd) + (x > y ? x : y);
}

// strides: q, k, v, dout, dv, each (b, s, head) in elements; multiples of 8,
// all pointers 16-byte aligned, hd a multiple of 8 up to 128. lens null or [b].
// Forward writes out and, unless null, lse; backward reads both and writes
// dq, dk, dv; either with pdta_attn_recompute_ws floats in ws. Grids must stay
// below 2^32 threads and sq*g below 2^31.
void pdta_attn_recompute(const void* q, const void* k, const void* v,
                         const void* dout, const long* st, void* out,
                         float* lse, void* dq, void* dk, void* dv,
                         const void* q_lens, const void* kv_lens, int lens64, int b, int sq, int sk, int hk, int g,
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
  a.out = out, a.dq = dq, a.dk = dk, a.dv = dv, a.lse = lse, a.delta = nullptr;
  a.vb = st[12], a.vs = st[13], a.vh = st[14];
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
