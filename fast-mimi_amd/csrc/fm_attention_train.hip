// Causal sliding-window attention for training: forward with the row's
// log-sum-exp, and the backward pass, which forms the probabilities again from
// it.  FP32, bfloat16 and float16; grouped query heads; padded batches.
//
// A key head's queries are rows r = t * G + g (position t, head g of its group
// of G), so grouped heads share every key tile that is loaded and the key and
// value gradients sum over them without atomics.  Query t stands at position
// p = S - T + t; key j is visible iff p - window < j <= p and p < length.
//
//   forward   S = Q K^T c, P = exp2(S - max), O = P V / sum P      (c = scale log2 e)
//   backward  P = exp2(S - lse), D = rowsum(dO O), dS = P (dO V^T - D)
//             dQ = dS K scale                     (one block: some rows, all their keys)
//             dV = P^T dO, dK = dS^T Q scale      (one block: some keys, all their rows)
//
// All products run on 32x32 MFMA tiles and are arranged so that what a lane
// holds of one is its operand of the next: S^T (keys x rows) leaves lane l with
// row l % 32 and sixteen keys of it, which is the B operand of O^T = V^T P^T
// once V^T is read in the same order of keys; no probability crosses lanes.
// FP32 inputs use three bf16 pieces of each factor (heads up to 64) or the FP32
// MFMA; 16-bit ones round P and dS (in [0, 1], or a product with it) to the
// inputs' type for the second product, as the operands of the 16-bit MFMA are;
// every sum, maximum and gradient is FP32.
//
// Long calls are bound by the matrix cores and the exponentials and conversions
// beside them, which add on this part: 2 x 4095 positions, 16/4 heads of 128,
// bfloat16, no window: forward 180 us (760 TFLOP/s), dQ 285, dK / dV 410.  Short
// ones by latency: 2500 positions, 8 heads of 64, window 250: 11.5, 15.5, 15.5 us.

#include "fm_common.h"

namespace {

typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2_v __attribute__((ext_vector_type(2)));
typedef float floatx2_v __attribute__((ext_vector_type(2)));
typedef unsigned uintx2_v __attribute__((ext_vector_type(2)));
typedef unsigned uintx4_v __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896341f;

// float16 ends at 2^16 and 2^-24, so what is rounded to it carries a power of two.
// The forward's probabilities, relative to a reference that the maximum may pass by
// 2^SLACK, stand 2^UP higher, and the gradients' (at most 1, and a rounding) 2^P_UP:
// a step is 2^-35 of a row's largest probability and 2^-38 of 1 then, where 2^-24
// would lose what thousands of small ones add up to.
template <typename T> constexpr bool SCALED = std::is_same<T, _Float16>::value;
template <typename T> constexpr float SLACK = SCALED<T> ? 4.0f : 8.0f;
template <typename T> constexpr float UP = SCALED<T> ? 11.0f : 0.0f;
template <typename T> constexpr float P_UP = SCALED<T> ? 14.0f : 0.0f;

template <typename T> struct Elem;
template <> struct Elem<float> {
  typedef floatx4 Frag;
  static constexpr int STEP = 8;  // contraction elements of one fragment pair (two lane halves of 16 bytes)
  static FM_DEVICE floatx16 mma(Frag a, Frag b, floatx16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = fm_mfma32(a[e], b[e], c);
    return c;
  }
  // Accumulator elements STEP / 2 * s .. of a lane as an operand.
  static FM_DEVICE Frag pack(const floatx16& p, int s) { return Frag{p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]}; }
  static FM_DEVICE float dot(Frag a, Frag b, float s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(a[e], b[e], s);
    return s;
  }
  static FM_DEVICE void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<floatx4*>(p) = floatx4{a, b, c, d};
  }
};
template <> struct Elem<__bf16> {
  typedef bf16x8 Frag;
  static constexpr int STEP = 16;
  static FM_DEVICE floatx16 mma(Frag a, Frag b, floatx16 c) { return fm_mfma32_bf16(a, b, c); }
  static FM_DEVICE unsigned two(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2_v{a, b}), bf16x2_v));
  }
  static FM_DEVICE Frag pack(const floatx16& p, int s) {
    uintx4_v u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = two(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
    return __builtin_bit_cast(Frag, u);
  }
  // What pack(p, s) = f left of each value, rounded in its turn.
  static FM_DEVICE Frag pack_rest(const floatx16& p, Frag f, int s) {
    uintx4_v u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = two(p[8 * s + 2 * e] - (float)f[2 * e], p[8 * s + 2 * e + 1] - (float)f[2 * e + 1]);
    return __builtin_bit_cast(Frag, u);
  }
  static FM_DEVICE float dot(Frag a, Frag b, float s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf((float)a[e], (float)b[e], s);
    return s;
  }
  static FM_DEVICE void store4(__bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uintx2_v*>(p) = uintx2_v{two(a, b), two(c, d)};
  }
};
template <> struct Elem<_Float16> {
  typedef halfx8 Frag;
  static constexpr int STEP = 16;
  static FM_DEVICE floatx16 mma(Frag a, Frag b, floatx16 c) { return fm_mfma32_f16(a, b, c); }
  static FM_DEVICE unsigned two(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2_v{a, b}), halfx2_v));
  }
  static FM_DEVICE Frag pack(const floatx16& p, int s) {
    uintx4_v u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = two(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
    return __builtin_bit_cast(Frag, u);
  }
  // What pack(p, s) = f left of each value, rounded in its turn.
  static FM_DEVICE Frag pack_rest(const floatx16& p, Frag f, int s) {
    uintx4_v u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = two(p[8 * s + 2 * e] - (float)f[2 * e], p[8 * s + 2 * e + 1] - (float)f[2 * e + 1]);
    return __builtin_bit_cast(Frag, u);
  }
  static FM_DEVICE float dot(Frag a, Frag b, float s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf((float)a[e], (float)b[e], s);
    return s;
  }
  static FM_DEVICE void store4(_Float16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uintx2_v*>(p) = uintx2_v{two(a, b), two(c, d)};
  }
};

// A strided [batch][rows][heads][head_dim] input; strides in elements.
struct View {
  const void* p;
  long batch, row, head;
};

struct Attn {
  View q, k, v, dout;
  const void* o;  // backward: the forward's output, contiguous
  void *out, *dk, *dv;  // forward: O; backward: dQ in out
  float* lse;      // [B][T][H], log2 of the row's sum of exponentials
  float* stats;    // [2][B][T][H]: lse, infinite for a row without keys; rowsum(dO O)
  float *part_o, *part_ml;  // split forward: unnormalised O [split][B][KV][R][DT], then (max, sum)
  const int* lengths;
  int B, T, S, H, KV, G, D, window, splits;
  FmDivisor by_g;
  float scale, scale2;
};

// Tiles in LDS keep 16-byte chunk c of row r at chunk c ^ swz(r), such that both
// reads below spread over all 64 banks (256 bytes): a fragment read takes the
// same chunk of 16 rows at a time, a transposed 16-bit read 64 bytes of 4 rows,
// an FP32 column read 128 bytes of two rows that lie 4 apart.
template <typename T, int DT>
FM_DEVICE int swz(int row) {
  if constexpr (sizeof(T) == 4) return ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3);
  else if constexpr (DT == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);  // two rows are 256 bytes
}

// How lanes read a tile's operands.  With the swizzle an exclusive-or, every
// address is one lane constant plus the tile's place, changed by constant bits:
// the kernels keep two registers of addresses, not one per read (`fresh` keeps
// the compiler from computing them all before the loop and holding them there).
template <typename T, int DT>
struct Reads {
  typedef typename Elem<T>::Frag Frag;
  static constexpr int PITCH = DT * (int)sizeof(T);

  static FM_DEVICE unsigned lds(const unsigned char* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
  }
  static FM_DEVICE unsigned fresh(unsigned a) {
    asm volatile("" : "+v"(a));
    return a;
  }

  // 32 rows as the A or B operand of a product over their columns: lane l holds
  // row l % 32, bytes 32 s + 16 (l / 32) .. + 15.
  static FM_DEVICE unsigned row_lane(int lane) {
    return (lane & 31) * PITCH + (((lane >> 5) ^ swz<T, DT>(lane & 31)) << 4);
  }
  static FM_DEVICE Frag row(unsigned a, int s) {
    return __builtin_bit_cast(Frag, *(const __attribute__((address_space(3))) uintx4_v*)(a ^ (32 * s)));
  }

  // Columns 0 .. DT - 1 of STEP rows as A operands (one per 32 columns) of a
  // product over the rows, in the order in which a lane holds a 32x32 result:
  // lane l holds column l % 32 of rows 8 i + 4 (l / 32) + 0..3.  16-bit tiles use
  // the LDS transpose read: each group of 16 lanes reads 4 rows x 16 columns,
  // lane i gets column i.  Its builtin makes the compiler wait for the next
  // tile's copies too, so the reads and their wait are one asm block.  FP32 tiles
  // read single values.
  static FM_DEVICE unsigned col_lane(int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 4)
      return 4 * half * PITCH + ((((lane & 31) >> 2) ^ swz<T, DT>(4 * half)) << 4) + (lane & 3) * 4;
    const int r = 4 * half + ((lane >> 2) & 3), chunk = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    return r * PITCH + ((chunk ^ swz<T, DT>(r)) << 4) + (lane & 1) * 8;
  }
  static FM_DEVICE void cols(unsigned a, int step, Frag (&f)[DT / 32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int dt = 0; dt < DT / 32; ++dt)
          f[dt][e] = *(const __attribute__((address_space(3))) float*)((a ^ ((swz<T, DT>(8 * step + e) ^ (8 * dt)) << 4)) +
                                                                       (8 * step + e) * PITCH);
    } else {
      a += 16 * step * PITCH;
      constexpr unsigned EIGHT = (DT == 128 ? 2 : 1) << 4;  // the swizzle of row r + 8 against row r's
      uintx2_v u[DT / 32][2];
      if constexpr (DT == 64)
        asm volatile(
            "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
            "ds_read_b64_tr_b16 %2, %6\n\tds_read_b64_tr_b16 %3, %7 offset:%8\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(u[0][0]), "=&v"(u[0][1]), "=&v"(u[1][0]), "=&v"(u[1][1])
            : "v"(a), "v"(a ^ EIGHT), "v"(a ^ 64), "v"(a ^ 64 ^ EIGHT), "n"(8 * PITCH));
      else
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
            "ds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
            "ds_read_b64_tr_b16 %4, %12\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
            "ds_read_b64_tr_b16 %6, %14\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(u[0][0]), "=&v"(u[0][1]), "=&v"(u[1][0]), "=&v"(u[1][1]), "=&v"(u[2][0]), "=&v"(u[2][1]),
              "=&v"(u[3][0]), "=&v"(u[3][1])
            : "v"(a), "v"(a ^ EIGHT), "v"(a ^ 64), "v"(a ^ 64 ^ EIGHT), "v"(a ^ 128), "v"(a ^ 128 ^ EIGHT), "v"(a ^ 192),
              "v"(a ^ 192 ^ EIGHT), "n"(8 * PITCH));
#pragma unroll
      for (int dt = 0; dt < DT / 32; ++dt)
        f[dt] = __builtin_bit_cast(Frag, (uintx4_v{u[dt][0][0], u[dt][0][1], u[dt][1][0], u[dt][1][1]}));
    }
  }
};

// Has the compiler wait for these loads here.  Where their first use is inside
// a loop it would wait there in every turn, for the next tile's copies as well.
template <typename F, int N>
FM_DEVICE void arrive(F (&f)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

// The operands of one row and the products with them, for tiles of ROWS rows.
//
// 16-bit inputs, and FP32 heads beyond 64: tiles lie in LDS as they are in memory,
// copied there directly; the FP32 products are FP32 MFMAs.
template <typename T, int DT>
constexpr bool SPLIT = std::is_same<T, float>::value && DT == 64;

template <typename T, int DT, int ROWS, bool SPLITS>
struct Engine {
  typedef Elem<T> E;
  typedef Reads<T, DT> R;
  typedef typename E::Frag Frag;
  static constexpr int N = DT / E::STEP, ND = DT / 32, TILE = ROWS * R::PITCH;

  // The B operand of one row straight from memory: chunk s of the lane's half,
  // zeros where the row is not live or the chunk lies past the head's width.
  struct Held {
    Frag f[N];
  };
  static FM_DEVICE void load(const T* row, bool live, int D, int lane, Held& h) {
    constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const int d = (2 * s + (lane >> 5)) * W;
      const bool ok = live && d < D;  // the row itself is always one of the tensor's
      uintx4_v u = *reinterpret_cast<const uintx4_v*>(row + (d < D ? d : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = ok ? u[e] : 0;
      h.f[s] = __builtin_bit_cast(Frag, u);
    }
  }
  static FM_DEVICE void here(Held& h) { arrive(h.f); }

  // s += 32 rows of a tile (lane address a) times B: a product over the head's
  // width.  The 16-bit forms read four steps' fragments before their products, so
  // that a wave does not wait for LDS at each (32 cycles do not cover a read);
  // FP32 products do.
  static constexpr int AHEAD = 4;
  static FM_DEVICE void products(unsigned a, const Held& b, floatx16& s) {
    Frag f[N];
#pragma unroll
    for (int c0 = 0; c0 < N; c0 += AHEAD) {
#pragma unroll
      for (int c = c0; c < c0 + AHEAD; ++c) f[c] = R::row(a, c);
      if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = c0; c < c0 + AHEAD; ++c) s = E::mma(f[c], b.f[c], s);
    }
  }
  // The same with B in LDS as well.
  static FM_DEVICE void products(unsigned a, unsigned b, floatx16& s) {
    Frag f[N], g[N];
#pragma unroll
    for (int c0 = 0; c0 < N; c0 += AHEAD) {
#pragma unroll
      for (int c = c0; c < c0 + AHEAD; ++c) f[c] = R::row(a, c), g[c] = R::row(b, c);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = c0; c < c0 + AHEAD; ++c) s = E::mma(f[c], g[c], s);
    }
  }

  // acc += (32 rows of a tile)^T times s, a product over the rows.  REST: the
  // second factor in two 16-bit pieces.
  template <bool REST>
  static FM_DEVICE void outer(unsigned a, const floatx16& s, floatx16 (&acc)[ND]) {
#pragma unroll
    for (int c = 0; c < 32 / E::STEP; ++c) {
      const Frag p = E::pack(s, c);
      Frag f[ND];
      R::cols(a, c, f);
      if constexpr (REST && sizeof(T) == 2) {
        const Frag low = E::pack_rest(s, p, c);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = E::mma(f[d], low, acc[d]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = E::mma(f[d], p, acc[d]);
    }
  }
};

// FP32 heads up to 64: every factor as three round-to-nearest bf16 pieces (exact
// to 2^-24) and each product as the six of them of order at most 2, summed in
// FP32 from the smallest: 768 matrix cycles per 32x32x64 where the FP32 MFMA takes
// 2048, at its error.  A block's threads bring the next tile into registers, and
// split it into three planes in LDS once all waves are done with the last one.
// An infinity has no such pieces, and where a product overflows, so may those of
// its factors' remainders, with either sign.  A block that meets a value of 2^36
// or more starts again on FP32 MFMAs: below, scores stay under 2^78 and dS under
// 2^81, so that no value that is split and no single product (2^117) comes near the
// largest one.  (dK sums such products over its rows and overflows where 2^11 of the
// largest meet, as an FP32 sum does: to infinity, as its terms are finite.  At the other end
// a piece may be lost below 2^-126: of values under 2^-102 more than an FP32
// rounding, and never more than 2^-126 of any.)
// 16 x 2500 frames, 8 heads, window 250: forward 250 -> 170 us, dQ 355 -> 270,
// dK / dV 500 -> 335 (there the matrix cores and the vector work, half of it the
// splitting, take turns).
template <int ROWS>
struct Engine<float, 64, ROWS, true> {
  typedef Reads<__bf16, 64> R;
  static constexpr int N = 4, ND = 2, PLANE = ROWS * 128, TILE = 3 * PLANE, UNITS = ROWS / 32;

  struct Held {
    bf16x8 f[3][N];
    float most;  // the largest magnitude
  };
  static FM_DEVICE float size(floatx4 a, floatx4 b, float u) {
#pragma unroll
    for (int e = 0; e < 4; ++e) u = fmaxf(u, fmaxf(fabsf(a[e]), fabsf(b[e])));
    return u;
  }
  static FM_DEVICE void split8(floatx4 lo, floatx4 hi, bf16x8 (&h)[3]) {
    bf16x4 a[3], b[3];
    split3(lo, a[0], a[1], a[2]);
    split3(hi, b[0], b[1], b[2]);
#pragma unroll
    for (int k = 0; k < 3; ++k) h[k] = __builtin_shufflevector(a[k], b[k], 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static FM_DEVICE void load(const float* row, bool live, int D, int lane, Held& h) {
    h.most = 0.0f;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      floatx4 v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = 16 * s + 8 * (lane >> 5) + 4 * u;
        const bool ok = live && d < D;
        v[u] = *reinterpret_cast<const floatx4*>(row + (d < D ? d : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] = ok ? v[u][e] : 0.0f;
      }
      h.most = size(v[0], v[1], h.most);
      bf16x8 p[3];
      split8(v[0], v[1], p);
#pragma unroll
      for (int k = 0; k < 3; ++k) h.f[k][s] = p[k];
    }
  }
  static FM_DEVICE void here(Held& h) {
#pragma unroll
    for (int k = 0; k < 3; ++k) arrive(h.f[k]);
    // Used behind the loop only: else the values would be kept until there.
    asm volatile("" : "+v"(h.most));
  }

  static FM_DEVICE floatx16 six(const bf16x8 (&a)[3], const bf16x8 (&b)[3], floatx16 s) {
    s = fm_mfma32_bf16(a[2], b[0], s);
    s = fm_mfma32_bf16(a[0], b[2], s);
    s = fm_mfma32_bf16(a[1], b[1], s);
    s = fm_mfma32_bf16(a[1], b[0], s);
    s = fm_mfma32_bf16(a[0], b[1], s);
    return fm_mfma32_bf16(a[0], b[0], s);
  }
  static FM_DEVICE void products(unsigned a, const Held& b, floatx16& s) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      bf16x8 f[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) f[k] = R::row(a + k * PLANE, c);
      const bf16x8 g[3] = {b.f[0][c], b.f[1][c], b.f[2][c]};
      s = six(f, g, s);
    }
  }
  // The same with B in LDS as well, in planes of its own size.
  template <int OTHER>
  static FM_DEVICE void products(unsigned a, unsigned b, floatx16& s) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      bf16x8 f[3], g[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) f[k] = R::row(a + k * PLANE, c), g[k] = R::row(b + k * OTHER, c);
      s = six(f, g, s);
    }
  }
  template <bool REST>
  static FM_DEVICE void outer(unsigned a, const floatx16& s, floatx16 (&acc)[ND]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8 p[3], f[3][ND];
      split8(floatx4{s[8 * c], s[8 * c + 1], s[8 * c + 2], s[8 * c + 3]},
             floatx4{s[8 * c + 4], s[8 * c + 5], s[8 * c + 6], s[8 * c + 7]}, p);
#pragma unroll
      for (int k = 0; k < 3; ++k) R::cols(a + k * PLANE, c, f[k]);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const bf16x8 g[3] = {f[0][d], f[1][d], f[2][d]};
        acc[d] = six(g, p, acc[d]);
      }
    }
  }

  // Rows of a tile on their way: thread i holds eight columns of each of UNITS rows.
  struct Flight {
    floatx4 v[UNITS][2];
  };
  template <typename Offset>
  static FM_DEVICE void bring(const void* base, int D, Flight& f, Offset offset) {
    const __amdgpu_buffer_rsrc_t buf = fm_buffer(base, INT_MAX);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int i = u * 256 + threadIdx.x, off = offset(i >> 3);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 8 * (i & 7) + 4 * k;
        f.v[u][k] = fm_buf_load4(buf, off >= 0 && d < D ? off + 4 * d : INT_MIN, 0);
      }
    }
  }
  // Returns the largest magnitude among this lane's values and `most`.
  static FM_DEVICE float publish(const Flight& f, unsigned char* tile, float most) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      most = size(f.v[u][0], f.v[u][1], most);
      asm volatile("" : "+v"(most));
      const int i = u * 256 + threadIdx.x, r = i >> 3;
      bf16x8 p[3];
      split8(f.v[u][0], f.v[u][1], p);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        *reinterpret_cast<bf16x8*>(tile + k * PLANE + r * 128 + (((i & 7) ^ swz<__bf16, 64>(r)) << 4)) = p[k];
    }
    return most;
  }
};

// The dot product of two rows, half of it in each lane half.
template <typename T, int DT>
FM_DEVICE float row_dot(const T* x, const T* y, bool live, int D, int lane) {
  constexpr int W = 16 / (int)sizeof(T);
  float s = 0.0f;
#pragma unroll
  for (int d0 = 0; d0 < DT; d0 += 2 * W) {
    const int d = d0 + (lane >> 5) * W, at = d < D ? d : 0;
    const typename Elem<T>::Frag a = *reinterpret_cast<const typename Elem<T>::Frag*>(x + at);
    const typename Elem<T>::Frag b = *reinterpret_cast<const typename Elem<T>::Frag*>(y + at);
    s = live && d < D ? Elem<T>::dot(a, b, s) : s;
  }
  return s;
}

// Starts the copy of ROWS rows into LDS (global -> LDS, 16 bytes a lane).
// offset(r) is the byte offset of tile row r from `base`, or negative for a
// row that is not there (zeros).
template <typename T, int DT, int ROWS, int WAVES, typename Offset>
FM_DEVICE void load_tile(const void* base, unsigned char* tile, int D, int wave, int lane, Offset offset) {
  constexpr int PITCH = DT * (int)sizeof(T), CPR = PITCH / 16, INSTR = ROWS * PITCH / 1024;
  static_assert(INSTR % WAVES == 0, "whole instructions per wave");
  const __amdgpu_buffer_rsrc_t buf = fm_buffer(base, INT_MAX);
#pragma unroll
  for (int u = 0; u < INSTR / WAVES; ++u) {
    const int i = wave * (INSTR / WAVES) + u;
    const int slot = i * 64 + lane, r = slot / CPR, chunk = (slot % CPR) ^ swz<T, DT>(r);
    const int off = offset(r);
    const bool ok = off >= 0 && chunk * 16 < D * (int)sizeof(T);
    fm_buf_load_lds16(buf, tile + i * 1024, ok ? off + chunk * 16 : INT_MIN, 0);
  }
}

// The sum or maximum of the two lane halves, in both (one register swap).
FM_DEVICE float half_sum(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
FM_DEVICE float half_max(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// The power of two that dS carries as a float16 operand, one for each column of its
// products (a row of dQ, a key of dK: a lane of either half), and with it the sums
// over the column, until their end.  At the start a step is 2^-72: times the largest
// float16 and over 2^21 rows under the smallest.  When a value passes 2^15 the level
// falls until that one lies between 2^8 and 2^9 (for infinities it stays), so that
// a step is at most 2^-32 of the column's largest dS.  (2 x 4095 positions, 16/4
// heads of 128, float16, backward: 683 -> 712 us.)
struct Level {
  int up = 48;
  // Whether any lane's largest magnitude passes 2^15 (called by whole waves).
  FM_DEVICE bool passed(float most) const { return __any(most > 32768.0f); }
  // Returns what the sums and the values are to be multiplied by.
  FM_DEVICE float lower(float most) {
    const int by = most > 32768.0f ? max(__builtin_amdgcn_frexp_expf(most) - 9, 0) : 0;
    up -= by;
    return __builtin_ldexpf(1.0f, -by);
  }
};
FM_DEVICE float column_most(const floatx16& s) {
  float most = fabsf(s[0]);
#pragma unroll
  for (int e = 1; e < 16; ++e) most = fmaxf(most, fabsf(s[e]));
  return half_max(most);
}
template <int ND>
FM_DEVICE void times(floatx16 (&acc)[ND], float f) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] *= f;
}

FM_DEVICE void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What the row kernels (forward, dQ) share: the rows of a block and wave and
// the keys they see.
template <int WQ>
struct Rows {
  int b, kh, len, R, r, t, p, p_lo, p_hi, b_lo, k_lo, k_hi;
  bool live;
  long row_index;  // into [B][T][H]
  FM_DEVICE Rows(const Attn& a, int wq, int lane) {
    b = blockIdx.x / a.KV, kh = blockIdx.x - b * a.KV;
    len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
    R = a.T * a.G;
    // The last rows see the most keys: they start first.
    const int r0 = (gridDim.y - 1 - blockIdx.y) * 32 * WQ, past = a.S - a.T;
    const int w0 = min(r0 + 32 * wq, R - 1), w1 = min(r0 + 32 * wq + 31, R - 1);
    p_lo = past + (int)fm_div(w0, a.by_g);  // the wave's positions
    p_hi = min(past + (int)fm_div(w1, a.by_g), len - 1);
    r = r0 + 32 * wq + (lane & 31);
    t = (int)fm_div(min(r, R - 1), a.by_g);
    p = past + t;
    live = r < R && p < len;
    row_index = ((long)b * a.T + t) * a.H + kh * a.G + (min(r, R - 1) - t * a.G);
    // The block's keys.
    b_lo = past + (int)fm_div(r0, a.by_g);
    const int b_hi = past + (int)fm_div(min(r0 + 32 * WQ, R) - 1, a.by_g);
    k_lo = max(0, b_lo - a.window + 1);
    k_hi = min(b_hi, len - 1);
  }
  template <typename T> FM_DEVICE const T* of(const View& v) const {
    return static_cast<const T*>(v.p) + b * v.batch;
  }
};

// O^T or dQ^T of the WK waves that shared rows but not keys, summed into their
// WK-th parts of the registers each; own: which rows (0 .. 4 / WK - 1).
template <int DT, int WK>
FM_DEVICE void merge(float* lds, floatx16 (&acc)[DT / 32], int own, int wk, int lane, float (&mine)[DT / 2 / WK]) {
  constexpr int N = DT / 2;
  lds += own * WK * N * 64;
#pragma unroll
  for (int i = 0; i < N; ++i) lds[(wk * N + i) * 64 + lane] = acc[i / 16][i % 16];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N / WK; ++i) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WK; ++w) s += lds[(w * N + wk * (N / WK) + i) * 64 + lane];
    mine[i] = s;
  }
}

// A lane's values first .. of a result row (groups of four columns), times f;
// zeros for a row that is not live.
template <typename T, int N>
FM_DEVICE void store_row(T* o, const float (&v)[N], float f, bool live, int first, int half, int D) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const int e = first + i, d = 32 * (e / 16) + 8 * (e % 16 / 4) + 4 * half;
    if (d < D)
      Elem<T>::store4(o + d, live ? v[i] * f : 0.0f, live ? v[i + 1] * f : 0.0f, live ? v[i + 2] * f : 0.0f,
                      live ? v[i + 3] * f : 0.0f);
  }
}

// Starts the copies of the keys and values k0 .. k_hi (at most KEYS) of a head.
template <typename T, int DT, int KEYS, int WAVES = 4>
FM_DEVICE void load_keys(const Attn& a, const T* kp, const T* vp, int k0, int k_hi, unsigned char* at, int wave, int lane) {
  constexpr int TILE = KEYS * DT * (int)sizeof(T);
  const int n = k_hi - k0, ks = (int)(a.k.row * (long)sizeof(T)), vs = (int)(a.v.row * (long)sizeof(T));
  load_tile<T, DT, KEYS, WAVES>(kp + k0 * a.k.row, at, a.D, wave, lane, [&](int r) { return r <= n ? r * ks : -1; });
  load_tile<T, DT, KEYS, WAVES>(vp + k0 * a.v.row, at + TILE, a.D, wave, lane, [&](int r) { return r <= n ? r * vs : -1; });
}

constexpr float BIG = 68719476736.0f;  // 2^36

// KEEP: bytes of LDS that a dK / dV block keeps its keys and values in.
template <typename T, int DT, int WQ, int WK, bool SPLITS, int KEEP = 0>
struct Tiling {
  static constexpr int NB = WK > 1 || sizeof(T) == 4 ? 1 : 2;  // 32-key tiles of a wave
  static constexpr int KEYS = 32 * NB * WK;
  static constexpr int TILE = Engine<T, DT, KEYS, SPLITS>::TILE;
  static constexpr int STAGES = 4 * TILE <= 131072 && !KEEP && !SPLITS ? 2 : 1;
  static constexpr int MERGE = WK > 1 ? WQ * WK * DT * 128 : 0;  // room for the waves' results
  static constexpr int LDS = std::max(KEEP + 2 * STAGES * TILE, MERGE);
};

// The same call, as something that the compiler does not recognise: what a second
// form shares with the first would else be held in registers all through it.
FM_DEVICE Attn again(Attn a) {
  int zero;
  asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
  for (const void** p : {&a.q.p, &a.k.p, &a.v.p, &a.dout.p, &a.o}) *p = static_cast<const char*>(*p) + zero;
  for (int* n : {&a.B, &a.T, &a.S, &a.H, &a.KV, &a.G, &a.D, &a.window}) *n += zero;
  a.lengths = a.lengths ? a.lengths + zero : nullptr;
  return a;
}

// A kernel's LDS: what either of its forms takes.
template <typename T, int DT, template <bool> class Form>
constexpr int lds_bytes() {
  if constexpr (SPLIT<T, DT>) return std::max(Form<true>::BYTES, Form<false>::BYTES);
  else return Form<false>::BYTES;
}

// Blocks per CU that the registers are held to.  At two (256 a lane) all of them
// are vector registers and no result passes through accumulation registers; the
// kernels that need more (heavy) run one block.
constexpr int blocks(int lds, bool heavy) { return lds > 81920 || heavy ? 1 : 2; }

// The key and value tiles of a row block (forward, dQ) on their way.
template <typename T, int DT, int KEYS, bool SPLITS>
struct KeyTiles {
  FM_DEVICE void start(const Attn& a, const T* kp, const T* vp, int k0, int k_hi, unsigned char* at, int wave, int lane) {
    load_keys<T, DT, KEYS>(a, kp, vp, k0, k_hi, at, wave, lane);
  }
};
template <typename T, int DT, int KEYS>
struct KeyTiles<T, DT, KEYS, true> {
  typedef Engine<T, DT, KEYS, true> G;
  typename G::Flight k, v;
  FM_DEVICE void start(const Attn& a, const T* kp, const T* vp, int k0, int k_hi, unsigned char*, int, int) {
    const int n = k_hi - k0, ks = (int)(a.k.row * (long)sizeof(T)), vs = (int)(a.v.row * (long)sizeof(T));
    G::bring(kp + k0 * a.k.row, a.D, k, [&](int r) { return r <= n ? r * ks : -1; });
    G::bring(vp + k0 * a.v.row, a.D, v, [&](int r) { return r <= n ? r * vs : -1; });
  }
  FM_DEVICE float publish(unsigned char* at, float most) {
    most = G::publish(v, at + G::TILE, G::publish(k, at, most));
    lds_barrier();
    return most;
  }
};

// The forms of a kernel return whether they are done; the split one is not where
// it met a value that wants FP32 products.
template <typename T, int DT, int WQ, int WK>
struct Forward {
  template <bool SPLITS>
  struct Form {
    static constexpr int BYTES = Tiling<T, DT, WQ, WK, SPLITS>::LDS + (WK > 1 ? 4 * 2 * 128 : 0);
  };
  static constexpr int LDS = lds_bytes<T, DT, Form>();
  static constexpr int BLOCKS = SPLIT<T, DT> && WK == 1 ? 3 : blocks(LDS, false);
  template <bool SPLITS> static FM_DEVICE bool run(const Attn& a, unsigned char* lds);
};
template <typename T, int DT, int WQ, int WK>
__global__ __launch_bounds__(256, (Forward<T, DT, WQ, WK>::BLOCKS)) void attention_forward_kernel(Attn a) {
  // One array for all of the block's LDS: among several the compiler tells the
  // direct copies' targets apart, and then waits for all copies at every read.
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Forward<T, DT, WQ, WK>::LDS];
  if constexpr (SPLIT<T, DT>) {
    if (!Forward<T, DT, WQ, WK>::template run<true>(a, lds)) Forward<T, DT, WQ, WK>::template run<false>(again(a), lds);
  } else {
    Forward<T, DT, WQ, WK>::template run<false>(a, lds);
  }
}

template <typename T, int DT, int WQ, int WK>
template <bool SPLITS>
FM_DEVICE bool Forward<T, DT, WQ, WK>::run(const Attn& a, unsigned char* lds) {
  typedef Tiling<T, DT, WQ, WK, SPLITS> L;
  typedef Engine<T, DT, L::KEYS, SPLITS> G;
  constexpr int ND = DT / 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave % WQ, wk = wave / WQ, half = lane >> 5;
  const Rows<WQ> w(a, wq, lane);
  typedef typename G::R R;
  const unsigned row_lane = R::row_lane(lane), col_lane = R::col_lane(lane);

  typename G::Held q;
  G::load(w.template of<T>(a.q) + w.t * a.q.row + (w.kh * a.G + (min(w.r, w.R - 1) - w.t * a.G)) * a.q.head, w.live, a.D, lane, q);
  floatx16 acc[ND] = {};
  float m = -INFINITY, l = 0.0f;  // l: of this lane's keys only

  int tiles = w.k_hi >= w.k_lo ? (w.k_hi - w.k_lo) / L::KEYS + 1 : 0, first = 0;
  if (a.splits > 1) {
    const int per = (tiles + a.splits - 1) / a.splits;
    first = blockIdx.z * per;
    tiles = min(tiles, first + per);
  }
  const T* kp = w.template of<T>(a.k) + w.kh * a.k.head;
  const T* vp = w.template of<T>(a.v) + w.kh * a.v.head;
  KeyTiles<T, DT, L::KEYS, SPLITS> next;
  float most = 0.0f;
  auto load = [&](int i) {
    next.start(a, kp, vp, w.k_lo + i * L::KEYS, w.k_hi, lds + (i - first) % L::STAGES * 2 * L::TILE, wave, lane);
  };
  if (first < tiles) load(first);
  G::here(q);
  for (int i = first; i < tiles; ++i) {
    tile_barrier();  // tile i is there, and every wave is past tile i - 1
    if constexpr (SPLITS) most = next.publish(lds, most);
    if ((L::STAGES == 2 || SPLITS) && i + 1 < tiles) load(i + 1);
    const unsigned char* kt = lds + (i - first) % L::STAGES * 2 * L::TILE;
    const unsigned char* vt = kt + L::TILE;
#pragma unroll
    for (int nb = 0; nb < L::NB; ++nb) {
      const int row = (wk * L::NB + nb) * 32, k0 = w.k_lo + i * L::KEYS + row;
      if (k0 > w.p_hi || k0 + 31 <= w.p_lo - a.window) continue;  // nothing that this wave sees
      floatx16 s = {};
      G::products(R::fresh(R::lds(kt) + row * R::PITCH + row_lane), q, s);
      if (k0 + 31 > w.p_lo || k0 <= w.p_hi - a.window || k0 + 31 > w.k_hi) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = k0 + 8 * (e >> 2) + 4 * half + (e & 3);
          s[e] = key <= w.p && key > w.p - a.window && key <= w.k_hi ? s[e] : -INFINITY;
        }
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top = half_max(top) * a.scale2;
      // m is a reference, not the maximum itself: it follows once a score passes it
      // by SLACK, so that the accumulators are rescaled a few times a row and not
      // in most tiles.  Until then exponentials reach 2^SLACK, far from any limit.
      if (__any(top > m + SLACK<T>)) {
        const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - (up == -INFINITY ? 0.0f : up));
        m = up;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[d][e] *= f;
      }
      const float sub = m == -INFINITY ? 0.0f : m - UP<T>;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, -sub));
        l += s[e];
      }
      G::template outer<false>(R::fresh(R::lds(vt) + row * R::PITCH + col_lane), s, acc);
    }
    if (L::STAGES == 1 && !SPLITS && i + 1 < tiles) {
      tile_barrier();
      load(i + 1);
    }
  }
  if constexpr (SPLITS)
    if (__syncthreads_or(fmaxf(most, q.most) >= BIG)) return false;
  l = half_sum(l);

  constexpr int MINE = DT / 2 / WK;
  float mine[MINE];
  if constexpr (WK > 1) {
    float(*ml)[WK][32] = reinterpret_cast<float(*)[WK][32]>(lds + L::LDS) + 2 * wq;
    if (half == 0) ml[0][wk][lane] = m, ml[1][wk][lane] = l;
    __syncthreads();
    const float own = m;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int u = 0; u < WK; ++u) m = fmaxf(m, ml[0][u][lane & 31]);
    const float sub = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < WK; ++u) l += ml[1][u][lane & 31] * __builtin_amdgcn_exp2f(ml[0][u][lane & 31] - sub);
    const float f = __builtin_amdgcn_exp2f(own - sub);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][e] *= f;
    merge<DT, WK>(reinterpret_cast<float*>(lds), acc, wq, wk, lane, mine);
  } else {
#pragma unroll
    for (int i = 0; i < MINE; ++i) mine[i] = acc[i / 16][i % 16];
  }
  if (w.r >= w.R) return true;
  const bool writes = half == 0 && wk == 0;
  if (a.splits > 1) {
    const long at = ((long)blockIdx.z * gridDim.x + blockIdx.x) * w.R + w.r;
    if (writes) *reinterpret_cast<floatx2_v*>(a.part_ml + 2 * at) = floatx2_v{m, l};
    store_row(a.part_o + at * DT, mine, 1.0f, true, wk * MINE, half, DT);
    return true;
  }
  // A row that sees nothing (padding) gives zeros.
  const bool some = w.live && l != 0.0f;
  if (writes) a.lse[w.row_index] = some ? m + (log2f(l) - UP<T>) : -INFINITY;
  store_row(static_cast<T*>(a.out) + w.row_index * a.D, mine, 1.0f / l, some, wk * MINE, half, a.D);
  return true;
}

// Joins the parts of a split forward: one wave per row, lane d of DT columns, eight
// parts in flight.  8 x 16 rows of 15 parts: 4 us (behind 14 for the parts, 8000 keys
// of 4 heads each at 4.7 TB/s).
template <typename T, int DT>
__global__ __launch_bounds__(256) void attention_join_kernel(Attn a) {
  const int lane = threadIdx.x & 63, R = a.T * a.G;
  const long rows = (long)a.B * a.KV * R, at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const int seq = (int)(at / R), r = (int)(at - (long)seq * R), b = seq / a.KV, kh = seq - b * a.KV;
  const int t = (int)fm_div(r, a.by_g);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
  const bool live = a.S - a.T + t < len;
  // Lane s holds split s's maximum and sum (at most 64 splits).
  floatx2_v ml{-INFINITY, 0.0f};
  if (lane < a.splits) ml = *reinterpret_cast<const floatx2_v*>(a.part_ml + 2 * (lane * rows + at));
  float m = ml[0];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float weight = __builtin_amdgcn_exp2f(ml[0] - (m == -INFINITY ? 0.0f : m));
  float l = ml[1] * weight;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, 64);
  float o[DT / 64] = {};
  constexpr int AHEAD = 8;
  for (int s = 0; s < a.splits; s += AHEAD) {
    float v[AHEAD][DT / 64];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int d = 0; d < DT / 64; ++d) v[u][d] = a.part_o[(min(s + u, a.splits - 1) * rows + at) * DT + 64 * d + lane];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const float f = __shfl(weight, min(s + u, 63), 64);
#pragma unroll
      for (int d = 0; d < DT / 64; ++d) o[d] = s + u < a.splits ? fmaf(v[u][d], f, o[d]) : o[d];
    }
  }
  const long row = ((long)b * a.T + t) * a.H + kh * a.G + (r - t * a.G);
  if (lane == 0) a.lse[row] = live && l != 0.0f ? m + (log2f(l) - UP<T>) : -INFINITY;
  T* out = static_cast<T*>(a.out) + row * a.D;
#pragma unroll
  for (int u = 0; u < DT / 64; ++u)
    if (64 * u + lane < a.D) out[64 * u + lane] = (T)(live && l != 0.0f ? o[u] / l : 0.0f);
}

// dQ, and rowsum(dO O) for the dK / dV kernel: rows and keys as the forward.
//
// 16-bit inputs: dS is two 16-bit pieces here (a fourth product), as its own
// rounding would put dQ at 1.5 times the error that rounding its result has.  And
// rowsum(dO O) from the rounded O is only nearly the sum over P dP; the sum of dS,
// zero but for that, puts it right for the dK / dV kernel.  Where a row sees few
// keys it would also be most of dQ's error (1.5 times the rounding's with 4 keys of
// ordinary scores, less than 1.1 from 32 on): blocks with such rows go over their
// keys twice (backward of 16 x 2500 frames without it / up to 31 keys / up to 63, under
// windows of 31, 48 and 63: 151 / 162 / 162, 158 / 161 / 172, 159 / 163 / 175 us; of 13
// frames 12 / 13 / 13).  Rows of more keys with one large probability keep it (1.4 times at 0.3, 2.2
// at 0.65): which they are is known after the pass only, and a second one for all
// would be 12-24% of the backward (16 x 2500, window 250: 201 -> 230 us).
template <typename T, int DT, int WQ, int WK>
struct QueryGradient {
  template <bool SPLITS>
  struct Form {
    static constexpr int BYTES = Tiling<T, DT, WQ, WK, SPLITS>::LDS + (WK > 1 ? 4 * 128 : 0);
  };
  static constexpr int LDS = lds_bytes<T, DT, Form>();
  static constexpr int BLOCKS = blocks(LDS, sizeof(T) == 4 && DT == 128);
  template <bool SPLITS> static FM_DEVICE bool run(const Attn& a, unsigned char* lds);
};
template <typename T, int DT, int WQ, int WK>
__global__ __launch_bounds__(256, (QueryGradient<T, DT, WQ, WK>::BLOCKS)) void attention_dq_kernel(Attn a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[QueryGradient<T, DT, WQ, WK>::LDS];
  if constexpr (SPLIT<T, DT>) {
    if (!QueryGradient<T, DT, WQ, WK>::template run<true>(a, lds)) QueryGradient<T, DT, WQ, WK>::template run<false>(again(a), lds);
  } else {
    QueryGradient<T, DT, WQ, WK>::template run<false>(a, lds);
  }
}

template <typename T, int DT, int WQ, int WK>
template <bool SPLITS>
FM_DEVICE bool QueryGradient<T, DT, WQ, WK>::run(const Attn& a, unsigned char* lds) {
  typedef Tiling<T, DT, WQ, WK, SPLITS> L;
  typedef Engine<T, DT, L::KEYS, SPLITS> G;
  constexpr int ND = DT / 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave % WQ, wk = wave / WQ, half = lane >> 5;
  const Rows<WQ> w(a, wq, lane);
  typedef typename G::R R;
  const unsigned row_lane = R::row_lane(lane), col_lane = R::col_lane(lane);

  const T* kp = w.template of<T>(a.k) + w.kh * a.k.head;
  const T* vp = w.template of<T>(a.v) + w.kh * a.v.head;
  const int tiles = w.k_hi >= w.k_lo ? (w.k_hi - w.k_lo) / L::KEYS + 1 : 0;
  KeyTiles<T, DT, L::KEYS, SPLITS> next;
  float most = 0.0f;
  auto load = [&](int i) {
    next.start(a, kp, vp, w.k_lo + i * L::KEYS, w.k_hi, lds + i % L::STAGES * 2 * L::TILE, wave, lane);
  };
  if (tiles) load(0);

  typename G::Held q, g;
  const int head = w.kh * a.G + (min(w.r, w.R - 1) - w.t * a.G);
  const T* grad = w.template of<T>(a.dout) + w.t * a.dout.row + head * a.dout.head;
  G::load(w.template of<T>(a.q) + w.t * a.q.row + head * a.q.head, w.live, a.D, lane, q);
  G::load(grad, w.live, a.D, lane, g);
  float delta = half_sum(row_dot<T, DT>(grad, static_cast<const T*>(a.o) + w.row_index * a.D, w.live, a.D, lane));
  // A row without keys takes every probability as zero.
  float lse = w.live ? a.lse[w.row_index] : INFINITY;
  lse = lse == -INFINITY ? INFINITY : lse;
  float rest = 0.0f;  // the sum of dS: what the rounding of O took from delta

  Level level;

  // The row's sum over both lane halves and all the waves that share it.
  auto total = [&]() {
    float sum = half_sum(SCALED<T> ? __builtin_ldexpf(rest, -level.up) : rest);
    if constexpr (WK > 1) {
      float(*rests)[32] = reinterpret_cast<float(*)[32]>(lds + L::LDS) + WK * wq;
      if (half == 0) rests[wk][lane] = sum;
      __syncthreads();
      sum = 0.0f;
#pragma unroll
      for (int u = 0; u < WK; ++u) sum += rests[u][lane & 31];
    }
    return sum;
  };

  floatx16 acc[ND] = {};
  G::here(q), G::here(g);
  float row_stats[2] = {lse, delta};
  arrive(row_stats);
  lse = row_stats[0], delta = row_stats[1];
  // With few keys (some row sees fewer than FEW) a first pass makes delta exact.
  constexpr int FEW = 32;
  bool first = sizeof(T) == 2 && tiles > 0 && min(w.b_lo + 1, a.window) < FEW;
  for (;; first = false) {
    for (int i = 0; i < tiles; ++i) {
      tile_barrier();
      if constexpr (SPLITS) most = next.publish(lds, most);
      if ((L::STAGES == 2 || SPLITS) && i + 1 < tiles) load(i + 1);
      const unsigned char* kt = lds + i % L::STAGES * 2 * L::TILE;
  #pragma unroll
      for (int nb = 0; nb < L::NB; ++nb) {
        const int row = (wk * L::NB + nb) * 32, k0 = w.k_lo + i * L::KEYS + row;
        if (k0 > w.p_hi || k0 + 31 <= w.p_lo - a.window) continue;
        floatx16 s = {}, dp = {};
        const unsigned at = R::fresh(R::lds(kt) + row * R::PITCH + row_lane);
        G::products(at, q, s);
        G::products(at + L::TILE, g, dp);
        const bool edge = k0 + 31 > w.p_lo || k0 <= w.p_hi - a.window || k0 + 31 > w.k_hi;
        const float sub = SCALED<T> ? lse - (float)level.up : lse;
  #pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, -sub));
          s[e] = p * (dp[e] - delta);
        }
        if (edge) {
  #pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = k0 + 8 * (e >> 2) + 4 * half + (e & 3);
            s[e] = key <= w.p && key > w.p - a.window && key <= w.k_hi && w.live ? s[e] : 0.0f;
          }
        }
        if constexpr (SCALED<T>) {
          const float top = column_most(s);
          if (level.passed(top)) {
            const float f = level.lower(top);
            rest *= f;
            times(acc, f);
  #pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= f;
          }
        }
  #pragma unroll
        for (int e = 0; e < 16; ++e) rest += s[e];
        if (!first) G::template outer<true>(R::fresh(R::lds(kt) + row * R::PITCH + col_lane), s, acc);
      }
      if (L::STAGES == 1 && !SPLITS && i + 1 < tiles) {
        tile_barrier();
        load(i + 1);
      }
    }
    if (!first) break;
    tile_barrier();  // every wave is past the last tile
    load(0);
    rest = total();
    delta += rest, rest = 0.0f;
  }
  if constexpr (SPLITS)
    if (__syncthreads_or(fmaxf(most, fmaxf(q.most, g.most)) >= BIG)) return false;
  rest = total();
  if constexpr (SCALED<T>) times(acc, __builtin_ldexpf(1.0f, -level.up));
  constexpr int MINE = DT / 2 / WK;
  float mine[MINE];
  if constexpr (WK > 1) {
    merge<DT, WK>(reinterpret_cast<float*>(lds), acc, wq, wk, lane, mine);
  } else {
#pragma unroll
    for (int i = 0; i < MINE; ++i) mine[i] = acc[i / 16][i % 16];
  }
  if (w.r >= w.R) return true;
  if (half == 0 && wk == 0) {
    a.stats[w.row_index] = lse - P_UP<T>;
    a.stats[(long)a.B * a.T * a.H + w.row_index] = sizeof(T) == 2 ? delta + rest : delta;
  }
  store_row(static_cast<T*>(a.out) + w.row_index * a.D, mine, a.scale, w.live, wk * MINE, half, a.D);
  return true;
}

// The query and gradient tiles of a key block on their way in registers.
template <typename T, int DT, int ROWS, bool SPLITS>
struct RowTiles {};
template <typename T, int DT, int ROWS>
struct RowTiles<T, DT, ROWS, true> {
  typename Engine<T, DT, ROWS, true>::Flight q, g;
};

// dK and dV of 32 keys a wave over every row that sees them.  WK waves take 32
// keys each and share the row tiles (many keys), WR waves take the same 32 keys
// and a WR-th of each row tile.
//
// The keys and values stay in registers as operands, but for 16-bit heads of
// 128: two accumulators of 64 registers each leave no room for them within the
// 256 of two waves per SIMD, without which products, exponentials and LDS reads
// follow one another.  Those blocks read them from LDS: four waves with two
// blocks to a CU, or eight waves where that many blocks would all run at once and
// the longest (the first keys of a sequence without a window) set the time.  2 x
// 4095 positions, 16/4 heads: 740 us from registers, 540 / 404 from LDS with four
// / eight waves; 16 heads x 2 x 2048: 190, 102 / 126.  Backward with four / eight
// waves (the rule takes eight up to 512 blocks): 8 heads x 2048 (256 blocks) 121 / 99
// us, 16 x 2048 (512) 129 / 116, 32 x 2048 (1024) 195 / 211, 64 x 2048 363 / 396; with a
// window of 250, where blocks are alike, 8 x 2500 (320) 44 / 52, 32 x 250 (128) 26 / 24,
// 128 x 250 (512) 39 / 44, 32 x 2500 (1280) 114 / 133.
template <typename T, int DT>
constexpr bool HELD = sizeof(T) == 2 && DT == 128;
//
// The rounding of P and dS to 16 bits puts dV and dK at 1.4 times the error of
// rounding the results.  Sums over few rows, where chance adds to that, have them
// in two pieces; a block of that many rows is one or two tiles long (backward of 16 x
// 13, 100 and 250 positions, never / up to 128 rows / up to 512: 13.0 / 13.4 / 13.4, 16.9 /
// 17.7 / 17.8, 25.2 / 25.6 / 26.8 us; 16 x 2500 under a window of 100: 172 / 170 / 184).
constexpr int FEW_ROWS = 128;
template <typename T, int DT, int WK, int WR>
struct KeyGradients {
  template <bool SPLITS>
  struct Form {
    static constexpr int KEEP = SPLITS ? Engine<T, DT, 32 * WK, SPLITS>::TILE : HELD<T, DT> ? 2 * 32 * WK * DT * 2 : 0;
    typedef Tiling<T, DT, WK, WR, SPLITS, KEEP> L;
    static constexpr int TURNS = SPLITS ? 2 : L::STAGES;
    static constexpr int BYTES = L::LDS + TURNS * 2 * L::KEYS * 4;
  };
  static constexpr int LDS = lds_bytes<T, DT, Form>();
  static constexpr int BLOCKS = HELD<T, DT> ? 2 : blocks(LDS, sizeof(T) == 4 && DT == 128);
  template <bool SPLITS> static FM_DEVICE bool run(const Attn& a, unsigned char* lds);
};
template <typename T, int DT, int WK, int WR>
__global__ __launch_bounds__(64 * WK * WR, (KeyGradients<T, DT, WK, WR>::BLOCKS)) void attention_dkv_kernel(Attn a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[KeyGradients<T, DT, WK, WR>::LDS];
  if constexpr (SPLIT<T, DT>) {
    if (!KeyGradients<T, DT, WK, WR>::template run<true>(a, lds)) KeyGradients<T, DT, WK, WR>::template run<false>(again(a), lds);
  } else {
    KeyGradients<T, DT, WK, WR>::template run<false>(a, lds);
  }
}

template <typename T, int DT, int WK, int WR>
template <bool SPLITS>
FM_DEVICE bool KeyGradients<T, DT, WK, WR>::run(const Attn& a, unsigned char* lds) {
  typedef Form<SPLITS> F;
  typedef typename F::L L;  // rows in the place of keys
  constexpr int KEEP = F::KEEP, TURNS = F::TURNS, WAVES = WK * WR;
  constexpr int ND = DT / 32, ROWS = L::KEYS;
  typedef Engine<T, DT, ROWS, SPLITS> G;
  float(*stat)[2][ROWS] = reinterpret_cast<float(*)[2][ROWS]>(lds + L::LDS);  // [stage]: lse, rowsum(dO O)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wk = wave % WK, wr = wave / WK, half = lane >> 5;
  typedef typename G::R R;
  const unsigned row_lane = R::row_lane(lane), col_lane = R::col_lane(lane);
  const int b = blockIdx.x / a.KV, kh = blockIdx.x - b * a.KV;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S, past = a.S - a.T;
  // The first keys are seen by the most rows and start first.
  const int k0 = (int)blockIdx.y * 32 * WK, w0 = k0 + 32 * wk, key = w0 + (lane & 31);
  const bool live = key < len;
  // Rows of the positions that see any of the block's keys.
  const int p_lo = max(k0, past);
  const int p_hi = min((long)min(k0 + 32 * WK, len) - 1 + a.window - 1, (long)len - 1);
  const int r_lo = (p_lo - past) * a.G, r_hi = (p_hi - past + 1) * a.G - 1;
  const int tiles = k0 < len && p_hi >= p_lo ? (r_hi - r_lo) / ROWS + 1 : 0;
  const bool few = sizeof(T) == 2 && r_hi - r_lo < FEW_ROWS;

  const T* qp = static_cast<const T*>(a.q.p) + b * a.q.batch + kh * a.G * a.q.head;
  const T* gp = static_cast<const T*>(a.dout.p) + b * a.dout.batch + kh * a.G * a.dout.head;
  RowTiles<T, DT, ROWS, SPLITS> next;
  float most = 0.0f;
  auto load = [&](int i) {
    const int r0 = r_lo + i * ROWS, t0 = (int)fm_div(r0, a.by_g), stage = i % TURNS;
    auto offset = [&](const View& v) {
      return [&, rs = (int)(v.row * (long)sizeof(T)), hs = (int)(v.head * (long)sizeof(T))](int u) {
        const int r = r0 + u;
        if (r > r_hi) return -1;
        const int t = (int)fm_div(r, a.by_g);
        return (t - t0) * rs + (r - t * a.G) * hs;
      };
    };
    if constexpr (SPLITS) {
      G::bring(qp + t0 * a.q.row, a.D, next.q, offset(a.q));
      G::bring(gp + t0 * a.dout.row, a.D, next.g, offset(a.dout));
    } else {
      unsigned char* at = lds + KEEP + stage * 2 * L::TILE;
      load_tile<T, DT, ROWS, WAVES>(qp + t0 * a.q.row, at, a.D, wave, lane, offset(a.q));
      load_tile<T, DT, ROWS, WAVES>(gp + t0 * a.dout.row, at + L::TILE, a.D, wave, lane, offset(a.dout));
    }
    // The rows' statistics, by direct copies as well: a value that passed through
    // registers would make this tile's copies be waited for.  A row past the last
    // reads zeros, which its zero operands leave without effect.
    const long first = ((long)b * a.T + t0) * a.H + kh * a.G;
    constexpr int CHUNKS = ROWS < 64 ? 1 : ROWS / 64;  // of 64 rows, or one of 32
    for (int u = wave; u < 2 * CHUNKS; u += WAVES) {
      const int which = u / CHUNKS, v = u % CHUNKS * 64 + lane, r = r0 + v, t = (int)fm_div(r, a.by_g);
      if (v < ROWS)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            fm_buffer(a.stats + which * ((long)a.B * a.T * a.H) + first, INT_MAX),
            (__attribute__((address_space(3))) void*)&stat[stage][which][u % CHUNKS * 64], 4,
            r <= r_hi ? ((t - t0) * a.H + r - t * a.G) * 4 : INT_MIN, 0, 0, 0);
    }
  };
  // From the last rows back: every block of a head sees those, so blocks that run
  // at the same time read the same rows.
  if (tiles) load(tiles - 1);
  typename G::Held kf, vf;
  const int at_key = min(key, a.S - 1);
  const T* kp = static_cast<const T*>(a.k.p) + b * a.k.batch + kh * a.k.head;
  const T* vp = static_cast<const T*>(a.v.p) + b * a.v.batch + kh * a.v.head;
  if constexpr (SPLITS) {
    G::load(kp + at_key * a.k.row, live, a.D, lane, kf);
    G::here(kf);
    typedef Engine<T, DT, 32 * WK, true> V;
    typename V::Flight values;
    const int n = min(len, k0 + 32 * WK) - 1 - k0, vs = (int)(a.v.row * (long)sizeof(T));
    V::bring(vp + k0 * a.v.row, a.D, values, [&](int r) { return r <= n ? r * vs : -1; });
    most = V::publish(values, lds, kf.most);
  } else if constexpr (KEEP > 0) {
    // The first tile's barrier waits for these copies; where there is none they would
    // still be on their way when the results take their place.
    if (tiles) load_keys<T, DT, 32 * WK, WAVES>(a, kp, vp, k0, min(len, k0 + 32 * WK) - 1, lds, wave, lane);
  } else {
    G::load(kp + at_key * a.k.row, live, a.D, lane, kf);
    G::load(vp + at_key * a.v.row, live, a.D, lane, vf);
    G::here(kf), G::here(vf);
  }
  floatx16 ak[ND] = {}, av[ND] = {};
  Level level;  // of dS; the probabilities' own part of it is P_UP
  for (int i = tiles - 1; i >= 0; --i) {
    tile_barrier();
    if constexpr (SPLITS) {
      most = G::publish(next.g, lds + KEEP + L::TILE, G::publish(next.q, lds + KEEP, most));
      lds_barrier();
    }
    if ((L::STAGES == 2 || SPLITS) && i > 0) load(i - 1);
    const int stage = i % TURNS;
    const unsigned char* qt = lds + KEEP + (SPLITS ? 0 : stage * 2 * L::TILE);
#pragma unroll
    for (int nb = 0; nb < L::NB; ++nb) {
      const int row = (wr * L::NB + nb) * 32, r0 = r_lo + i * ROWS + row;
      if (r0 > r_hi) continue;
      const int lo = past + (int)fm_div(r0, a.by_g), hi = past + (int)fm_div(min(r0 + 31, r_hi), a.by_g);
      if (w0 > hi || w0 + 31 <= lo - a.window) continue;  // no row here sees these keys
      floatx16 s = {}, dp = {};
      const unsigned at = R::fresh(R::lds(qt) + row * R::PITCH + row_lane);
      if constexpr (SPLITS) {
        G::products(at, kf, s);
        G::template products<KEEP / 3>(at + L::TILE, R::fresh(R::lds(lds) + 32 * wk * R::PITCH + row_lane), dp);
      } else if constexpr (KEEP > 0) {
        const unsigned held = R::fresh(R::lds(lds) + 32 * wk * R::PITCH + row_lane);
        G::products(at, held, s);
        G::products(at + L::TILE, held + KEEP / 2, dp);
      } else {
        G::products(at, kf, s);
        G::products(at + L::TILE, vf, dp);
      }
      // Rows past the last are zeros, whose products with infinities are not.
      const bool edge = w0 + 31 > lo || w0 <= hi - a.window || r0 + 31 > r_hi;
      const float f = SCALED<T> ? __builtin_ldexpf(1.0f, level.up - (int)P_UP<T>) : 1.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const floatx4 lse = *reinterpret_cast<const floatx4*>(&stat[stage][0][row + 8 * g + 4 * half]);
        const floatx4 delta = *reinterpret_cast<const floatx4*>(&stat[stage][1][row + 8 * g + 4 * half]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.scale2, -lse[e]));
          s[4 * g + e] = p;
          dp[4 * g + e] = p * (SCALED<T> ? (dp[4 * g + e] - delta[e]) * f : dp[4 * g + e] - delta[e]);
        }
      }
      if (edge) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = r0 + 8 * (e >> 2) + 4 * half + (e & 3), p = past + (int)fm_div(r, a.by_g);
          const bool ok = key <= p && key > p - a.window && r <= r_hi;
          s[e] = ok ? s[e] : 0.0f;
          dp[e] = ok ? dp[e] : 0.0f;
        }
      }
      if constexpr (SCALED<T>) {
        const float top = column_most(dp);
        if (level.passed(top)) {
          const float by = level.lower(top);
          times(ak, by);
#pragma unroll
          for (int e = 0; e < 16; ++e) dp[e] *= by;
        }
      }
      const unsigned to = R::fresh(R::lds(qt) + row * R::PITCH + col_lane);
#pragma unroll 1
      for (int pieces = few ? 2 : 1;;) {
        G::template outer<false>(to + L::TILE, s, av);
        G::template outer<false>(to, dp, ak);
        if (sizeof(T) == 4 || --pieces == 0) break;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] -= (float)(T)s[e], dp[e] -= (float)(T)dp[e];
      }
    }
    if (L::STAGES == 1 && !SPLITS && i > 0) {
      tile_barrier();
      load(i - 1);
    }
  }
  if constexpr (SPLITS)
    if (__syncthreads_or(most >= BIG)) return false;
  if constexpr (SCALED<T>) times(ak, __builtin_ldexpf(1.0f, -level.up));
  constexpr int MINE = DT / 2 / WR;
  const long row_index = ((long)b * a.S + key) * a.KV + kh;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    floatx16(&acc)[ND] = which ? av : ak;
    float mine[MINE];
    if constexpr (WR > 1) {
      __syncthreads();
      merge<DT, WR>(reinterpret_cast<float*>(lds), acc, wk, wr, lane, mine);
    } else {
#pragma unroll
      for (int i = 0; i < MINE; ++i) mine[i] = acc[i / 16][i % 16];
    }
    if (key < a.S)  // padding takes no gradient
      store_row(static_cast<T*>(which ? a.dv : a.dk) + row_index * a.D, mine, which ? __builtin_exp2f(-P_UP<T>) : a.scale, live, wr * MINE,
                half, a.D);
  }
  return true;
}

int check(const Attn& a, int dtype) {
  if (a.B < 0 || a.T < 0 || a.S < 0 || a.H <= 0 || a.KV <= 0 || a.D <= 0 || a.window <= 0 || !(a.scale > 0.0f) ||
      a.scale2 == INFINITY || a.H % a.KV || a.T > a.S || dtype < DT_F32 || dtype > DT_F16)
    return FM_BAD_ARGUMENT;
  const int unit = dtype == DT_F32 ? 4 : 8, size = dtype == DT_F32 ? 4 : 2;
  if (a.D > 128 || a.D % unit) return FM_UNSUPPORTED;
  // A grid holds 65535 blocks of 32 rows or keys and 2^23 sequences (heads: offsets
  // of a tile's statistics).
  if ((long)a.T * a.G > 32l * 65535 || a.S > 32 * 65535 || (long)a.B * a.KV > 1 << 23 || a.H > 1 << 20) return FM_UNSUPPORTED;
  for (const View* v : {&a.q, &a.k, &a.v, &a.dout}) {
    if (!v->p) continue;
    // 16-byte rows, and a tile's rows within reach of 32-bit offsets.
    if ((reinterpret_cast<uintptr_t>(v->p) & 15) || v->batch % unit || v->row % unit || v->head % unit) return FM_UNSUPPORTED;
    if (v->batch < 0 || v->row < 0 || v->head < 0) return FM_UNSUPPORTED;
    if (v->row > INT_MAX / size / 256 || v->head > INT_MAX / size / 2 / a.G) return FM_UNSUPPORTED;
  }
  return FM_OK;
}

// Key splits of the forward: a call of few rows over many keys (single tokens)
// has one block per 32 rows and key head; its keys are cut until some 512
// blocks run, at least four tiles (of 128 keys) each.
int forward_splits(const Attn& a) {
  const long blocks = (long)a.B * a.KV * fm_ceil_div((long)a.T * a.G, 32);
  const int tiles = fm_ceil_div(std::min<long>(a.S, (long)a.window + a.T - 1), 128);
  return (int)std::max<long>(1, std::min<long>({tiles / 4, 512 / std::max<long>(blocks, 1), 64}));
}

// How many of a block's four waves take rows (or keys) of their own, the rest
// sharing them: four where that leaves about three blocks a CU, two where one
// is left for each, else one.  Backward with one / two / four, 64 channels, window
// 250, bfloat16: 8 heads x 1000 (125 blocks of 64 rows) 20 / 23 / 35 us, 8 x 2500 (320) 39
// / 30 / 36, 8 x 10000 (1264; 632 of 128) 100 / 68 / 71, 128 x 1000 (1024 of 128) 146 / 94 /
// 81; FP32 the same order.  (128 heads of 128 channels x 500, 512 of 128: forward two
// / four 26 / 22, the largest loss seen.)
int own_waves(const Attn& a, long rows) {
  const long seqs = (long)a.B * a.KV;
  return seqs * fm_ceil_div(rows, 128) >= 768 ? 4 : seqs * fm_ceil_div(rows, 64) >= 256 ? 2 : 1;
}

size_t workspace_floats(const Attn& a, int splits) {
  return splits > 1 ? (size_t)splits * a.B * a.KV * a.T * a.G * ((a.D > 64 ? 128 : 64) + 2) : 0;
}

#define FM_ATTENTION_LAUNCH(kernel, own, rows, z)                                                       \
  do {                                                                                                  \
    const dim3 grid((unsigned)(a.B * a.KV), fm_ceil_div(rows, 32 * (own)), z);                          \
    if ((own) == 4) hipLaunchKernelGGL((kernel<T, DT, 4, 1>), grid, dim3(256), 0, stream, a);           \
    else if ((own) == 2) hipLaunchKernelGGL((kernel<T, DT, 2, 2>), grid, dim3(256), 0, stream, a);      \
    else hipLaunchKernelGGL((kernel<T, DT, 1, 4>), grid, dim3(256), 0, stream, a);                      \
  } while (0)

template <typename T, int DT>
int forward(const Attn& a, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  const int waves = a.splits > 1 ? 1 : own_waves(a, rows);
  FM_ATTENTION_LAUNCH(attention_forward_kernel, waves, rows, a.splits);
  if (a.splits > 1)
    hipLaunchKernelGGL((attention_join_kernel<T, DT>), dim3(fm_ceil_div(a.B * a.KV * rows, 4)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int DT>
int backward(const Attn& a, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  if (rows > 0) FM_ATTENTION_LAUNCH(attention_dq_kernel, own_waves(a, rows), rows, 1);
  const int own = own_waves(a, a.S);
  if constexpr (HELD<T, DT>) {
    const dim3 grid((unsigned)(a.B * a.KV), fm_ceil_div(a.S, 64));
    if ((long)grid.x * grid.y > 512) hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 2>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 4>), grid, dim3(512), 0, stream, a);
  } else {
    FM_ATTENTION_LAUNCH(attention_dkv_kernel, own, a.S, 1);
  }
  return (int)hipGetLastError();
}

#define FM_ATTENTION_TYPES(run)                                            \
  (dtype == DT_F32    ? (a.D > 64 ? run<float, 128>(a, stream) : run<float, 64>(a, stream))   \
   : dtype == DT_BF16 ? (a.D > 64 ? run<__bf16, 128>(a, stream) : run<__bf16, 64>(a, stream)) \
                      : (a.D > 64 ? run<_Float16, 128>(a, stream) : run<_Float16, 64>(a, stream)))

Attn sizes(int batch, int queries, int keys, int heads, int kv_heads, int head_dim, int window, float scale) {
  Attn a{};
  a.B = batch, a.T = queries, a.S = keys, a.H = heads, a.KV = kv_heads, a.D = head_dim;
  a.G = kv_heads > 0 && heads > 0 ? heads / kv_heads : 1;
  a.window = window, a.scale = scale, a.scale2 = scale * LOG2E;
  a.by_g = fm_divisor((unsigned)std::max(a.G, 1));
  return a;
}

}  // namespace

extern "C" {

size_t fm_attention_forward_workspace_bytes(int batch, int queries, int keys, int heads, int kv_heads, int head_dim,
                                            int window) {
  const Attn a = sizes(batch, queries, keys, heads, kv_heads, head_dim, window, 1.0f);
  if (check(a, DT_F32) != FM_OK && check(a, DT_BF16) != FM_OK) return 0;
  if (batch == 0 || queries == 0) return 0;
  return workspace_floats(a, forward_splits(a)) * sizeof(float);
}

int fm_attention_forward(const void* q, long q_batch, long q_row, long q_head, const void* k, long k_batch, long k_row,
                         long k_head, const void* v, long v_batch, long v_row, long v_head, const int* lengths, int batch,
                         int queries, int keys, int heads, int kv_heads, int head_dim, int window, float scale, int dtype,
                         void* out, float* lse, float* workspace, size_t workspace_bytes, hipStream_t stream) {
  Attn a = sizes(batch, queries, keys, heads, kv_heads, head_dim, window, scale);
  a.q = View{q, q_batch, q_row, q_head}, a.k = View{k, k_batch, k_row, k_head}, a.v = View{v, v_batch, v_row, v_head};
  a.lengths = lengths, a.out = out, a.lse = lse;
  if (const int status = check(a, dtype)) return status;
  if (batch == 0 || queries == 0) return FM_OK;
  if (!q || !k || !v || !out || !lse) return FM_BAD_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(out) & 15) return FM_UNSUPPORTED;
  a.splits = forward_splits(a);
  if (a.splits > 1) {
    const size_t need = workspace_floats(a, a.splits) * sizeof(float);
    if (!workspace || workspace_bytes < need) return FM_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FM_UNSUPPORTED;
    a.part_o = workspace;
    a.part_ml = workspace + (size_t)a.splits * a.B * a.KV * a.T * a.G * (a.D > 64 ? 128 : 64);
  }
  return FM_ATTENTION_TYPES(forward);
}

int fm_attention_backward(const void* dout, long dout_batch, long dout_row, long dout_head, const void* q, long q_batch,
                          long q_row, long q_head, const void* k, long k_batch, long k_row, long k_head, const void* v,
                          long v_batch, long v_row, long v_head, const void* out, const float* lse, const int* lengths,
                          int batch, int queries, int keys, int heads, int kv_heads, int head_dim, int window, float scale,
                          int dtype, void* dq, void* dk, void* dv, float* stats, hipStream_t stream) {
  Attn a = sizes(batch, queries, keys, heads, kv_heads, head_dim, window, scale);
  a.q = View{q, q_batch, q_row, q_head}, a.k = View{k, k_batch, k_row, k_head}, a.v = View{v, v_batch, v_row, v_head};
  a.dout = View{dout, dout_batch, dout_row, dout_head};
  a.o = out, a.lengths = lengths, a.lse = const_cast<float*>(lse);
  a.out = dq, a.dk = dk, a.dv = dv, a.stats = stats, a.splits = 1;
  if (const int status = check(a, dtype)) return status;
  if (batch == 0 || keys == 0) return FM_OK;
  if (!k || !v || !dk || !dv || (queries > 0 && (!dout || !q || !out || !lse || !dq || !stats))) return FM_BAD_ARGUMENT;
  for (const void* p : {out, (const void*)dq, (const void*)dk, (const void*)dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return FM_UNSUPPORTED;
  return FM_ATTENTION_TYPES(backward);
}

}  // extern "C"
