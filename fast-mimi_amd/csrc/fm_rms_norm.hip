// RMS norm of a branch added to its residual stream: forward, backward, and the
// forward with its output in 8 bits.  Branch FP32, bfloat16 or float16; stream and
// weight of that type or FP32; every sum in FP32.
//
//   forward   h = x + res, r = 1 / sqrt(mean h^2 + eps), y = h r w
//   backward  hh = (x + res) r, g = dy w, dh = dstream + r (g - hh mean(g hh)),
//             dw = sum over rows of dy hh
//   8 bits    of each 128 channels of y: e the least with max |y| <= 448 2^e,
//             y 2^-e rounded to e4m3, e + 127 kept in a byte (e8m0)
//
// y comes from the sum before it is rounded to the stream's type.  All are bound by
// memory: a row is read once, held in registers, and reduced by the lanes that hold
// it.  Rows start anywhere: 16-byte accesses need no alignment on this part, so
// channels that are not whole vectors cost their last vector only.
//
// 40001 x 4096, bfloat16 on an FP32 stream: forward 327 us (6.0 TB/s), backward 460 (5.7; a large copy
// reaches 4.9), the join 7; 1001 x 2048 bfloat16 in 8 bits 7; 13 x 512 FP32 2.6 and 6.0, by latency.  In 8 bits
// as they are: rows 16000 x 2048 17 (5.9 TB/s), weights 8192 x 8192, once each, 105 (read twice, by single values).

#include "fm_rows.h"

namespace {

// Elements of a lane's vector: 16 bytes of the stream, so that the stores of neighbouring
// lanes lie side by side.
template <typename S>
constexpr int VEC = 16 / (int)sizeof(S);

// E consecutive elements at any address.
template <typename T, int E>
using AnyVec = typename Vec<T, E>::type __attribute__((aligned(sizeof(T))));

struct Rms {
  const void *x, *res, *w, *dy, *dh;  // x, res: backward, either may be NULL; dh: the stream's gradient, or NULL
  void *y, *sum, *scales, *dx, *dres, *dw;
  float *rstd, *part;  // part: [blocks][C]
  long rows, ld_x, ld_res, ld_dy, ld_dh;
  int C, blocks, wide;  // wide: FP32 weights
  float eps;
};

// Vector i of a row of C elements, zeros past its end.
template <typename T, int E>
FM_DEVICE typename Vec<T, E>::type row_load(const T* row, int i, int C) {
  typename Vec<T, E>::type t{};
  const T* at = row + i * E;
  if ((i + 1) * E <= C) {
    t = *reinterpret_cast<const AnyVec<T, E>*>(at);
  } else {
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (i * E + e < C) t[e] = at[e];
  }
  return t;
}
// PAST: past the L2.
template <typename T, int E, bool PAST = false>
FM_DEVICE void row_store(T* row, int i, int C, typename Vec<T, E>::type t) {
  T* at = row + i * E;
  if ((i + 1) * E <= C) {
    auto to = reinterpret_cast<AnyVec<T, E>*>(at);
    if constexpr (PAST) __builtin_nontemporal_store(t, to);
    else *to = t;
  } else {
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (i * E + e < C) at[e] = t[e];
  }
}

// Vector i of the weights, of T or FP32; ones without any.
template <typename T, int E>
FM_DEVICE void weight_load(const Rms& a, int i, float (&w)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = 1.0f;
  if (!a.w) return;
  if (sizeof(T) == 4 || a.wide) {
    const typename Vec<float, E>::type t = row_load<float, E>(static_cast<const float*>(a.w), i, a.C);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = t[e];
  } else {
    const typename Vec<T, E>::type t = row_load<T, E>(static_cast<const T*>(a.w), i, a.C);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = widen(t[e]);
  }
}
template <typename T>
FM_DEVICE float one_weight(const Rms& a, int c) {
  if (!a.w) return 1.0f;
  return sizeof(T) == 4 || a.wide ? static_cast<const float*>(a.w)[c] : widen(static_cast<const T*>(a.w)[c]);
}
template <typename T>
FM_DEVICE void store_weight_gradient(const Rms& a, long c, float v) {
  if (sizeof(T) == 4 || a.wide) static_cast<float*>(a.dw)[c] = v;
  else static_cast<T*>(a.dw)[c] = (T)v;
}

// The scale byte of 128 values whose largest magnitude is `most`: 255 (NaN) for an
// infinity or NaN among them.
FM_DEVICE int scale_byte(float most) {
  const unsigned u = __builtin_bit_cast(unsigned, most);
  return u >= 0x7f800000u ? 255 : max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u), 0);
}
// Four values times 2^-(byte - 127), to e4m3.
FM_DEVICE unsigned four_in_8_bits(float a, float b, float c, float d, int byte) {
  const int by = 127 - byte;
  int u = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(a, by), __builtin_ldexpf(b, by), 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(c, by), __builtin_ldexpf(d, by), u, true);
}

// Writes vector i of a row in 8 bits.  The lanes of a block's 128 channels call it
// together; GROUP of them (neighbours) hold one.
template <int E, int GROUP>
FM_DEVICE void store_8_bits(const float (&v)[E], unsigned char* row, unsigned char* scales, int i, int C) {
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float m = fabsf(v[e]);
    // As integers: a NaN is above every other magnitude.
    most = __builtin_bit_cast(float, max(__builtin_bit_cast(int, most), __builtin_bit_cast(int, m)));
  }
  const int byte = scale_byte(lanes_max<GROUP>(most));
  if (i * E >= C) return;
  if (i * E % 128 == 0) scales[i * E / 128] = (unsigned char)byte;
  typename Vec<unsigned char, E>::type t;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const unsigned u = four_in_8_bits(v[e], v[e + 1], v[e + 2], v[e + 3], byte);
#pragma unroll
    for (int k = 0; k < 4; ++k) t[e + k] = (unsigned char)(u >> (8 * k));
  }
  row_store<unsigned char, E>(row, i, C, t);
}

// Lane p of a row holds vectors p, p + LPR, ... (NV of them, E elements each).
template <typename T, typename S, int NV, int LPR, bool BITS8, bool PAST>
__global__ __launch_bounds__(256) void rms_forward_kernel(Rms a) {
  constexpr int E = VEC<S>;
  __shared__ float waves[4];
  const int p = threadIdx.x % LPR;
  const long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const S* res = a.res ? static_cast<const S*>(a.res) + row * a.ld_res : nullptr;
  float v[NV][E], w[NV][E];
  float s = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = p + u * LPR;
    const typename Vec<T, E>::type t = row_load<T, E>(x, i, a.C);
    typename Vec<S, E>::type r{};
    if (res) r = row_load<S, E>(res, i, a.C);
#pragma unroll
    for (int e = 0; e < E; ++e) v[u][e] = widen(t[e]) + widen(r[e]);
  }
  // The weights are on their way during the sum.
#pragma unroll
  for (int u = 0; u < NV; ++u) weight_load<T, E>(a, p + u * LPR, w[u]);
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(v[u][e], v[u][e], s);
  if (a.sum) {
    S* h = static_cast<S*>(a.sum) + row * a.C;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      typename Vec<S, E>::type t;
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = (S)v[u][e];
      row_store<S, E, PAST>(h, p + u * LPR, a.C, t);
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<LPR>(s, waves) / (float)a.C + a.eps);
  if (p == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = p + u * LPR;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = v[u][e] * rstd * w[u][e];
    if constexpr (BITS8) {
      const int blocks = (a.C + 127) / 128;
      store_8_bits<E, (128 / E < LPR ? 128 / E : LPR)>(y, static_cast<unsigned char*>(a.y) + row * a.C,
                                                       static_cast<unsigned char*>(a.scales) + row * blocks, i, a.C);
    } else {
      typename Vec<T, E>::type t;
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = (T)y[e];
      row_store<T, E, PAST>(static_cast<T*>(a.y) + row * a.C, i, a.C, t);
    }
  }
}

// The sum over a row's lanes; with more than 64, its waves, through `waves` (of its own
// for each sum between two barriers).
template <int LPR>
FM_DEVICE float lanes_sum(float v, float* waves) {
  v = row_sum<(LPR < 64 ? LPR : 64)>(v);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int u = 0; u < LPR / 64; ++u) v += waves[u];
  }
  return v;
}

// dh, and this block's share of dw: a row group walks rows blockIdx * groups + g,
// + gridDim * groups, ... with the columns' sums in registers; the block joins its
// groups through LDS in order and writes one partial row (or, when it is the only
// block, the gradient itself).
template <typename T, typename S, int NV, int LPR, bool PAST>
__global__ __launch_bounds__(LPR < 256 ? 256 : LPR) void rms_backward_kernel(Rms a) {
  constexpr int E = VEC<S>, GROUPS = LPR < 256 ? 256 / LPR : 1;
  typedef typename Vec<T, E>::type VT;
  typedef typename Vec<S, E>::type VS;
  __shared__ float joined[GROUPS > 1 ? 256 * E : 1], waves[2][LPR > 64 ? LPR / 64 : 1];
  const int p = threadIdx.x % LPR, g = threadIdx.x / LPR;
  float wv[NV][E], dw[NV][E];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    weight_load<T, E>(a, p + u * LPR, wv[u]);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[u][e] = 0.0f;
  }
  const float inv = 1.0f / (float)a.C;
  VT xv[NV], xn[NV], gv[NV], gn[NV];
  VS rv[NV], rn[NV], sv[NV], sn[NV];
  float rstd, rstd_n = 0.0f;
  const long step = (long)gridDim.x * GROUPS;
  // The next row is on its way while this one is worked on.
  auto load = [&](long row) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = p + u * LPR;
      xn[u] = VT{}, rn[u] = VS{}, sn[u] = VS{};
      if (a.x) xn[u] = row_load<T, E>(static_cast<const T*>(a.x) + row * a.ld_x, i, a.C);
      if (a.res) rn[u] = row_load<S, E>(static_cast<const S*>(a.res) + row * a.ld_res, i, a.C);
      if (a.dh) sn[u] = row_load<S, E>(static_cast<const S*>(a.dh) + row * a.ld_dh, i, a.C);
      gn[u] = row_load<T, E>(dy, i, a.C);
    }
    rstd_n = a.rstd[row];
  };
  int turn = 0;
  long row = (long)blockIdx.x * GROUPS + g;
  if (row < a.rows) load(row);
  for (; row < a.rows; row += step) {
#pragma unroll
    for (int u = 0; u < NV; ++u) xv[u] = xn[u], rv[u] = rn[u], gv[u] = gn[u], sv[u] = sn[u];
    rstd = rstd_n;
    if (row + step < a.rows) load(row + step);
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float hh = (widen(xv[u][e]) + widen(rv[u][e])) * rstd, d = widen(gv[u][e]);
        s = fmaf(d * wv[u][e], hh, s);
        dw[u][e] = fmaf(d, hh, dw[u][e]);
      }
    s = lanes_sum<LPR>(s, waves[turn]) * inv, turn ^= 1;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      VS t;
      VT b;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float hh = (widen(xv[u][e]) + widen(rv[u][e])) * rstd;
        const float dh = fmaf(rstd, fmaf(widen(gv[u][e]), wv[u][e], -hh * s), widen(sv[u][e]));
        t[e] = (S)dh, b[e] = (T)dh;
      }
      row_store<S, E, PAST>(static_cast<S*>(a.dres) + row * a.C, p + u * LPR, a.C, t);
      if (a.dx) row_store<T, E, PAST>(static_cast<T*>(a.dx) + row * a.C, p + u * LPR, a.C, b);
    }
  }
  if (!a.dw) return;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) joined[e * 256 + threadIdx.x] = dw[u][e];
      __syncthreads();
      if (g != 0) continue;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (p + u * LPR) * E + e;
      if (c >= a.C) continue;
      float s = dw[u][e];
      if constexpr (GROUPS > 1) {
        s = 0.0f;
        for (int j = 0; j < GROUPS; ++j) s += joined[e * 256 + j * LPR + p];
      }
      if (a.blocks > 1) a.part[(long)blockIdx.x * a.C + c] = s;
      else store_weight_gradient<T>(a, c, s);
    }
  }
}

// Any number of channels: one block per row (forward) or per run of rows
// (backward), the row read again for each step.
template <typename T, typename S, bool BITS8>
__global__ __launch_bounds__(256) void rms_forward_any_kernel(Rms a) {
  __shared__ float waves[4];
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const S* res = a.res ? static_cast<const S*>(a.res) + row * a.ld_res : nullptr;
  auto h = [&](int c) { return widen(x[c]) + (res ? widen(res[c]) : 0.0f); };
  float s = 0.0f;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float v = h(c);
    s = fmaf(v, v, s);
    if (a.sum) static_cast<S*>(a.sum)[row * a.C + c] = (S)v;
  }
  const float rstd = 1.0f / sqrtf(row_sum<256>(s, waves) / (float)a.C + a.eps);
  if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
  if constexpr (BITS8) {
    const int blocks = (a.C + 127) / 128;
    // Vectors of four channels, 32 lanes to a block; whole waves go round together.
    for (int c0 = 0; c0 < a.C; c0 += 1024) {
      const int i = c0 / 4 + threadIdx.x;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 4 * i + e;
        y[e] = c < a.C ? h(c) * rstd * one_weight<T>(a, c) : 0.0f;
      }
      store_8_bits<4, 32>(y, static_cast<unsigned char*>(a.y) + row * a.C, static_cast<unsigned char*>(a.scales) + row * blocks,
                          i, a.C);
    }
  } else {
    for (int c = threadIdx.x; c < a.C; c += 256)
      static_cast<T*>(a.y)[row * a.C + c] = (T)(h(c) * rstd * one_weight<T>(a, c));
  }
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void rms_backward_any_kernel(Rms a) {
  __shared__ float waves[2][4];
  float* part = a.part + (long)blockIdx.x * a.C;
  bool first = true;
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1, first = false) {
    const T* x = a.x ? static_cast<const T*>(a.x) + row * a.ld_x : nullptr;
    const S* res = a.res ? static_cast<const S*>(a.res) + row * a.ld_res : nullptr;
    auto h = [&](int c) { return (x ? widen(x[c]) : 0.0f) + (res ? widen(res[c]) : 0.0f); };
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const S* dh = a.dh ? static_cast<const S*>(a.dh) + row * a.ld_dh : nullptr;
    const float rstd = a.rstd[row];
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float hh = h(c) * rstd, d = widen(dy[c]);
      s = fmaf(d * one_weight<T>(a, c), hh, s);
      if (a.dw) part[c] = first ? d * hh : fmaf(d, hh, part[c]);
    }
    s = row_sum<256>(s, waves[turn]) / (float)a.C;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float hh = h(c) * rstd;
      const float v = fmaf(rstd, fmaf(widen(dy[c]), one_weight<T>(a, c), -hh * s), dh ? widen(dh[c]) : 0.0f);
      static_cast<S*>(a.dres)[row * a.C + c] = (S)v;
      if (a.dx) static_cast<T*>(a.dx)[row * a.C + c] = (T)v;
    }
  }
}

// dw from the blocks' partial rows: 32 columns a block, 32 threads to a column, each
// summing every 32nd row in order, then joined in order.
template <typename T>
__global__ __launch_bounds__(1024) void rms_join_kernel(Rms a) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const long col = (long)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (col < a.C) {
    const float* from = a.part + col;
#pragma unroll 4
    for (int r = g; r < a.blocks; r += 32) s += from[(long)r * a.C];
  }
  sums[g][c] = s;
  __syncthreads();
  if (g != 0 || col >= a.C) return;
  float total = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j) total += sums[j][c];
  store_weight_gradient<T>(a, col, total);
}

// No rows: a zero gradient.
template <typename T>
__global__ __launch_bounds__(256) void rms_zero_kernel(Rms a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < a.C) store_weight_gradient<T>(a, c, 0.0f);
}

// Rows as they are, in 8 bits: a lane a vector.  A row has whole 128-channel blocks of
// vectors, so that a block's lanes are neighbours.
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(Rms a, unsigned vectors, unsigned per_row, FmDivisor by) {
  constexpr int E = 16 / (int)sizeof(T);
  const unsigned at = blockIdx.x * 256 + threadIdx.x;
  if ((at & ~63u) >= vectors) return;  // whole waves
  const unsigned row = at < vectors ? fm_div(at, by) : 0;
  const int i = at < vectors ? (int)(at - row * per_row) : a.C;  // C: past every row's end
  const typename Vec<T, E>::type t = row_load<T, E>(static_cast<const T*>(a.x) + row * a.ld_x, i, a.C);
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = widen(t[e]);
  store_8_bits<E, 128 / E>(v, static_cast<unsigned char*>(a.y) + (long)row * a.C,
                           static_cast<unsigned char*>(a.scales) + (long)row * ((a.C + 127) / 128), i, a.C);
}

// Weights [N][K] in 8 bits, one scale to 128 x 128 of them: a block each.
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* w, int N, int K, unsigned char* out, unsigned char* scales) {
  __shared__ int waves[4];
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128, k = k0 + (threadIdx.x & 31) * 4;
  const int rows = min(128, N - n0);
  auto values = [&](int r, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < K ? widen(w[(long)(n0 + r) * K + k + e]) : 0.0f;
  };
  int most = 0;
  for (int r = threadIdx.x >> 5; r < rows; r += 8) {
    float v[4];
    values(r, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) most = max(most, __builtin_bit_cast(int, fabsf(v[e])));
  }
  most = __builtin_bit_cast(int, lanes_max<64>(__builtin_bit_cast(float, most)));
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = most;
  __syncthreads();
  most = max(max(waves[0], waves[1]), max(waves[2], waves[3]));
  const int byte = scale_byte(__builtin_bit_cast(float, most));
  if (threadIdx.x == 0) scales[(long)blockIdx.y * gridDim.x + blockIdx.x] = (unsigned char)byte;
  for (int r = threadIdx.x >> 5; r < rows; r += 8) {
    float v[4];
    values(r, v);
    const unsigned u = four_in_8_bits(v[0], v[1], v[2], v[3], byte);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < K) out[(long)(n0 + r) * K + k + e] = (unsigned char)(u >> (8 * e));
  }
}

constexpr int MOST_CHANNELS = 1 << 26;
constexpr long MOST_ROWS = 1 << 23;  // of a launch: a grid has at most 2^32 threads
// Bytes of the stream from which on results go past the L2, whose eight parts hold 32 MB (through / past, us, inputs
// that are not in the caches; in brackets with a product that reads y and a norm that reads h next.  bfloat16 x 4096:
// 16 MB 11.9 / 11.6 (42 / 44), 32 MB 25.6 / 21.0 (74 / 73), 64 MB 48 / 48 (150 / 138), 256 MB 196 / 191 (489 / 472); with an
// FP32 stream 24 MB 14.0 / 13.4 (46 / 45), 48 MB 33 / 25 (81 / 76), 128 MB 81 / 73 (204 / 191); backward 64 MB 65 / 58.  At 32 MB
// and above nothing lost more than 3%, below it what reads y lost up to 6%).
constexpr long PAST_FROM = 32l << 20;

int rms_check(const Rms& a, int dtype, int stype, int wtype) {
  if (a.rows < 0 || a.C <= 0 || dtype < DT_F32 || dtype > DT_F16 || (stype != dtype && stype != DT_F32) ||
      (wtype != dtype && wtype != DT_F32) || !(a.eps >= 0.0f))
    return FM_BAD_ARGUMENT;
  if (a.rows > 1 && (a.ld_x < 0 || a.ld_res < 0 || a.ld_dy < 0 || a.ld_dh < 0)) return FM_BAD_ARGUMENT;
  if (a.rows >= INT_MAX || a.C > MOST_CHANNELS) return FM_UNSUPPORTED;
  return FM_OK;
}

enum Pass { FORWARD, BITS8, BACKWARD };

// The lanes and vectors of a row: the rule of plan(), rows being whole vectors here, but for
// forward rows that leave a block a vector each or half that (us, 2048 bfloat16 channels in 8 bits, a
// wave / a block a row: 13 rows 4.5 / 3.4, 1001 5.3 / 4.8, 4000 12.1 / 12.2, 16000 36 / 35; 1024, half
// of the lanes idle: 16000 19 / 25).
Plan forward_plan(int C, int e) {
  const int n = (C + e - 1) / e;
  return n > 128 && n <= 256 ? Plan{e, 1, 256} : plan(n * e, 16 / e, true);
}
// The backward pass holds three or four tensors' vectors twice (a row and the next), so at most
// two of each a lane: four leave one wave to a SIMD (4000 x 2048 bfloat16, four in a wave / one in a
// block a row: 29 / 19 us; 40000 x 4096 with an FP32 stream, four / two / one in 256 / 512 / 1024
// lanes: 506 / 520 / 475).
Plan backward_plan(int C, int e) {
  const int n = (C + e - 1) / e;
  if (n <= 16) return {e, 1, 16};
  if (n <= 128) return {e, n <= 64 ? 1 : 2, 64};
  if (n <= 512) return {e, n <= 256 ? 1 : 2, 256};
  if (n <= 1024) return {e, 1, 1024};
  return n <= 2048 && e == 4 ? Plan{e, 2, 1024} : Plan{e, 0, 64};
}

template <typename T, typename S, int NV, int LPR, Pass PASS, bool PAST>
void launch(const Rms& a, hipStream_t stream) {
  if constexpr (PASS == BACKWARD)
    hipLaunchKernelGGL((rms_backward_kernel<T, S, NV, LPR, PAST>), dim3(a.blocks), dim3(std::max(256, LPR)), 0, stream, a);
  else
    hipLaunchKernelGGL((rms_forward_kernel<T, S, NV, LPR, PASS == BITS8, PAST>), dim3(fm_ceil_div(a.rows, 256 / LPR)), dim3(256),
                       0, stream, a);
}

// False where the plan has no kernel (none of those above).
template <typename T, typename S, Pass PASS, bool PAST>
bool launch_plan(const Rms& a, const Plan& p, hipStream_t stream) {
  if (p.lpr == 16) return launch<T, S, 1, 16, PASS, PAST>(a, stream), true;
  if (p.lpr == 64 && p.nv == 1) return launch<T, S, 1, 64, PASS, PAST>(a, stream), true;
  if (p.lpr == 64 && p.nv == 2) return launch<T, S, 2, 64, PASS, PAST>(a, stream), true;
  if (p.lpr == 256 && p.nv == 1) return launch<T, S, 1, 256, PASS, PAST>(a, stream), true;
  if (p.lpr == 256 && p.nv == 2) return launch<T, S, 2, 256, PASS, PAST>(a, stream), true;
  if constexpr (PASS == BACKWARD) {
    if (p.lpr == 1024 && p.nv == 1) return launch<T, S, 1, 1024, PASS, PAST>(a, stream), true;
    if constexpr (sizeof(S) == 4)
      if (p.lpr == 1024) return launch<T, S, 2, 1024, PASS, PAST>(a, stream), true;
  } else {
    if (p.nv == 4) return launch<T, S, 4, 256, PASS, PAST>(a, stream), true;
    if constexpr (sizeof(S) == 4)
      if (p.nv == 8) return launch<T, S, 8, 256, PASS, PAST>(a, stream), true;
  }
  return false;
}

template <typename T, typename S, Pass PASS>
int run(Rms a, hipStream_t stream) {
  const Plan p = PASS == BACKWARD ? backward_plan(a.C, VEC<S>) : forward_plan(a.C, VEC<S>);
  if (PASS == BACKWARD && a.rows == 0) {
    hipLaunchKernelGGL((rms_zero_kernel<T>), dim3(fm_ceil_div(a.C, 256)), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
  }
  if (PASS != BACKWARD && a.rows > MOST_ROWS) {
    Rms part = a;
    for (long first = 0; first < a.rows; first += MOST_ROWS) {
      part.rows = std::min(MOST_ROWS, a.rows - first);
      part.x = static_cast<const T*>(a.x) + first * a.ld_x;
      if (a.res) part.res = static_cast<const S*>(a.res) + first * a.ld_res;
      if (a.sum) part.sum = static_cast<S*>(a.sum) + first * a.C;
      part.y = static_cast<char*>(a.y) + first * a.C * (PASS == BITS8 ? 1 : sizeof(T));
      if (a.scales) part.scales = static_cast<char*>(a.scales) + first * ((a.C + 127) / 128);
      if (a.rstd) part.rstd = a.rstd + first;
      if (const int status = run<T, S, PASS>(part, stream)) return status;
    }
    return FM_OK;
  }
  a.blocks = PASS == BACKWARD ? backward_blocks(a.rows, p, sizeof(T)) : 0;
  if (p.nv == 0) {
    if constexpr (PASS == BACKWARD)
      hipLaunchKernelGGL((rms_backward_any_kernel<T, S>), dim3(a.blocks), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((rms_forward_any_kernel<T, S, PASS == BITS8>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
  } else if (PASS != BITS8 && a.rows * a.C * (long)sizeof(S) >= PAST_FROM) {
    if (!launch_plan<T, S, PASS, PASS != BITS8>(a, p, stream)) return FM_UNSUPPORTED;
  } else {
    if (!launch_plan<T, S, PASS, false>(a, p, stream)) return FM_UNSUPPORTED;
  }
  if (PASS == BACKWARD && a.dw && (a.blocks > 1 || p.nv == 0))
    hipLaunchKernelGGL((rms_join_kernel<T>), dim3(fm_ceil_div(a.C, 32)), dim3(1024), 0, stream, a);
  return (int)hipGetLastError();
}

template <Pass PASS>
int dispatch(Rms a, int dtype, int stype, int wtype, hipStream_t stream) {
  a.wide = wtype == DT_F32;
  if (dtype == DT_F32) return run<float, float, PASS>(a, stream);
  if (stype == DT_F32) return dtype == DT_BF16 ? run<__bf16, float, PASS>(a, stream) : run<_Float16, float, PASS>(a, stream);
  return dtype == DT_BF16 ? run<__bf16, __bf16, PASS>(a, stream) : run<_Float16, _Float16, PASS>(a, stream);
}

template <typename T>
int quantize(Rms a, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(T);
  const long per_row = (a.C + 127) / 128 * (128 / E), most = std::max<long>(1, (1u << 30) / per_row);
  const FmDivisor by = fm_divisor((unsigned)per_row);
  const Rms whole = a;
  for (long first = 0; first < whole.rows; first += most) {
    a.rows = std::min(most, whole.rows - first);
    a.x = static_cast<const T*>(whole.x) + first * whole.ld_x;
    a.y = static_cast<char*>(whole.y) + first * whole.C;
    a.scales = static_cast<char*>(whole.scales) + first * ((whole.C + 127) / 128);
    const long vectors = a.rows * per_row;
    hipLaunchKernelGGL((quantize_kernel<T>), dim3(fm_ceil_div(vectors, 256)), dim3(256), 0, stream, a, (unsigned)vectors,
                       (unsigned)per_row, by);
  }
  return (int)hipGetLastError();
}

template <typename T>
int quantize_weight(const void* w, int N, int K, void* out, void* scales, hipStream_t stream) {
  hipLaunchKernelGGL((quantize_weight_kernel<T>), dim3(fm_ceil_div(K, 128), fm_ceil_div(N, 128)), dim3(256), 0, stream,
                     static_cast<const T*>(w), N, K, static_cast<unsigned char*>(out), static_cast<unsigned char*>(scales));
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int fm_rms_norm_forward(const void* x, long ld_x, const void* residual, long ld_residual, const void* gamma, long rows,
                        int channels, float eps, int dtype, int stream_dtype, int weight_dtype, void* y, void* h, float* rstd,
                        hipStream_t stream) {
  Rms a{};
  a.x = x, a.res = residual, a.w = gamma, a.y = y, a.sum = h, a.rstd = rstd;
  a.rows = rows, a.ld_x = ld_x, a.ld_res = ld_residual, a.C = channels, a.eps = eps;
  if (const int status = rms_check(a, dtype, stream_dtype, weight_dtype)) return status;
  if (rows == 0) return FM_OK;
  if (!x || !y || !rstd || (residual && !h)) return FM_BAD_ARGUMENT;
  return dispatch<FORWARD>(a, dtype, stream_dtype, weight_dtype, stream);
}

int fm_rms_norm_quantized(const void* x, long ld_x, const void* residual, long ld_residual, const void* gamma, long rows,
                          int channels, float eps, int dtype, int stream_dtype, int weight_dtype, void* y, void* scales, void* h,
                          hipStream_t stream) {
  Rms a{};
  a.x = x, a.res = residual, a.w = gamma, a.y = y, a.scales = scales, a.sum = h;
  a.rows = rows, a.ld_x = ld_x, a.ld_res = ld_residual, a.C = channels, a.eps = eps;
  if (const int status = rms_check(a, dtype, stream_dtype, weight_dtype)) return status;
  if (rows == 0) return FM_OK;
  if (!x || !y || !scales || (residual && !h)) return FM_BAD_ARGUMENT;
  return dispatch<BITS8>(a, dtype, stream_dtype, weight_dtype, stream);
}

// Room for the most blocks that the call runs; none where its plan is one block.
size_t fm_rms_norm_backward_workspace_bytes(long rows, int channels) {
  if (rows <= 0 || channels <= 0) return 0;
  if (rows <= (channels <= 512 ? 4 * ONE_BLOCK : channels <= 8192 ? ONE_BLOCK : 0)) return 0;
  return (size_t)std::min<long>(1024, rows) * channels * sizeof(float);
}

int fm_rms_norm_backward(const void* dy, long ld_dy, const void* x, long ld_x, const void* residual, long ld_residual,
                         const void* gamma, const float* rstd, const void* dh, long ld_dh, long rows, int channels, int dtype,
                         int stream_dtype, int weight_dtype, void* dx, void* dresidual, void* dgamma, float* workspace,
                         size_t workspace_bytes, hipStream_t stream) {
  Rms a{};
  a.x = x, a.res = residual, a.dy = dy, a.w = gamma, a.dh = dh, a.dx = dx, a.dres = dresidual, a.dw = dgamma;
  a.rstd = const_cast<float*>(rstd), a.part = workspace;
  a.rows = rows, a.ld_x = ld_x, a.ld_res = ld_residual, a.ld_dy = ld_dy, a.ld_dh = ld_dh, a.C = channels;
  if (const int status = rms_check(a, dtype, stream_dtype, weight_dtype)) return status;
  if (rows == 0 && !dgamma) return FM_OK;
  if (rows > 0 && ((!x && !residual) || !dy || !dresidual || !rstd)) return FM_BAD_ARGUMENT;
  if (rows > 0 && dgamma && workspace_bytes < fm_rms_norm_backward_workspace_bytes(rows, channels)) return FM_WORKSPACE_TOO_SMALL;
  if (workspace_bytes > 0 && !workspace) return FM_BAD_ARGUMENT;
  return dispatch<BACKWARD>(a, dtype, stream_dtype, weight_dtype, stream);
}

int fm_quantize_rows(const void* x, long ld_x, long rows, int channels, int dtype, void* y, void* scales, hipStream_t stream) {
  Rms a{};
  a.x = x, a.ld_x = ld_x, a.rows = rows, a.C = channels, a.y = y, a.scales = scales;
  if (const int status = rms_check(a, dtype, dtype, dtype)) return status;
  if (rows == 0) return FM_OK;
  if (!x || !y || !scales) return FM_BAD_ARGUMENT;
  return dtype == DT_F32 ? quantize<float>(a, stream) : dtype == DT_BF16 ? quantize<__bf16>(a, stream) : quantize<_Float16>(a, stream);
}

int fm_quantize_weight(const void* weight, int out_features, int in_features, int dtype, void* values, void* scales,
                       hipStream_t stream) {
  if (out_features <= 0 || in_features <= 0 || dtype < DT_F32 || dtype > DT_F16 || !weight || !values || !scales)
    return FM_BAD_ARGUMENT;
  if (out_features > 128 * 65535 || in_features > MOST_CHANNELS) return FM_UNSUPPORTED;
  return dtype == DT_F32    ? quantize_weight<float>(weight, out_features, in_features, values, scales, stream)
         : dtype == DT_BF16 ? quantize_weight<__bf16>(weight, out_features, in_features, values, scales, stream)
                            : quantize_weight<_Float16>(weight, out_features, in_features, values, scales, stream);
}

}  // extern "C"
