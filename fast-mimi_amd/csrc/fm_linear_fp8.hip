// Products of 8-bit activations and weights with a power of two to every 128 of them:
//
//   y[m][n] = sum over blocks b of 2^(sx[m][b] + sw[n / 128][b] - 254) sum over k in b of x[m][k] w[n][k]
//
// x [M][K] and w [N][K] are e4m3, the scales e8m0, K a multiple of 16.  The matrix
// instructions take the scales themselves (a byte for each row of 32 or 128 values),
// so one FP32 accumulator runs over all of K and no vector work is left per block.
//
// They line up eight neighbouring products by the largest and drop the bits that lie more than 2^-13 below its
// power of two, each time they add eight to the accumulator (measured, in either form of the
// instruction): in all 2e-5 of the results' size with normal values, 1e-4 with values that spread
// over 2^-4 to 2^4, little beside the half step of a 16-bit result (2e-3 and 2.4e-4) but where large products
// cancel.  FP32 results would lose bits by it, so those are summed from bfloat16 products, which are
// exact: e4m3 times a power of two is a bfloat16, at half the matrix rate.
//
// Many rows are bound by the matrix cores and what feeds them: 8192^3 in 413 to 437 us (2510 to 2660 TFLOP/s; up to
// 520 as the clock goes), FP32 results 883; without its loads from memory it takes a tenth less.
// Few rows are bound by latency and the weights' bytes: 1 x 4096 to 6144 6.5 us (25 MB; 8.4 under the tracer), 32 x 8192
// to 2048 8.8 with the join.  (All in a queue of captured calls, bfloat16.)

#include "fm_common.h"

#include <cstdio>

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2_v __attribute__((ext_vector_type(2)));
typedef unsigned uintx4_v __attribute__((ext_vector_type(4)));
typedef float floatx2_v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2_v __attribute__((ext_vector_type(2)));

struct Linear {
  const unsigned char *x, *sx, *w, *sw;
  void* y;
  float* part;  // split sums [split][M][N]
  int M, N, K, KB, splits, tiles_m, tiles_n;
};

FM_DEVICE intx8 join(intx4 a, intx4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
FM_DEVICE float scale_of(int byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight of a lane's e4m3 values (dwords 2 i, 2 i + 1) times the power of two, as bfloat16.
FM_DEVICE bf16x8 to_bf16(intx8 v, int i, float scale) {
  bf16x8 f;
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + d], scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + d], scale, true);
    f[4 * d] = lo[0], f[4 * d + 1] = lo[1], f[4 * d + 2] = hi[0], f[4 * d + 3] = hi[1];
  }
  return f;
}

template <typename T>
FM_DEVICE unsigned two(float a, float b) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2_v{a, b}), bf16x2_v));
  else return __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2_v{a, b}), halfx2_v));
}

// ------------------------------------------------------------ many rows
// A block forms BM rows of x by BN of w, four waves of WM x WN.  128-deep tiles of both
// travel global -> LDS (16 bytes a lane) in two stages, and from there, half a tile at a
// time, into one of two sets of registers: while the products of one half run, the other
// half's (or the next tile's) operands are read.  A tile's second half is in registers before
// its one barrier, so behind it the next but one tile takes its place, and the products go
// on at once; its loads go out one by one between them (16 in a row hold the wave up: 8192^3
// 442 us, so 412).
//
// A row of a tile is 128 bytes, its 16-byte chunk c at chunk c ^ (row / 2 % 8): a fragment read takes
// the same chunk of 16 rows, 256 bytes over all banks.  Of a 64-deep half lane l holds chunks
// l / 32 and l / 32 + 2 of its row: which values of k does not matter as long as both operands
// hold the same.  The weights are the A operand, so that a lane ends with runs of four outputs of one row.
template <typename T, int BM, int BN, int BLOCKS>
__global__ __launch_bounds__(256, BLOCKS) void linear_tile_kernel(Linear a) {
  constexpr int WM = BM / 2, WN = BN / 2, MT = WM / 32, NT = WN / 32, STAGE = (BM + BN) * 128;
  constexpr int LOADS = (BM + BN) / 32, P = MT * NT, F = MT + NT;  // a wave's loads of 8 rows, products and operands
  static_assert(LOADS % 2 == 0 && 128 % WN == 0, "pairs of loads; a wave's rows of w share their scales");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE];
  // The wave's number as a scalar: its loads' bases are, too.
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r = lane & 31;
  const int wm = wave & 1, wn = wave >> 1;

  // Blocks of one XCD (block % 8) take neighbouring tiles: eight tiles of rows by as
  // many of columns as follow, so that both operands come from its L2 several times.
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int at = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (at >= total) return;
  const int band = 8 * a.tiles_n, first = at / band * 8, rows = min(8, a.tiles_m - first), in = at % band;
  const int m0 = (first + in % rows) * BM, n0 = in / rows * BN;

  // This block's part of K, in blocks of 128 values.
  const int split = blockIdx.y, per_split = (a.KB + a.splits - 1) / a.splits;
  const int b_lo = min(a.KB, split * per_split), b_hi = min(a.KB, b_lo + per_split);

  // This wave's loads: rows of x (the first two waves, where the tile is square), or of w.
  const __amdgpu_buffer_rsrc_t buf_x = fm_buffer(a.x + (long)m0 * a.K, INT_MAX), buf_w = fm_buffer(a.w + (long)n0 * a.K, INT_MAX);
  int offset[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int i = wave * LOADS + u, row = 8 * i + lane / 8, own = row - (8 * i < BM ? 0 : BM);
    offset[u] = own < (8 * i < BM ? a.M - m0 : a.N - n0) ? own * a.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4) : INT_MIN;
  }
  const int chunk[2] = {((lane & 7) ^ (lane >> 4)) << 4, ((lane & 7) ^ ((lane >> 4) + 4)) << 4};  // of even and odd loads
  auto load = [&](int b, int stage, int u) {
    const int i = wave * LOADS + u, left = b < b_hi ? a.K - b * 128 : 0;  // a chunk past the end reads zeros
    fm_buf_load_lds16(8 * i < BM ? buf_x : buf_w, lds + stage * STAGE + i * 1024, chunk[u & 1] < left ? offset[u] : INT_MIN, b * 128);
  };

  // Scales: of a lane's own row of each 32 of x, and one byte for all of the wave's rows of w.
  const unsigned char *sx[MT], *sw = a.sw + (long)(min(n0 + wn * WN, a.N - 1) / 128) * a.KB;
#pragma unroll
  for (int i = 0; i < MT; ++i) sx[i] = a.sx + (long)min(m0 + wm * WM + 32 * i + r, a.M - 1) * a.KB;
  int next_x[MT], next_w;
  auto scales = [&](int b) {
#pragma unroll
    for (int i = 0; i < MT; ++i) next_x[i] = sx[i][b];
    next_w = sw[b];
  };

  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const unsigned lane_at = base + r * 128 + ((half ^ ((r >> 1) & 7)) << 4);
  struct Operands {
    intx8 f[F];  // of x, of w
  } first_half, second_half;
  auto fetch = [&](Operands& o, int stage, int s, int p) {
    typedef const __attribute__((address_space(3))) intx4 Chunk;
    const unsigned from = lane_at + stage * STAGE + (p < MT ? wm * WM + 32 * p : BM + wn * WN + 32 * (p - MT)) * 128;
    o.f[p] = join(*(Chunk*)(from ^ (64 * s)), *(Chunk*)(from ^ (64 * s + 32)));
  };

  floatx16 acc[NT][MT] = {};
  int x_scale[MT], w_scale;
  // All products of a half, with something between one and the next.
  auto products = [&](const Operands& o, auto between) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[j][i] = fm_mfma32_bf16(to_bf16(o.f[MT + j], c, scale_of(w_scale)), to_bf16(o.f[i], c, scale_of(x_scale[i])), acc[j][i]);
        } else {
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(o.f[MT + j], o.f[i], acc[j][i], 0, 0, 0, w_scale, 0, x_scale[i]);
        }
        between(j * MT + i);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // Operands go between the products one each, a little behind them, or all that are due.
  auto due = [](int p, auto fetch_one) {
#pragma unroll
    for (int u = P >= F + 2 ? p - 2 : p * F / P; u < (P >= F + 2 ? p - 1 : (p + 1) * F / P); ++u)
      if (u >= 0 && u < F) fetch_one(u);
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  if (b_lo < b_hi) {
    scales(b_lo);
#pragma unroll
    for (int u = 0; u < LOADS; ++u) load(b_lo, 0, u);
    barrier();
#pragma unroll
    for (int u = 0; u < LOADS; ++u) load(b_lo + 1, 1, u);
#pragma unroll
    for (int p = 0; p < F; ++p) fetch(first_half, 0, 0, p);
    for (int b = b_lo; b < b_hi; ++b) {
      const int stage = (b - b_lo) & 1;
      w_scale = next_w;
#pragma unroll
      for (int i = 0; i < MT; ++i) x_scale[i] = next_x[i];
      products(first_half, [&](int p) { due(p, [&](int u) { fetch(second_half, stage, 1, u); }); });
      barrier();
      // Ahead of the tile's loads: waiting for one behind them would be waiting for all.
      scales(min(b + 1, b_hi - 1));
      __builtin_amdgcn_sched_barrier(0);
      products(second_half, [&](int p) {
#pragma unroll
        for (int u = p * LOADS / P; u < (p + 1) * LOADS / P; ++u) load(b + 2, stage, u);
        due(p, [&](int u) { fetch(first_half, stage ^ 1, 0, u); });
      });
    }
    // The copies of the two tiles past the end (zeros) must not outlive the block's LDS.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // Lane l: row l % 32 of x, rows 8 g + 4 (l / 32) .. + 3 of w.
  const bool vectors = (a.N & 7) == 0;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + wm * WM + 32 * i + r;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + wn * WN + 32 * j;
      const floatx16& v = acc[j][i];
      if (a.splits > 1 || sizeof(T) == 4) {
        float* y = a.splits > 1 ? a.part + ((long)split * a.M + m) * a.N : static_cast<float*>(a.y) + (long)m * a.N;
        if (m >= a.M) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = n + 8 * g + 4 * half;
          if (vectors && c < a.N) *reinterpret_cast<floatx4*>(y + c) = floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
          if (!vectors)
            for (int e = 0; e < 4; ++e)
              if (c + e < a.N) y[c + e] = v[4 * g + e];
        }
      } else if constexpr (sizeof(T) == 2) {
        // The lane halves swap every other four outputs: runs of eight, 16 bytes.
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          const unsigned p[2] = {two<T>(v[4 * g], v[4 * g + 1]), two<T>(v[4 * g + 2], v[4 * g + 3])};
          const unsigned q[2] = {two<T>(v[4 * g + 4], v[4 * g + 5]), two<T>(v[4 * g + 6], v[4 * g + 7])};
          // Lower half: outputs 8 g .. + 7 of its row; upper half: 8 (g + 1) .. + 7.
          const auto lo = __builtin_amdgcn_permlane32_swap(p[0], q[0], false, false);
          const auto hi = __builtin_amdgcn_permlane32_swap(p[1], q[1], false, false);
          const uintx4_v u{(unsigned)lo[0], (unsigned)hi[0], (unsigned)lo[1], (unsigned)hi[1]};
          const int c = n + 8 * g + 8 * half;
          if (m >= a.M || c >= a.N) continue;
          T* y = static_cast<T*>(a.y) + (long)m * a.N + c;
          if (vectors) *reinterpret_cast<uintx4_v*>(y) = u;
          else
            for (int e = 0; e < 8; ++e)
              if (c + e < a.N) y[e] = __builtin_bit_cast(T, (unsigned short)(u[e / 2] >> (16 * (e & 1))));
        }
      }
    }
  }
}

// The parts of a call whose K is split, joined in order.
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(Linear a) {
  const long n = (long)a.M * a.N, at = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  T* y = static_cast<T*>(a.y);
  if (n % 4 == 0) {
    floatx4 s = *reinterpret_cast<const floatx4*>(a.part + at);
    for (int k = 1; k < a.splits; ++k) {
      const floatx4 t = *reinterpret_cast<const floatx4*>(a.part + k * n + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += t[e];
    }
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uintx2_v*>(y + at) = uintx2_v{two<T>(s[0], s[1]), two<T>(s[2], s[3])};
    else *reinterpret_cast<floatx4*>(y + at) = s;
  } else {
    for (long i = at; i < std::min(at + 4, n); ++i) {
      float s = a.part[i];
      for (int k = 1; k < a.splits; ++k) s += a.part[k * n + i];
      y[i] = (T)s;
    }
  }
}

// ------------------------------------------------------------- few rows
// The bytes of up to four scales from `from` on, of `left` that the row still has; zeros
// (2^-127, of zero values) behind them.  Nothing past the scales' `total` bytes is read.
FM_DEVICE unsigned four_scales(const unsigned char* scales, long total, long from, int left) {
  if (left <= 0) return 0;
  unsigned v = 0;
  if (total >= 4) {
    const long there = min(from, total - 4);
    __builtin_memcpy(&v, scales + there, 4);
    v >>= 8 * (int)(from - there);
  } else {
    for (int i = 0; i < 3; ++i)
      if (from + i < total) v |= (unsigned)scales[from + i] << (8 * i);
  }
  return left >= 4 ? v : v & ((1u << (8 * left)) - 1);
}

// Up to 16 MT rows of x by 16 of w a block, operands straight from memory: each weight is
// read once in all.  The waves take four blocks of 128 values each in turn, with
// all of their loads on the way at once, and add their sums through LDS in order.
template <typename T, int MT>
__global__ __launch_bounds__(512) void linear_rows_kernel(Linear a) {
  constexpr int WAVES = 8, U = 4;  // blocks of a wave
  __shared__ float sums[WAVES][MT][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const __amdgpu_buffer_rsrc_t buf_w = fm_buffer(a.w + (long)n0 * a.K, INT_MAX), buf_x = fm_buffer(a.x + (long)m0 * a.K, INT_MAX);
  // Lane l holds chunks l / 16 and l / 16 + 4 of a block.
  const int at_w = n0 + r < a.N ? r * a.K + quarter * 16 : INT_MIN;
  int at_x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) at_x[i] = m0 + 16 * i + r < a.M ? (16 * i + r) * a.K + quarter * 16 : INT_MIN;
  const long sw = (long)(n0 / 128) * a.KB, sw_total = (long)((a.N + 127) / 128) * a.KB, sx_total = (long)a.M * a.KB;
  floatx4 acc[MT] = {};
  for (int b0 = 4 * wave; b0 < a.KB; b0 += 4 * WAVES) {
    intx4 wf[U][2], xf[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (b0 + u) * 128 + 64 * h;
        const bool there = quarter * 16 < a.K - k;
        auto get = [&](__amdgpu_buffer_rsrc_t buf, int at) {
          return __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(buf, there ? at : INT_MIN, k, 0));
        };
        wf[u][h] = get(buf_w, at_w);
#pragma unroll
        for (int i = 0; i < MT; ++i) xf[u][i][h] = get(buf_x, at_x[i]);
      }
    // Behind the operands, so that those do not wait for them.
    __builtin_amdgcn_sched_barrier(0);
    const unsigned w_scale = four_scales(a.sw, sw_total, sw + b0, a.KB - b0);
    unsigned x_scale[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
      x_scale[i] = four_scales(a.sx, sx_total, (long)min(m0 + 16 * i + r, a.M - 1) * a.KB + b0, a.KB - b0);
    auto product = [&](auto which) {
      constexpr int B = decltype(which)::value;
      const intx8 w8 = join(wf[B][0], wf[B][1]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const intx8 x8 = join(xf[B][i][0], xf[B][i][1]);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(w8, c, scale_of(w_scale >> (8 * B) & 255)),
                                                             to_bf16(x8, c, scale_of(x_scale[i] >> (8 * B) & 255)), acc[i], 0, 0, 0);
        } else {
          acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[i], 0, 0, B, w_scale, B, x_scale[i]);
        }
      }
    };
    product(std::integral_constant<int, 0>{}), product(std::integral_constant<int, 1>{});
    product(std::integral_constant<int, 2>{}), product(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][i][e][lane] = acc[i][e];
  __syncthreads();
  // Output o of the block: column n0 + o % 16 of row m0 + o / 16.
  for (int o = threadIdx.x; o < 256 * MT; o += 64 * WAVES) {
    const int c = o & 15, m = o >> 4, from = (c >> 2) * 16 + (m & 15);
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) s += sums[k][m >> 4][c & 3][from];
    if (m0 + m < a.M && n0 + c < a.N) static_cast<T*>(a.y)[(long)(m0 + m) * a.N + n0 + c] = (T)s;
  }
}

// How a call runs.  Rows a block (0: the few-row kernel), columns a block, parts of K.
//
// Few rows up to 16, and up to 32 where the weights are 2 MB or less and latency is all
// (us, few rows / the best of 64 x 64 tiles: 1 x 4096 to 6144 6.5 / 7.3, 16 x 8192 to 2048 9.6 / 8.5, 32 x
// 1008 to 1000 3.3 / 4.3, 32 x 4096 to 6144 15.5 / 8.9).
//
// Of the larger tiles those more than half of which hold results (the rule / 256 x 256 tiles, whose rounds the first
// three fill: 65536 x 1024 to 64 14.3 / 18.6, to 128 16.6 / 21.3, 64 x 2048 to 65536 22.5 / 27.1; 20000 x 1024 to 64, 64 x 64 / 64
// x 128, 5.7 / 7.3; just above half, 256 x 256 / 128 x 128, 129 x 2048 to 65536 30.8 / 36.5, 300 x 1024 to 65536 37.5 / 34.2).
//
// 256 x 256 tiles, one block to a CU, where their last round of 256 is nearly full: they
// read the least per product (4096^3 61 us; 128 x 128 79, 64 x 128 97, 64 x 64 129).  Else
// 128 x 128 (two to a CU) from 400 tiles on (1001 x 2048 to 8192 22.0; 64 x 128 27.1), 64
// x 128 from 300 on (500 x 4096 to 6144 23.5; 128 x 128 25.8, 64 x 64 27.1), else 64 x 64
// (256 x 2048 to 8192 9.1; 64 x 128 8.7), whose K is split, up to 512 blocks of eight or more of its
// 128s: the parts go through memory (256 x 8192 to 2048, in 2 / 4 / 8: 21.4 / 16.7 / 19.9; 300 x
// 1040 to 200, in 1 / 2: 4.6 / 5.7).  Of 40 sizes tried most were within 8% of the best of six plans; further behind
// are rounds of 256 x 256 that are not as full (3000 x 8192 to 3000, 144 tiles: 113 us, 256 x 256 84; 16000 x 2048 to
// 520, 189: 33 / 27) and 256 tiles of 64 x 64 that are split (1000 x 4096 to 1000, in 1 / 2: 12.1 / 17.6).
struct LinearPlan {
  int bm, bn, splits;
};
LinearPlan linear_plan(long M, int N, int K) {
  if (M <= 16 || (M <= 32 && (long)N * K <= 1 << 21)) return {0, 0, 1};
  auto tiles = [&](int bm, int bn) { return (long)fm_ceil_div(M, bm) * fm_ceil_div(N, bn); };
  auto full = [&](int bm, int bn) { return 2 * M * N > tiles(bm, bn) * bm * bn; };
  const long large = tiles(256, 256);
  if (full(256, 256) && 4 * large >= 3 * ((large + 255) / 256 * 256)) return {256, 256, 1};
  if (full(128, 128) && tiles(128, 128) >= 400) return {128, 128, 1};
  if (full(64, 128) && tiles(64, 128) >= 300) return {64, 128, 1};
  const long small = tiles(64, 64);
  return {64, 64, (int)std::max<long>(1, std::min<long>({512 / small, fm_ceil_div(K, 128) / 8, 8}))};
}

template <typename T>
int run(Linear a, const LinearPlan& p, hipStream_t stream) {
  if (p.bm == 0) {
    const dim3 grid(fm_ceil_div(a.N, 16));
    if (a.M <= 16) hipLaunchKernelGGL((linear_rows_kernel<T, 1>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((linear_rows_kernel<T, 2>), grid, dim3(512), 0, stream, a);
    return (int)hipGetLastError();
  }
  a.splits = p.splits, a.tiles_m = fm_ceil_div(a.M, p.bm), a.tiles_n = fm_ceil_div(a.N, p.bn);
  const dim3 grid(fm_ceil_div((long)a.tiles_m * a.tiles_n, 8) * 8, p.splits);
  if (p.bm == 256) hipLaunchKernelGGL((linear_tile_kernel<T, 256, 256, 1>), grid, dim3(256), 0, stream, a);
  else if (p.bm == 128) hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2>), grid, dim3(256), 0, stream, a);
  else if (p.bn == 128) hipLaunchKernelGGL((linear_tile_kernel<T, 64, 128, 3>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((linear_tile_kernel<T, 64, 64, 4>), grid, dim3(256), 0, stream, a);
  if (p.splits > 1)
    hipLaunchKernelGGL(linear_join_kernel<T>, dim3(fm_ceil_div((long)a.M * a.N, 1024)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t fm_linear_fp8_workspace_bytes(long rows, int in_features, int out_features) {
  if (rows <= 0 || in_features <= 0 || out_features <= 0) return 0;
  const LinearPlan p = linear_plan(rows, out_features, in_features);
  return p.splits > 1 ? (size_t)p.splits * rows * out_features * sizeof(float) : 0;
}

int fm_linear_fp8_plan(long rows, int in_features, int out_features, char* buf, int size) {
  if (!buf || size <= 0 || rows <= 0 || in_features <= 0 || out_features <= 0) return FM_BAD_ARGUMENT;
  const LinearPlan p = linear_plan(rows, out_features, in_features);
  if (p.bm == 0) snprintf(buf, (size_t)size, "linear_rows_kernel<%d>", rows <= 16 ? 1 : 2);
  else snprintf(buf, (size_t)size, "linear_tile_kernel<%d, %d> splits=%d", p.bm, p.bn, p.splits);
  return FM_OK;
}

int fm_linear_fp8(const void* x, const void* x_scales, const void* weight, const void* weight_scales, long rows,
                  int in_features, int out_features, int dtype, void* y, float* workspace, size_t workspace_bytes,
                  hipStream_t stream) {
  if (rows < 0 || in_features <= 0 || out_features <= 0 || dtype < DT_F32 || dtype > DT_F16) return FM_BAD_ARGUMENT;
  // A tile's rows within 32-bit offsets, tiles and joined outputs within a grid.
  if (in_features % 16 || in_features > 1 << 22 || rows > 1 << 24 || out_features > 1 << 24 || rows * out_features > 1l << 40)
    return FM_UNSUPPORTED;
  if (rows == 0) return FM_OK;
  if (!x || !x_scales || !weight || !weight_scales || !y) return FM_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(y)) & 15)
    return FM_UNSUPPORTED;
  const LinearPlan p = linear_plan(rows, out_features, in_features);
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < (size_t)p.splits * rows * out_features * sizeof(float)) return FM_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FM_UNSUPPORTED;
  }
  Linear a{};
  a.x = static_cast<const unsigned char*>(x), a.sx = static_cast<const unsigned char*>(x_scales);
  a.w = static_cast<const unsigned char*>(weight), a.sw = static_cast<const unsigned char*>(weight_scales);
  a.y = y, a.part = workspace, a.M = (int)rows, a.N = out_features, a.K = in_features, a.KB = fm_ceil_div(in_features, 128);
  a.splits = 1;
  return dtype == DT_F32 ? run<float>(a, p, stream) : dtype == DT_BF16 ? run<__bf16>(a, p, stream) : run<_Float16>(a, p, stream);
}

}  // extern "C"
