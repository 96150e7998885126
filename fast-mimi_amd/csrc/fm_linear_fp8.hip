// Products of 8-bit activations and weights with a power of two to every 128 of them:
//
//   y[m][n] = sum over blocks b of 2^(sx[m][b] + sw[n / 128][b] - 254) sum over k in b of x[m][k] w[n][k]
//
// x [M][K] and w [N][K] are e4m3, the scales e8m0, K a multiple of 16.  The matrix
// instructions take the scales themselves (a byte for each row of 32 or 128 values),
// so one FP32 accumulator runs over all of K and no vector work is left per block.
//
// They line up eight products by the largest and drop what lies 2^-13 below it, each time they
// add eight to the accumulator (measured, in either form of the instruction): 1.5e-5 of the
// result's size with normal values, little beside the half step of a 16-bit result (2e-3
// and 2.4e-4).  FP32 results would lose bits by it, so those are summed from bfloat16 products, which are
// exact: e4m3 times a power of two is a bfloat16, at half the matrix rate.

#include "fm_common.h"

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
// A block forms BM rows of x by BN of w, waves of WM x WN.  128-deep tiles of both
// travel global -> LDS (16 bytes a lane) in two stages, the next one on its way during
// the products.  A row of a tile is 128 bytes, its 16-byte chunk c at chunk c ^ (row / 2 % 8): a fragment
// read takes the same chunk of 16 rows, 256 bytes over all banks.  The weights are the A operand, so that
// a lane ends with runs of four outputs of one row.
//
// Of a 64-deep product lane l holds chunks l / 32 and l / 32 + 2: which values of k does not
// matter as long as both operands hold the same.
template <typename T, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int WAVES = (BM / WM) * (BN / WN), STAGE = (BM + BN) * 128;
};

template <typename T, int BM, int BN, int WM, int WN, int BLOCKS>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), BLOCKS) void linear_tile_kernel(Linear a) {
  constexpr int WAVES = (BM / WM) * (BN / WN), MT = WM / 32, NT = WN / 32, STAGE = (BM + BN) * 128;
  constexpr int LOADS = (BM + BN) / 8 / WAVES;  // instructions of 8 rows each, a wave
  static_assert((BM / 8) % LOADS == 0, "a wave loads rows of one operand");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wm = wave % (BM / WM), wn = wave / (BM / WM);

  // Blocks of one XCD (block % 8) take neighbouring tiles: eight tiles of rows by as
  // many of columns as follow, so that both operands come from its L2 several times.
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int at = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (at >= total) return;
  const int band = 8 * a.tiles_n, first = at / band * 8, rows = min(8, a.tiles_m - first), in = at % band;
  const int m0 = (first + in % rows) * BM, n0 = in / rows * BN;

  const int split = blockIdx.y, per_split = (a.KB + a.splits - 1) / a.splits;
  const int b_lo = split * per_split, b_hi = min(a.KB, b_lo + per_split);

  // This wave's loads: rows of x, or of w.
  const bool of_w = wave * LOADS * 8 >= BM;
  const int limit = of_w ? a.N - n0 : a.M - m0;
  const __amdgpu_buffer_rsrc_t buf = fm_buffer(of_w ? a.w + (long)n0 * a.K : a.x + (long)m0 * a.K, INT_MAX);
  int offset[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int r = (wave * LOADS + u) * 8 + lane / 8, row = of_w ? r - BM : r;
    offset[u] = row < limit ? row * a.K + (((lane & 7) ^ ((r >> 1) & 7)) << 4) : INT_MIN;
  }
  const int chunk[2] = {((lane & 7) ^ ((lane >> 4) & 3)) << 4, ((lane & 7) ^ (((lane >> 4) & 3) + 4)) << 4};
  auto load = [&](int b, int stage) {
    const int left = a.K - b * 128;  // a chunk past the end reads zeros
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = wave * LOADS + u;
      fm_buf_load_lds16(buf, lds + stage * STAGE + i * 1024, chunk[i & 1] < left ? offset[u] : INT_MIN, b * 128);
    }
  };

  // Scales: a lane's own row of each tile of x, one byte for all of the wave's rows of w
  // (or 32 of them, where a block's are not whole 128s).
  const unsigned char* sx[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) sx[i] = a.sx + (long)min(m0 + wm * WM + 32 * i + (lane & 31), a.M - 1) * a.KB;
  const unsigned char* sw = a.sw + (long)(min(n0 + wn * WN, a.N - 1) / 128) * a.KB;
  static_assert(WN <= 128 && 128 % WN == 0 && BN % WN == 0, "a wave's rows of w share their scales");
  int next_x[MT], next_w = 0;
  auto scales = [&](int b) {
#pragma unroll
    for (int i = 0; i < MT; ++i) next_x[i] = sx[i][b];
    next_w = sw[b];
  };

  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int r = lane & 31;
  const unsigned lane_at = base + r * 128 + ((half ^ ((r >> 1) & 7)) << 4);
  auto fragment = [&](unsigned at, int s) {
    const auto p = [&](int u) { return *(const __attribute__((address_space(3))) intx4*)(at ^ (64 * s + 32 * u)); };
    return join(p(0), p(1));
  };

  floatx16 acc[NT][MT] = {};
  if (b_lo < b_hi) load(b_lo, 0), scales(b_lo);
  for (int b = b_lo; b < b_hi; ++b) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int x_scale[MT], w_scale = next_w;
#pragma unroll
    for (int i = 0; i < MT; ++i) x_scale[i] = next_x[i];
    const int stage = (b - b_lo) & 1;
    if (b + 1 < b_hi) load(b + 1, stage ^ 1), scales(b + 1);
    const unsigned x_at = lane_at + stage * STAGE + wm * WM * 128, w_at = lane_at + stage * STAGE + (BM + wn * WN) * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      intx8 xf[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[i] = fragment(x_at + i * 4096, s);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const intx8 wf = fragment(w_at + j * 4096, s);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bf16x8 f = to_bf16(wf, c, scale_of(w_scale));
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[j][i] = fm_mfma32_bf16(f, to_bf16(xf[i], c, scale_of(x_scale[i])), acc[j][i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf, xf[i], acc[j][i], 0, 0, 0, w_scale, 0, x_scale[i]);
        }
      }
    }
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
// Up to 16 MT rows of x by 16 of w a block, whose waves take every WAVES-th 128-deep block
// of K, operands straight from memory (each weight is read once in all), and add their
// sums through LDS in order.
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear_rows_kernel(Linear a) {
  __shared__ float sums[WAVES][MT][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const unsigned char* w = a.w + (long)min(n0 + r, a.N - 1) * a.K;
  const unsigned char* sw = a.sw + (long)(n0 / 128) * a.KB;
  const unsigned char *x[MT], *sx[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long m = min(m0 + 16 * i + r, a.M - 1);
    x[i] = a.x + m * a.K, sx[i] = a.sx + m * a.KB;
  }
  // Lane l holds chunks l / 16 and l / 16 + 4 of a block.
  auto two_chunks = [&](const unsigned char* row, int b) {
    intx4 p{}, q{};
    const int k = b * 128 + quarter * 16;
    if (k < a.K) p = *reinterpret_cast<const intx4*>(row + k);
    if (k + 64 < a.K) q = *reinterpret_cast<const intx4*>(row + k + 64);
    return join(p, q);
  };
  floatx4 acc[MT] = {};
#pragma unroll 4
  for (int b = wave; b < a.KB; b += WAVES) {
    const intx8 wf = two_chunks(w, b);
    const int w_scale = sw[b];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const intx8 xf = two_chunks(x[i], b);
      const int x_scale = sx[i][b];
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(wf, c, scale_of(w_scale)), to_bf16(xf, c, scale_of(x_scale)),
                                                           acc[i], 0, 0, 0);
      } else {
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[i], 0, 0, 0, w_scale, 0, x_scale);
      }
    }
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

constexpr int FEW = 64;  // rows that the few-row kernel takes

struct LinearPlan {
  int bm, bn, splits;
};
LinearPlan linear_plan(long M, int N, int K) {
  if (M <= FEW) return {0, 0, 1};
  if (fm_ceil_div(M, 256) * fm_ceil_div(N, 256) >= 224) return {256, 256, 1};
  const long tiles = (long)fm_ceil_div(M, 128) * fm_ceil_div(N, 128);
  const int blocks = fm_ceil_div(K, 128);
  int splits = 1;
  while (tiles * splits * 2 <= 512 && blocks / (splits * 2) >= 4) splits *= 2;
  return {128, 128, splits};
}

template <typename T>
int run(Linear a, const LinearPlan& p, hipStream_t stream) {
  if (p.bm == 0) {
    const dim3 grid(fm_ceil_div(a.N, 16));
    if (a.M <= 16) hipLaunchKernelGGL((linear_rows_kernel<T, 1, 8>), grid, dim3(512), 0, stream, a);
    else if (a.M <= 32) hipLaunchKernelGGL((linear_rows_kernel<T, 2, 8>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((linear_rows_kernel<T, 4, 8>), grid, dim3(512), 0, stream, a);
    return (int)hipGetLastError();
  }
  a.splits = p.splits, a.tiles_m = fm_ceil_div(a.M, p.bm), a.tiles_n = fm_ceil_div(a.N, p.bn);
  const dim3 grid(fm_ceil_div((long)a.tiles_m * a.tiles_n, 8) * 8, p.splits);
  if (p.bm == 256) hipLaunchKernelGGL((linear_tile_kernel<T, 256, 256, 64, 128, 1>), grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 64, 64, 2>), grid, dim3(256), 0, stream, a);
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

int fm_linear_fp8(const void* x, const void* x_scales, const void* weight, const void* weight_scales, long rows,
                  int in_features, int out_features, int dtype, void* y, float* workspace, size_t workspace_bytes,
                  hipStream_t stream) {
  if (rows < 0 || in_features <= 0 || out_features <= 0 || dtype < DT_F32 || dtype > DT_F16) return FM_BAD_ARGUMENT;
  if (in_features % 16 || in_features > 1 << 22 || rows > 1 << 24 || out_features > 1 << 24) return FM_UNSUPPORTED;
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
