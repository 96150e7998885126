// Products of 8-bit activations and weights with a power of two to every 128 of them:
//
//   y[m][n] = sum over blocks b of 2^(sx[m][b] + sw[n / 128][b] - 254) sum over k in b of x[m][k] w[n][k]
//
// x [M][K] and w [N][K] are e4m3, the scales e8m0, K a multiple of 16; sums in FP32.
// The matrix instructions take the scales themselves (a byte for each row of 32 or 128
// values), so one accumulator runs over all of K and no vector work is left per block.

#include "fm_common.h"

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));

struct Linear {
  const unsigned char *x, *sx, *w, *sw;
  void* y;
  float* part;  // split sums [split][M][N]
  int M, N, K, KB, splits;
};

// D += A B on 32 x 32, 64 deep: lane l holds row (column) l % 32 and 32 values of k, any as
// long as both operands hold the same; result layout of fm_mfma32.
FM_DEVICE floatx16 mfma32_fp8(intx8 a, intx8 b, floatx16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// Eight of a lane's e4m3 values (dwords 2 i, 2 i + 1) times 2^(byte - 127), as bfloat16: exact.
FM_DEVICE bf16x8 to_bf16(intx4 v, int i, float scale) {
  bf16x8 f;
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + d], scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + d], scale, true);
    f[4 * d] = lo[0], f[4 * d + 1] = lo[1], f[4 * d + 2] = hi[0], f[4 * d + 3] = hi[1];
  }
  return f;
}
FM_DEVICE float scale_of(int byte) { return __builtin_bit_cast(float, byte == 0 ? 0x400000 : byte == 255 ? 0x7fc00000 : byte << 23); }

// One wave: 32 rows of x by 32 of w, operands straight from memory.  Of a block of 128
// values lane l takes 16-byte chunks l / 32, + 2 (first product) and + 4, + 6 (second).
template <typename T>
__global__ __launch_bounds__(64) void linear_simple_kernel(Linear a) {
  const int lane = threadIdx.x, half = lane >> 5;
  const int n = blockIdx.x * 32 + (lane & 31), m = blockIdx.y * 32 + (lane & 31);
  const unsigned char* w = a.w + (long)min(n, a.N - 1) * a.K;
  const unsigned char* x = a.x + (long)min(m, a.M - 1) * a.K;
  const unsigned char* sw = a.sw + (long)(min(n, a.N - 1) / 128) * a.KB;
  const unsigned char* sx = a.sx + (long)min(m, a.M - 1) * a.KB;
  floatx16 acc = {};
  for (int b = 0; b < a.KB; ++b) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      intx8 f[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = b * 128 + 64 * s + 32 * u + 16 * half;
        intx4 p{}, q{};
        if (k < a.K) p = *reinterpret_cast<const intx4*>(w + k), q = *reinterpret_cast<const intx4*>(x + k);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc = fm_mfma32_bf16(to_bf16(p, i, scale_of(sw[b])), to_bf16(q, i, scale_of(sx[b])), acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) f[0][4 * u + e] = p[e], f[1][4 * u + e] = q[e];
      }
      if constexpr (sizeof(T) == 2) acc = mfma32_fp8(f[0], f[1], acc, sw[b], sx[b]);
    }
  }
  if (m >= a.M) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = blockIdx.x * 32 + fm_mfma32_row(r, lane);
    if (row < a.N) static_cast<T*>(a.y)[(long)m * a.N + row] = (T)acc[r];
  }
}

}  // namespace

extern "C" {

size_t fm_linear_fp8_workspace_bytes(long rows, int in_features, int out_features) { return 0; }

int fm_linear_fp8(const void* x, const void* x_scales, const void* weight, const void* weight_scales, long rows,
                  int in_features, int out_features, int dtype, void* y, float* workspace, size_t workspace_bytes,
                  hipStream_t stream) {
  if (rows < 0 || in_features <= 0 || out_features <= 0 || dtype < DT_F32 || dtype > DT_F16) return FM_BAD_ARGUMENT;
  if (in_features % 16 || rows > 32l * 65535) return FM_UNSUPPORTED;
  if (rows == 0) return FM_OK;
  if (!x || !x_scales || !weight || !weight_scales || !y) return FM_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight)) & 15) return FM_UNSUPPORTED;
  Linear a{};
  a.x = static_cast<const unsigned char*>(x), a.sx = static_cast<const unsigned char*>(x_scales);
  a.w = static_cast<const unsigned char*>(weight), a.sw = static_cast<const unsigned char*>(weight_scales);
  a.y = y, a.M = (int)rows, a.N = out_features, a.K = in_features, a.KB = fm_ceil_div(in_features, 128);
  const dim3 grid(fm_ceil_div(a.N, 32), fm_ceil_div(a.M, 32));
  if (dtype == DT_F32) hipLaunchKernelGGL(linear_simple_kernel<float>, grid, dim3(64), 0, stream, a);
  else if (dtype == DT_BF16) hipLaunchKernelGGL(linear_simple_kernel<__bf16>, grid, dim3(64), 0, stream, a);
  else hipLaunchKernelGGL(linear_simple_kernel<_Float16>, grid, dim3(64), 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"
