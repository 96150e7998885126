// LayerNorm for training: forward with the row statistics, and the backward
// pass with the weight and bias gradients.  FP32, bfloat16 and float16 inputs,
// FP32 or same-type weights; every sum in FP32.
//
//   forward   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), y = (x - mu) r w + b
//   backward  xh = (x - mu) r, g = dy w, dx = r (g - mean g - xh mean(g xh)),
//             dw = sum over rows of dy xh, db = sum over rows of dy
//
// Both are bound by memory: a row is read once, kept in registers, and reduced
// by the LPR lanes that hold it.

#include "fm_rows.h"

namespace {

struct Norm {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float *mean, *rstd, *part;  // part: [blocks][2][C]
  long rows, ld_x, ld_dy;
  int C, blocks;
  float eps;
};

// Lane p of a row holds vectors p, p + LPR, ... (NV of them, E elements each).
// 160000 x 512 FP32: 107 us, 6.1 TB/s.
template <typename T, typename W, int E, int NV, int LPR>
__global__ __launch_bounds__(256) void norm_forward_kernel(Norm a) {
  typedef typename Vec<T, E>::type VT;
  typedef typename Vec<W, E>::type VW;
  __shared__ float waves[2][4];
  const int p = threadIdx.x % LPR;
  const long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (row >= a.rows) return;
  const VT* x = reinterpret_cast<const VT*>(static_cast<const T*>(a.x) + row * a.ld_x);
  const int n = a.C / E;
  float v[NV][E];
  float s = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    VT t{};
    if (p + u * LPR < n) t = x[p + u * LPR];
#pragma unroll
    for (int e = 0; e < E; ++e) v[u][e] = widen(t[e]), s += v[u][e];
  }
  // The weights are on their way during the sums, where the registers allow (20000
  // rows: 8192 bfloat16 channels 144 -> 124 us, 2047 64 -> 51; 4095, with 32 single
  // elements a lane, 263 -> 293).
  constexpr bool EARLY = NV * E <= (E == 1 ? 8 : 32);
  const VW* w = static_cast<const VW*>(a.w);
  const VW* b = static_cast<const VW*>(a.b);
  VW wv[NV], bv[NV];
  auto weights = [&](int u) {
    const int i = p + u * LPR;
    wv[u] = bv[u] = VW{};
    if (w && i < n) wv[u] = w[i];
    if (b && i < n) bv[u] = b[i];
  };
  if constexpr (EARLY) {
#pragma unroll
    for (int u = 0; u < NV; ++u) weights(u);
  }
  const float mean = row_sum<LPR>(s, waves[0]) / (float)a.C;
  float q = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[u][e] = p + u * LPR < n ? v[u][e] - mean : 0.0f;
      q = fmaf(v[u][e], v[u][e], q);
    }
  const float rstd = 1.0f / sqrtf(row_sum<LPR>(q, waves[1]) / (float)a.C + a.eps);
  if (p == 0) a.mean[row] = mean, a.rstd[row] = rstd;
  VT* y = reinterpret_cast<VT*>(static_cast<T*>(a.y) + row * a.C);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = p + u * LPR;
    if (i >= n) break;
    if constexpr (!EARLY) weights(u);
    VT t;
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = (T)fmaf(v[u][e] * rstd, w ? widen(wv[u][e]) : 1.0f, b ? widen(bv[u][e]) : 0.0f);
    y[i] = t;
  }
}

// dx, and this block's share of dw and db: a row group walks rows blockIdx *
// groups + g, + gridDim * groups, ... with the columns' sums in registers; the
// block joins its groups through LDS in order and writes one partial row (or,
// when it is the only block, the gradients themselves).  160000 x 512 FP32: 195 us,
// 5.0 TB/s.
template <typename T, typename W, int E, int NV, int LPR>
__global__ __launch_bounds__(256) void norm_backward_kernel(Norm a) {
  typedef typename Vec<T, E>::type VT;
  typedef typename Vec<W, E>::type VW;
  constexpr int GROUPS = 256 / LPR;
  __shared__ float joined[256 * E], waves[2][2][4];
  const int p = threadIdx.x % LPR, g = threadIdx.x / LPR, n = a.C / E;
  float wv[NV][E], dw[NV][E], db[NV][E];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    VW t{};
    if (a.w && p + u * LPR < n) t = static_cast<const VW*>(a.w)[p + u * LPR];
#pragma unroll
    for (int e = 0; e < E; ++e) wv[u][e] = a.w ? widen(t[e]) : 1.0f, dw[u][e] = db[u][e] = 0.0f;
  }
  const float inv = 1.0f / (float)a.C;
  // The next row is on its way while this one is worked on, where the registers
  // allow (4000 x 512 FP32: 9.3 -> 8.0 us; long calls are bound by memory either way).
  constexpr bool AHEAD = NV * E <= 32;
  VT xv[NV], gv[NV], xn[NV], gn[NV];
  float mean, rstd, mean_n = 0.0f, rstd_n = 0.0f;
  const long step = (long)gridDim.x * GROUPS;
  auto load = [&](long row) {
    const VT* x = reinterpret_cast<const VT*>(static_cast<const T*>(a.x) + row * a.ld_x);
    const VT* dy = reinterpret_cast<const VT*>(static_cast<const T*>(a.dy) + row * a.ld_dy);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      xn[u] = gn[u] = VT{};
      if (p + u * LPR < n) xn[u] = x[p + u * LPR], gn[u] = dy[p + u * LPR];
    }
    mean_n = a.mean[row], rstd_n = a.rstd[row];
  };
  int turn = 0;
  long row = (long)blockIdx.x * GROUPS + g;
  if (AHEAD && row < a.rows) load(row);
  for (; row < a.rows; row += step) {
    if (!AHEAD) load(row);
#pragma unroll
    for (int u = 0; u < NV; ++u) xv[u] = xn[u], gv[u] = gn[u];
    mean = mean_n, rstd = rstd_n;
    if (AHEAD && row + step < a.rows) load(row + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float xh = (widen(xv[u][e]) - mean) * rstd, d = widen(gv[u][e]), t = d * wv[u][e];
        s1 += t;
        s2 = fmaf(t, xh, s2);
        dw[u][e] = fmaf(d, xh, dw[u][e]);
        db[u][e] += d;
      }
    row_sums<LPR>(s1, s2, waves[turn]);
    s1 *= inv, s2 *= inv, turn ^= 1;
    VT* dx = reinterpret_cast<VT*>(static_cast<T*>(a.dx) + row * a.C);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (p + u * LPR >= n) break;
      VT t;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float xh = (widen(xv[u][e]) - mean) * rstd;
        t[e] = (T)(rstd * (fmaf(widen(gv[u][e]), wv[u][e], -s1) - xh * s2));
      }
      dx[p + u * LPR] = t;
    }
  }
  if (!a.dw && !a.db) return;
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) joined[e * 256 + threadIdx.x] = k ? db[u][e] : dw[u][e];
      __syncthreads();
      if (g == 0 && p + u * LPR < n) {
        float s[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          s[e] = 0.0f;
          for (int j = 0; j < GROUPS; ++j) s[e] += joined[e * 256 + j * LPR + p];
        }
        const int c = (p + u * LPR) * E;
        if (a.blocks > 1) {
          float* to = a.part + ((long)blockIdx.x * 2 + k) * a.C + c;
#pragma unroll
          for (int e = 0; e < E; ++e) to[e] = s[e];
        } else if (W* to = static_cast<W*>(k ? a.db : a.dw)) {
#pragma unroll
          for (int e = 0; e < E; ++e) to[c + e] = (W)s[e];
        }
      }
    }
}

// Any number of channels and any alignment: one block per row (forward) or per
// run of rows (backward), the row read again for each step.  Column sums stay
// in the block's own partial rows.
template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_forward_any_kernel(Norm a) {
  __shared__ float sums[2][4];
  auto block_sum = [&](float v, int k) {
    v = row_sum<64>(v);
    if ((threadIdx.x & 63) == 0) sums[k][threadIdx.x >> 6] = v;
    __syncthreads();
    return (sums[k][0] + sums[k][1]) + (sums[k][2] + sums[k][3]);
  };
  const long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  float s = 0.0f;
  for (int c = threadIdx.x; c < a.C; c += 256) s += widen(x[c]);
  const float mean = block_sum(s, 0) / (float)a.C;
  float q = 0.0f;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float d = widen(x[c]) - mean;
    q = fmaf(d, d, q);
  }
  const float rstd = 1.0f / sqrtf(block_sum(q, 1) / (float)a.C + a.eps);
  if (threadIdx.x == 0) a.mean[row] = mean, a.rstd[row] = rstd;
  const W* w = static_cast<const W*>(a.w);
  const W* b = static_cast<const W*>(a.b);
  T* y = static_cast<T*>(a.y) + row * a.C;
  for (int c = threadIdx.x; c < a.C; c += 256)
    y[c] = (T)fmaf((widen(x[c]) - mean) * rstd, w ? widen(w[c]) : 1.0f, b ? widen(b[c]) : 0.0f);
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_backward_any_kernel(Norm a) {
  __shared__ float sums[2][2][4];
  const W* w = static_cast<const W*>(a.w);
  float* part = a.part + (long)blockIdx.x * 2 * a.C;
  bool first = true;
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1, first = false) {
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float xh = (widen(x[c]) - mean) * rstd, d = widen(dy[c]), g = d * (w ? widen(w[c]) : 1.0f);
      s1 += g;
      s2 = fmaf(g, xh, s2);
      if (a.dw || a.db) {
        part[c] = first ? d * xh : fmaf(d, xh, part[c]);
        part[a.C + c] = first ? d : part[a.C + c] + d;
      }
    }
    s1 = row_sum<64>(s1), s2 = row_sum<64>(s2);
    if ((threadIdx.x & 63) == 0) sums[turn][0][threadIdx.x >> 6] = s1, sums[turn][1][threadIdx.x >> 6] = s2;
    __syncthreads();
    s1 = ((sums[turn][0][0] + sums[turn][0][1]) + (sums[turn][0][2] + sums[turn][0][3])) / (float)a.C;
    s2 = ((sums[turn][1][0] + sums[turn][1][1]) + (sums[turn][1][2] + sums[turn][1][3])) / (float)a.C;
    T* dx = static_cast<T*>(a.dx) + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float xh = (widen(x[c]) - mean) * rstd;
      dx[c] = (T)(rstd * (fmaf(widen(dy[c]), w ? widen(w[c]) : 1.0f, -s1) - xh * s2));
    }
  }
}

// dw and db from the blocks' partial rows: 32 columns a block, 32 threads to a
// column, each summing every 32nd row in order, then joined in order.
template <typename W>
__global__ __launch_bounds__(1024) void norm_join_kernel(Norm a) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const long col = (long)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (col < 2l * a.C) {
    const float* from = a.part + col;
#pragma unroll 4
    for (int r = g; r < a.blocks; r += 32) s += from[(long)r * 2 * a.C];
  }
  sums[g][c] = s;
  __syncthreads();
  if (g != 0 || col >= 2l * a.C) return;
  float total = 0.0f;
#pragma unroll
  for (int j = 0; j < 32; ++j) total += sums[j][c];
  W* to = static_cast<W*>(col < a.C ? a.dw : a.db);
  if (to) to[col < a.C ? col : col - a.C] = (W)total;
}

// No rows: zero gradients.
template <typename W>
__global__ __launch_bounds__(256) void norm_zero_kernel(Norm a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  if (a.dw) static_cast<W*>(a.dw)[c] = (W)0.0f;
  if (a.db) static_cast<W*>(a.db)[c] = (W)0.0f;
}

int norm_check(const Norm& a, int dtype, int wtype) {
  if (a.rows < 0 || a.C <= 0 || dtype < DT_F32 || dtype > DT_F16 || (wtype != dtype && wtype != DT_F32) ||
      (a.rows > 1 && (a.ld_x < 0 || a.ld_dy < 0)))
    return FM_BAD_ARGUMENT;
  if (a.rows >= INT_MAX) return FM_UNSUPPORTED;
  return FM_OK;
}

bool aligned(const Norm& a, int size) {
  uintptr_t u = 0;
  for (const void* p : {a.x, a.dy, a.w, a.b, (const void*)a.y, (const void*)a.dx, (const void*)a.dw, (const void*)a.db})
    u |= reinterpret_cast<uintptr_t>(p);
  return (u & 15) == 0 && a.ld_x * size % 16 == 0 && a.ld_dy * size % 16 == 0;
}

template <typename T, typename W, int E, int NV, int LPR>
void launch(const Norm& a, bool back, hipStream_t stream) {
  if (back)
    hipLaunchKernelGGL((norm_backward_kernel<T, W, E, NV, LPR>), dim3(a.blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((norm_forward_kernel<T, W, E, NV, LPR>), dim3(fm_ceil_div(a.rows, 256 / LPR)), dim3(256), 0, stream,
                       a);
}

// False where the plan has no kernel (none of plan()'s).
template <typename T, typename W, int E>
bool launch_width(const Norm& a, const Plan& p, bool back, hipStream_t stream) {
  if (p.lpr == 16) return launch<T, W, E, 1, 16>(a, back, stream), true;
  if (p.lpr == 64) {
    if (p.nv == 1) return launch<T, W, E, 1, 64>(a, back, stream), true;
    if (p.nv == 2) return launch<T, W, E, 2, 64>(a, back, stream), true;
    if (p.nv == 4) return launch<T, W, E, 4, 64>(a, back, stream), true;
    if constexpr (E == 1)
      if (p.nv == 8) return launch<T, W, E, 8, 64>(a, back, stream), true;
  } else {
    if constexpr (E > 1)
      if (p.nv == 2) return launch<T, W, E, 2, 256>(a, back, stream), true;
    if (p.nv == 4) return launch<T, W, E, 4, 256>(a, back, stream), true;
    if constexpr (E < 8)
      if (p.nv == 8) return launch<T, W, E, 8, 256>(a, back, stream), true;
    if constexpr (E == 1)
      if (p.nv == 32) return launch<T, W, E, 32, 256>(a, back, stream), true;
  }
  return false;
}

template <typename T, typename W>
int run(Norm a, bool back, hipStream_t stream) {
  const Plan p = plan(a.C, sizeof(T), aligned(a, sizeof(T)));
  if (back && a.rows == 0) {
    hipLaunchKernelGGL((norm_zero_kernel<W>), dim3(fm_ceil_div(a.C, 256)), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
  }
  constexpr long MOST = 1 << 23;  // rows of a forward launch: a grid has at most 2^32 threads
  if (!back && a.rows > MOST) {
    Norm part = a;
    for (long first = 0; first < a.rows; first += MOST) {
      part.rows = std::min(MOST, a.rows - first);
      part.x = static_cast<const T*>(a.x) + first * a.ld_x;
      part.y = static_cast<T*>(a.y) + first * a.C;
      part.mean = a.mean + first, part.rstd = a.rstd + first;
      if (const int status = run<T, W>(part, false, stream)) return status;
    }
    return FM_OK;
  }
  a.blocks = back ? backward_blocks(a.rows, p, sizeof(T)) : 0;
  if (p.nv == 0) {
    if (back)
      hipLaunchKernelGGL((norm_backward_any_kernel<T, W>), dim3(a.blocks), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((norm_forward_any_kernel<T, W>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
  } else if (p.e == 1) {
    if (!launch_width<T, W, 1>(a, p, back, stream)) return FM_UNSUPPORTED;
  } else {
    if (!launch_width<T, W, 16 / sizeof(T)>(a, p, back, stream)) return FM_UNSUPPORTED;
  }
  if (back && (a.dw || a.db) && (a.blocks > 1 || p.nv == 0))
    hipLaunchKernelGGL((norm_join_kernel<W>), dim3(fm_ceil_div(2l * a.C, 32)), dim3(1024), 0, stream, a);
  return (int)hipGetLastError();
}

int run_types(const Norm& a, int dtype, int wtype, bool back, hipStream_t stream) {
  if (dtype == DT_F32) return run<float, float>(a, back, stream);
  if (dtype == DT_BF16) return wtype == DT_F32 ? run<__bf16, float>(a, back, stream) : run<__bf16, __bf16>(a, back, stream);
  return wtype == DT_F32 ? run<_Float16, float>(a, back, stream) : run<_Float16, _Float16>(a, back, stream);
}

}  // namespace

extern "C" {

int fm_layer_norm_forward(const void* x, long ld_x, const void* gamma, const void* beta, long rows, int channels, float eps,
                          int dtype, int weight_dtype, void* y, float* mean, float* rstd, hipStream_t stream) {
  Norm a{};
  a.x = x, a.w = gamma, a.b = beta, a.y = y, a.mean = mean, a.rstd = rstd;
  a.rows = rows, a.ld_x = ld_x, a.C = channels, a.eps = eps;
  if (const int status = norm_check(a, dtype, weight_dtype)) return status;
  if (rows == 0) return FM_OK;
  if (!x || !y || !mean || !rstd) return FM_BAD_ARGUMENT;
  return run_types(a, dtype, weight_dtype, false, stream);
}

// Room for the most blocks that any alignment of the same call runs; none where
// each of its plans is one block.
size_t fm_layer_norm_backward_workspace_bytes(long rows, int channels) {
  if (rows <= 0 || channels <= 0) return 0;
  if (rows <= (channels <= 512 ? 4 * ONE_BLOCK : channels <= 8192 ? ONE_BLOCK : 0)) return 0;
  return (size_t)std::min<long>(1024, rows) * 2 * channels * sizeof(float);
}

int fm_layer_norm_backward(const void* dy, long ld_dy, const void* x, long ld_x, const void* gamma, const float* mean,
                           const float* rstd, long rows, int channels, int dtype, int weight_dtype, void* dx, void* dgamma,
                           void* dbeta, float* workspace, size_t workspace_bytes, hipStream_t stream) {
  Norm a{};
  a.x = x, a.dy = dy, a.w = gamma, a.dx = dx, a.dw = dgamma, a.db = dbeta;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.part = workspace;
  a.rows = rows, a.ld_x = ld_x, a.ld_dy = ld_dy, a.C = channels;
  if (const int status = norm_check(a, dtype, weight_dtype)) return status;
  if (rows == 0 && !dgamma && !dbeta) return FM_OK;
  if (rows > 0 && (!x || !dy || !dx || !mean || !rstd)) return FM_BAD_ARGUMENT;
  if (rows > 0 && (dgamma || dbeta) &&
      workspace_bytes < fm_layer_norm_backward_workspace_bytes(rows, channels))
    return FM_WORKSPACE_TOO_SMALL;
  if (workspace_bytes > 0 && !workspace) return FM_BAD_ARGUMENT;
  return run_types(a, dtype, weight_dtype, true, stream);
}

}  // extern "C"
