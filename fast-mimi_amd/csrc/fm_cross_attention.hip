// Attention to the states of another sequence, forward and backward, for training
// and for single tokens: every query sees keys 0 .. key_lengths[b] - 1, whatever its
// position.  FP32, bfloat16 and float16; grouped query heads; padded queries and keys.
//
//   S = Q K^T c, P = exp2(S - max), O = P V / sum P      (c = scale log2 e)
//   P = exp2(S - lse), D = rowsum(dO O), dS = P (dO V^T - D)
//   dQ = dS K scale, dV = P^T dO, dK = dS^T Q scale
//
// The tiles, operands and loops are the causal kernels' (fm_attention.h) without their
// window.  What differs is the shape of the calls: the two lengths have nothing to do
// with each other, so either may be too short to fill the chip.  A forward or dQ block
// walks the keys and a dK / dV block the rows of its sequence; where there are few blocks and a
// long walk, it is cut, and the parts are joined in their order.
//
// Long calls are bound by the matrix cores and the exponentials beside them, dK / dV with heads of 128
// by LDS reads: 2 x 4095 over 4001, 16 / 4 heads of 128, bfloat16: forward 317 us (850 TFLOP/s), dQ 510,
// dK / dV 771 (under the tracer; the whole pass 1500).  2500 over up to 300 keys, 8 heads of 64, 8 items: 25, 43, 50 and the
// join 7 us (120).  FP32, 4 x 2048 over 1024, 8 / 4 heads of 128: 294, 473, 659 us (117, 109 and 104 TFLOP/s).  A token over
// 8000 keys by memory: 8 items, 16 / 4 heads of 64, float16, 66 MB in 13.4 us (4.9 TB/s), the join 4.

#include "fm_attention.h"

namespace {

// dQ, or dK and dV, from the parts of a cut walk: four of the DT columns a lane, eight parts in
// flight (2500 over 8 x 300 keys, 8 heads of 64, bfloat16, three parts: with one column a lane the backward
// takes 113 us, with four 105; 3 over 4000, 8 / 2 heads of 64, 16 parts: both 18).
template <typename T, int DT, bool KEYS>
__global__ __launch_bounds__(256) void cross_join_kernel(Attn a) {
  constexpr int LPR = DT / 4, AHEAD = 8;
  const int lane = threadIdx.x % LPR, col = 4 * lane, R = a.T * a.G;
  const long seqs = (long)a.B * a.KV, rows = KEYS ? 2 * seqs * a.S : seqs * R;
  const long at = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (at >= rows) return;
  floatx4 sum = {};
  for (int s = 0; s < a.splits; s += AHEAD) {
    floatx4 v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      v[u] = *reinterpret_cast<const floatx4*>(a.part_o + (min(s + u, a.splits - 1) * rows + at) * DT + col);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) sum += s + u < a.splits ? v[u] : floatx4{};
  }
  T* out;
  if constexpr (KEYS) {
    const long which = at / (seqs * a.S), row = at - which * seqs * a.S, seq = row / a.S, key = row - seq * a.S;
    const long b = seq / a.KV, kh = seq - b * a.KV;
    out = static_cast<T*>(which ? a.dv : a.dk) + ((b * a.S + key) * a.KV + kh) * a.D;
  } else {
    const int seq = (int)(at / R), r = (int)(at - (long)seq * R), b = seq / a.KV, kh = seq - b * a.KV, t = (int)fm_div(r, a.by_g);
    const long row = ((long)b * a.T + t) * a.H + kh * a.G + (r - t * a.G);
    out = static_cast<T*>(a.out) + row * a.D;
    // The sum of dS puts rowsum(dO O) from the rounded O right (see attention_dq_kernel).
    if (sizeof(T) == 2) {
      float rest = 0.0f;
      for (int s = lane; s < a.splits; s += LPR) rest += a.part_ml[s * rows + at];
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) rest += __shfl_xor(rest, o, 64);
      if (lane == 0) a.stats[(long)a.B * a.T * a.H + row] += rest;
    }
  }
  typename Vec<T, 4>::type y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)sum[e];
  if (col < a.D) *reinterpret_cast<typename Vec<T, 4>::type*>(out + col) = y;
}

long sequences(const Attn& a) { return (long)a.B * a.KV; }

// Into how many parts a walk of `tiles` (of 128) is cut that `blocks` blocks, 256 at most, make for `results` rows.
// What a number of them takes, in half tiles: as many rounds of 256 blocks, or, in 16 bits, one of 256 or some of 512
// that take half as long again, as they need, and what a second launch and the parts' way through memory cost.
// Uncut / cut (us): forward 250 over 1000, 8 heads of 64, FP32 31.6 / 17.6, bfloat16 11.7 / 11.0; 1 over 3611, 2 of
// 128, FP32 (29 parts) 40 / 17; 30 over 300, 4 of 64 (3), FP32 15.9 / 12.8, bfloat16 7.4 / 9.4; 500 over 500, 16 of
// 128 (2), FP32 31 / 46; 3 x 168 over 3812, 8 of 64 (5), FP32 104 / 77.  256 / 512 blocks: 120 over 4000, 8 of 64, bfloat16
// 12.7 / 13.7, 4000 over 4000, one of 64, bfloat16 23.5 / 20.8.  Two tiles a part / one: 1 over 8000, 4 key heads of 64,
// float16 12.3 / 13.4.  dK / dV: 400 over 30, 4 of 64, bfloat16 (4) 20.4 / 17.7, 500 over 500, 8 of 128 (4) 32.7 / 38.1.
int cut(const Attn& a, long blocks, int tiles, long results, bool wide) {
  if (blocks == 0 || blocks > 256) return 1;
  const long most = std::min(64, wide ? tiles : std::max(std::min(tiles, 8), tiles / 2));
  int best = 1;
  long least = 2 * tiles + 1;
  auto consider = [&](long parts) {
    if (parts < 2) return;
    const long n = blocks * parts, rounds = wide ? 2 * ((n + 255) / 256) : n <= 256 ? 2 : 3 * ((n + 511) / 512);
    const long cost = rounds * ((tiles + parts - 1) / parts) + 2 * (!wide ? 3 + parts * results / 4096 : a.D > 64 ? 1 : 2);
    if (cost < least) least = cost, best = (int)parts;
  };
  for (long parts = 2; parts <= std::min(most, 8l); ++parts) consider(parts);
  consider(std::min(most, 256 / blocks)), consider(std::min(most, 512 / blocks));
  return best;
}

// A block's waves with rows (or keys) of their own: four where that leaves 384 blocks, two where 256
// (heads beyond 64: 192) are left, else one, but those that share them have 32 each at least to walk.  With two / four (us):
// forward 2 x 4096 over 500, 8 heads of 64 (512 blocks of 128 rows) 21.3 / 20.0, 4 x 2000 over 500, 8 / 2 heads
// of 128 (504) 37 / 31, 2 x 1000 over 1000, 16 / 4 heads of 128 (256) 31.7 / 34.4; with one / two: 2000 over
// 200, 8 / 2 heads of 128 (250 of 64) 17.0 / 11.4, 7 x 1069 over 1004, 2 of 64 (238) 15.6 / 17.9.  With one / two / four: 13
// over 7, FP32 9.1 / 8.1 / 7.4; 13 over 40 9.1 / 8.0 / 9.3; 60 over 100, 8 heads of 128, FP32 13.2 / 17.9 / 23.6.
int waves_apart(const Attn& a, long own, long walked) {
  const long seqs = sequences(a);
  const int most = seqs * fm_ceil_div(own, 128) >= 384 ? 4 : seqs * fm_ceil_div(own, 64) >= (a.D > 64 ? 192 : 256) ? 2 : 1;
  return std::max(most, walked <= 32 || (most == 2 && walked < 128) ? 4 : walked <= 64 ? 2 : 1);
}

struct Shape {
  int waves, splits;
};
Shape row_shape(const Attn& a, bool wide) {  // forward, dQ; wide: FP32
  const long rows = (long)a.T * a.G;
  const int splits = cut(a, sequences(a) * fm_ceil_div(rows, 32), fm_ceil_div(a.S, 128), sequences(a) * rows, wide);
  return {splits > 1 ? 1 : waves_apart(a, rows, a.S), splits};
}
// dK / dV.  Where the blocks are no two to a CU, long walks are cut as well, if that fills the
// rounds of 512 to nine tenths (whole backward, uncut / so, us: 8 x 2500 over 300, 8 heads of 64, FP32 320 / 284,
// bfloat16 110 / 106, with lengths from 0 to 300 101 / 98; 4 x 2048 over 1024, 8 / 4 heads of 64, FP32 394 / 338).
Shape key_shape(const Attn& a, bool wide) {
  const long rows = (long)a.T * a.G;
  const int own = !wide && a.D > 64 ? 64 : 32;  // keys of a block that is cut
  const int tiles = fm_ceil_div(rows, 128), splits = cut(a, sequences(a) * fm_ceil_div(a.S, own), tiles, sequences(a) * a.S, wide);
  if (splits > 1) return {1, splits};
  const int waves = waves_apart(a, a.S, rows);
  const long blocks = sequences(a) * fm_ceil_div(a.S, 32 * waves);
  if (blocks < 512 && a.D <= 64)
    for (int s = 1; s <= tiles / 6; ++s)
      if (10 * blocks * s >= 9 * ((blocks * s + 511) / 512 * 512)) return {waves, s};
  return {waves, 1};
}

size_t backward_floats(const Attn& a, bool wide) {
  const size_t dt = a.D > 64 ? 128 : 64;
  const size_t q = row_shape(a, wide).splits, k = key_shape(a, wide).splits;
  return std::max(q > 1 ? q * sequences(a) * a.T * a.G * (dt + 1) : 0, k > 1 ? k * 2 * sequences(a) * a.S * dt : 0);
}

#define FM_CROSS_LAUNCH(kernel, own, rows, z)                                                                \
  do {                                                                                                       \
    const dim3 grid((unsigned)sequences(a), fm_ceil_div(rows, 32 * (own)), z);                               \
    if ((own) == 4) hipLaunchKernelGGL((kernel<T, DT, 4, 1, true>), grid, dim3(256), 0, stream, a);          \
    else if ((own) == 2) hipLaunchKernelGGL((kernel<T, DT, 2, 2, true>), grid, dim3(256), 0, stream, a);     \
    else hipLaunchKernelGGL((kernel<T, DT, 1, 4, true>), grid, dim3(256), 0, stream, a);                     \
  } while (0)

template <typename T, int DT>
int cross_forward(Attn a, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  FM_CROSS_LAUNCH(attention_forward_kernel, row_shape(a, sizeof(T) == 4).waves, rows, a.splits);
  if (a.splits > 1)
    hipLaunchKernelGGL((attention_join_kernel<T, DT, true>), dim3(fm_ceil_div(sequences(a) * rows, 4)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int DT>
int cross_backward(Attn a, float* workspace, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  a.part_o = workspace;
  if (rows > 0) {
    const Shape shape = row_shape(a, sizeof(T) == 4);
    a.splits = shape.splits;
    a.part_ml = workspace + (size_t)a.splits * sequences(a) * rows * DT;
    FM_CROSS_LAUNCH(attention_dq_kernel, shape.waves, rows, a.splits);
    if (a.splits > 1)
      hipLaunchKernelGGL((cross_join_kernel<T, DT, false>), dim3(fm_ceil_div(sequences(a) * rows, 1024 / DT)), dim3(256), 0, stream, a);
  }
  if (a.S > 0) {
    const Shape shape = key_shape(a, sizeof(T) == 4);
    a.splits = shape.splits;
    if constexpr (HELD<T, DT>) {
      const dim3 grid((unsigned)sequences(a), fm_ceil_div(a.S, 64), a.splits);
      if ((long)grid.x * grid.y * grid.z > 512)
        hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 2, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 4, true>), grid, dim3(512), 0, stream, a);
    } else {
      FM_CROSS_LAUNCH(attention_dkv_kernel, shape.waves, a.S, a.splits);
    }
    if (a.splits > 1)
      hipLaunchKernelGGL((cross_join_kernel<T, DT, true>), dim3(fm_ceil_div(2 * sequences(a) * a.S, 1024 / DT)), dim3(256), 0, stream, a);
  }
  return (int)hipGetLastError();
}

// Joins need no limit of their own: only walks of fewer than 512 blocks, of 128 rows or keys at most, are cut.
int cross_check(const Attn& a, int dtype) { return check(a, dtype, true); }

Attn cross_sizes(int batch, int queries, int keys, int heads, int kv_heads, int head_dim, float scale) {
  Attn a{};
  a.B = batch, a.T = queries, a.S = keys, a.H = heads, a.KV = kv_heads, a.D = head_dim;
  a.G = kv_heads > 0 && heads > 0 ? heads / kv_heads : 1;
  a.window = 1, a.scale = scale, a.scale2 = scale * LOG2E, a.splits = 1;
  a.by_g = fm_divisor((unsigned)std::max(a.G, 1));
  return a;
}

}  // namespace

extern "C" {

size_t fm_cross_attention_forward_workspace_bytes(int batch, int queries, int keys, int heads, int kv_heads, int head_dim) {
  const Attn a = cross_sizes(batch, queries, keys, heads, kv_heads, head_dim, 1.0f);
  if (cross_check(a, DT_F32) != FM_OK && cross_check(a, DT_BF16) != FM_OK) return 0;
  if (batch == 0 || queries == 0) return 0;
  return workspace_floats(a, std::max(row_shape(a, true).splits, row_shape(a, false).splits)) * sizeof(float);
}

int fm_cross_attention_forward(const void* q, long q_batch, long q_row, long q_head, const void* k, long k_batch, long k_row,
                               long k_head, const void* v, long v_batch, long v_row, long v_head, const int* key_lengths,
                               const int* query_lengths, int batch, int queries, int keys, int heads, int kv_heads,
                               int head_dim, float scale, int dtype, void* out, float* lse, float* workspace,
                               size_t workspace_bytes, hipStream_t stream) {
  Attn a = cross_sizes(batch, queries, keys, heads, kv_heads, head_dim, scale);
  a.q = View{q, q_batch, q_row, q_head}, a.k = View{k, k_batch, k_row, k_head}, a.v = View{v, v_batch, v_row, v_head};
  a.lengths = key_lengths, a.query_lengths = query_lengths, a.out = out, a.lse = lse;
  if (const int status = cross_check(a, dtype)) return status;
  if (batch == 0 || queries == 0) return FM_OK;
  if (!q || !out || !lse || (keys > 0 && (!k || !v))) return FM_BAD_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(out) & 15) return FM_UNSUPPORTED;
  a.splits = row_shape(a, dtype == DT_F32).splits;
  if (a.splits > 1) {
    if (!workspace || workspace_bytes < workspace_floats(a, a.splits) * sizeof(float)) return FM_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FM_UNSUPPORTED;
    a.part_o = workspace;
    a.part_ml = workspace + (size_t)a.splits * sequences(a) * a.T * a.G * (a.D > 64 ? 128 : 64);
  }
  return FM_ATTENTION_TYPES(cross_forward);
}

size_t fm_cross_attention_backward_workspace_bytes(int batch, int queries, int keys, int heads, int kv_heads, int head_dim) {
  const Attn a = cross_sizes(batch, queries, keys, heads, kv_heads, head_dim, 1.0f);
  if (cross_check(a, DT_F32) != FM_OK && cross_check(a, DT_BF16) != FM_OK) return 0;
  return batch == 0 || queries == 0 ? 0 : std::max(backward_floats(a, true), backward_floats(a, false)) * sizeof(float);
}

int fm_cross_attention_backward(const void* dout, long dout_batch, long dout_row, long dout_head, const void* q, long q_batch,
                                long q_row, long q_head, const void* k, long k_batch, long k_row, long k_head, const void* v,
                                long v_batch, long v_row, long v_head, const void* out, const float* lse,
                                const int* key_lengths, const int* query_lengths, int batch, int queries, int keys, int heads,
                                int kv_heads, int head_dim, float scale, int dtype, void* dq, void* dk, void* dv, float* stats,
                                float* workspace, size_t workspace_bytes, hipStream_t stream) {
  Attn a = cross_sizes(batch, queries, keys, heads, kv_heads, head_dim, scale);
  a.q = View{q, q_batch, q_row, q_head}, a.k = View{k, k_batch, k_row, k_head}, a.v = View{v, v_batch, v_row, v_head};
  a.dout = View{dout, dout_batch, dout_row, dout_head};
  a.o = out, a.lengths = key_lengths, a.query_lengths = query_lengths, a.lse = const_cast<float*>(lse);
  a.out = dq, a.dk = dk, a.dv = dv, a.stats = stats;
  if (const int status = cross_check(a, dtype)) return status;
  if (batch == 0 || queries == 0) return batch == 0 || keys == 0 ? FM_OK : FM_BAD_ARGUMENT;
  if (!dout || !q || !out || !lse || !dq || !stats || (keys > 0 && (!k || !v || !dk || !dv))) return FM_BAD_ARGUMENT;
  for (const void* p : {out, (const void*)dq, (const void*)dk, (const void*)dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return FM_UNSUPPORTED;
  if (const size_t need = backward_floats(a, dtype == DT_F32) * sizeof(float)) {
    if (!workspace || workspace_bytes < need) return FM_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FM_UNSUPPORTED;
  }
  const auto run = [&](auto kernel) { return kernel(a, workspace, stream); };
  const bool wide = a.D > 64;
  if (dtype == DT_F32) return wide ? run(cross_backward<float, 128>) : run(cross_backward<float, 64>);
  if (dtype == DT_BF16) return wide ? run(cross_backward<__bf16, 128>) : run(cross_backward<__bf16, 64>);
  return wide ? run(cross_backward<_Float16, 128>) : run(cross_backward<_Float16, 64>);
}

}  // extern "C"
