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

#include "fm_attention.h"

namespace {

// Key splits of the forward: a call of few rows over many keys (single tokens)
// has one block per 32 rows and key head; its keys are cut until some 512
// blocks run, at least four tiles (of 128 keys) each.
int forward_splits(const Attn& a) {
  const long blocks = (long)a.B * a.KV * fm_ceil_div((long)a.T * a.G, 32);
  const int tiles = fm_ceil_div(std::min<long>(a.S, (long)a.window + a.T - 1), 128);
  return (int)std::max<long>(1, std::min<long>({tiles / 4, 512 / std::max<long>(blocks, 1), 64}));
}

#define FM_ATTENTION_LAUNCH(kernel, own, rows, z)                                                       \
  do {                                                                                                  \
    const dim3 grid((unsigned)(a.B * a.KV), fm_ceil_div(rows, 32 * (own)), z);                          \
    if ((own) == 4) hipLaunchKernelGGL((kernel<T, DT, 4, 1, false>), grid, dim3(256), 0, stream, a);           \
    else if ((own) == 2) hipLaunchKernelGGL((kernel<T, DT, 2, 2, false>), grid, dim3(256), 0, stream, a);      \
    else hipLaunchKernelGGL((kernel<T, DT, 1, 4, false>), grid, dim3(256), 0, stream, a);                      \
  } while (0)

template <typename T, int DT>
int forward(const Attn& a, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  const int waves = a.splits > 1 ? 1 : own_waves(a, rows);
  FM_ATTENTION_LAUNCH(attention_forward_kernel, waves, rows, a.splits);
  if (a.splits > 1)
    hipLaunchKernelGGL((attention_join_kernel<T, DT, false>), dim3(fm_ceil_div(a.B * a.KV * rows, 4)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int DT>
int backward(const Attn& a, hipStream_t stream) {
  const long rows = (long)a.T * a.G;
  if (rows > 0) FM_ATTENTION_LAUNCH(attention_dq_kernel, own_waves(a, rows), rows, 1);
  const int own = own_waves(a, a.S);
  if constexpr (HELD<T, DT>) {
    const dim3 grid((unsigned)(a.B * a.KV), fm_ceil_div(a.S, 64));
    if ((long)grid.x * grid.y > 512) hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 2, false>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_dkv_kernel<T, DT, 2, 4, false>), grid, dim3(512), 0, stream, a);
  } else {
    FM_ATTENTION_LAUNCH(attention_dkv_kernel, own, a.S, 1);
  }
  return (int)hipGetLastError();
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
