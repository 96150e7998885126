// Rotary positions: pairs of a head's channels turned by the angle of their position,
// queries and keys in one launch, in either order of the pairs, the channels behind
// the rotated ones copied.  The gradient is the rotation by the opposite angle.
//
//   (a, b) -> scale (a cos - b sin, b cos + a sin),  angle = position * frequency
//
// The angle is counted in turns with its rounding error beside it in 64 bits, so that
// positions of any size lose nothing; what is left of it behind whole quarters goes
// through FP32 polynomials.  A thread has E pairs of one position, whose sines and cosines it
// forms once for its heads: less vector work per byte than memory takes, and no table to
// read.  Each element is read and written once, which is what bounds it.

#include "fm_common.h"

namespace {

struct Part {
  const void* x;
  void* y;  // [batch][length][heads][D]
  long batch, row, head;  // strides of x, elements
  int heads;
};

struct Rotary {
  Part q, k;  // k.heads may be 0
  const double* frequencies;
  const void* positions;  // [batch or 1][length] of 4 or 8 bytes, or NULL: first + 0, 1, ...
  long positions_batch, first;
  int wide, B, T, D, half, units, per_block, group;
  float scale, sign;
  FmDivisor by_units, by_length;
};

template <typename T, int E>
struct AnyVec {
  typedef typename Vec<T, E>::type type __attribute__((aligned(sizeof(T))));
};
template <typename T>
struct AnyVec<T, 1> {
  typedef typename Vec<T, 1>::type type;
};
template <typename T, int E>
FM_DEVICE typename Vec<T, E>::type any_load(const T* at) {
  return *reinterpret_cast<const typename AnyVec<T, E>::type*>(at);
}
template <typename T, int E>
FM_DEVICE void any_store(T* at, typename Vec<T, E>::type v) {
  *reinterpret_cast<typename AnyVec<T, E>::type*>(at) = v;
}

// Sine and cosine of position * frequency.  1 / (2 pi) is the sum of two doubles; with
// the products' remainders the turns are exact to 2^-90 of themselves, their fraction
// to 2^-53.  Within an eighth of a turn the Taylor terms up to the 9th and 10th power
// leave 2e-9 and 2e-10.
FM_DEVICE void turn(double position, double frequency, float& sine, float& cosine) {
  constexpr double HIGH = 0x1.45f306dc9c883p-3, LOW = -0x1.6b01ec5417056p-57;
  const double f = frequency * HIGH, f_low = fma(frequency, HIGH, -f) + frequency * LOW;
  const double t = position * f, t_low = fma(position, f, -t) + position * f_low;
  double r = (t - rint(t)) + t_low;
  const double quarter = rint(4.0 * r);
  r = fma(quarter, -0.25, r);
  const float a = (float)(r * 6.283185307179586), aa = a * a;
  float s = fmaf(aa, 1.0f / 362880, -1.0f / 5040);
  s = fmaf(aa, s, 1.0f / 120);
  s = fmaf(aa, s, -1.0f / 6);
  s = fmaf(a * aa, s, a);
  float c = fmaf(aa, -1.0f / 3628800, 1.0f / 40320);
  c = fmaf(aa, c, -1.0f / 720);
  c = fmaf(aa, c, 1.0f / 24);
  c = fmaf(aa, c, -0.5f);
  c = fmaf(aa, c, 1.0f);
  const int q = (int)quarter;
  sine = q & 1 ? c : s;
  cosine = q & 1 ? s : c;
  sine = q & 2 ? -sine : sine;
  cosine = (q + 1) & 2 ? -cosine : cosine;
}

template <typename T, int E, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary a) {
  const int local = (int)fm_div(threadIdx.x, a.by_units), unit = threadIdx.x - local * a.units;
  const long n = (long)blockIdx.x * a.per_block + local;
  if (local >= a.per_block || n >= (long)a.B * a.T) return;
  const int b = (int)fm_div((unsigned)n, a.by_length), t = (int)(n - (long)b * a.T);
  const int pair = unit * E;
  const bool turns = pair < a.half;
  float sine[E], cosine[E];
  if (turns) {
    double position = (double)(a.first + t);
    if (a.positions) {
      const long at = b * a.positions_batch + t;
      position = a.wide ? (double)static_cast<const long*>(a.positions)[at] : (double)static_cast<const int*>(a.positions)[at];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      turn(position, a.frequencies[pair + e], sine[e], cosine[e]);
      sine[e] *= a.sign, cosine[e] *= a.scale;
    }
  }
  // The unit's two vectors within a head; of the copied channels the last may have one.
  const int rest = 2 * a.half + 2 * (pair - a.half);
  const int first = turns ? (INTERLEAVED ? 2 * pair : pair) : rest;
  const int second = turns && !INTERLEAVED ? a.half + pair : first + E;
  const bool both = second < a.D;
  const int heads = a.q.heads + a.k.heads, h0 = blockIdx.y * a.group;
  for (int h = h0; h < min(h0 + a.group, heads); ++h) {
    const bool key = h >= a.q.heads;
    const Part& p = key ? a.k : a.q;
    const int head = key ? h - a.q.heads : h;
    const T* x = static_cast<const T*>(p.x) + b * p.batch + t * p.row + head * p.head;
    T* y = static_cast<T*>(p.y) + (n * p.heads + head) * a.D;
    typename Vec<T, E>::type u = any_load<T, E>(x + first), v{}, ou = u, ov;
    if (both) v = any_load<T, E>(x + second);
    ov = v;
    if (turns) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (INTERLEAVED && E > 1) {
          // Pairs 2 e and 2 e + 1 of the two vectors' values in a row.
          const float x0 = (float)(2 * e < E ? u[2 * e % E] : v[2 * e % E]);
          const float x1 = (float)(2 * e < E ? u[(2 * e + 1) % E] : v[(2 * e + 1) % E]);
          const float y0 = x0 * cosine[e] - x1 * sine[e], y1 = x1 * cosine[e] + x0 * sine[e];
          if (2 * e < E) ou[2 * e % E] = (T)y0, ou[(2 * e + 1) % E] = (T)y1;
          else ov[2 * e % E] = (T)y0, ov[(2 * e + 1) % E] = (T)y1;
        } else {
          const float x0 = (float)u[e], x1 = (float)v[e];
          ou[e] = (T)(x0 * cosine[e] - x1 * sine[e]);
          ov[e] = (T)(x1 * cosine[e] + x0 * sine[e]);
        }
      }
    }
    any_store<T, E>(y + first, ou);
    if (both) any_store<T, E>(y + second, ov);
  }
}

template <typename T, int E>
void launch(const Rotary& a, int interleaved, hipStream_t stream) {
  const long positions = (long)a.B * a.T;
  const dim3 grid(fm_ceil_div(positions, a.per_block), fm_ceil_div(a.q.heads + a.k.heads, a.group));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, E, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, E, false>), grid, dim3(256), 0, stream, a);
}

// Pairs of a thread: 16 bytes of each of its two vectors where both the rotated and the
// copied channels are whole vectors, 8, or single elements.
int pairs(const Rotary& a, int size) {
  for (int e : {16 / size, 4})
    if (a.half % e == 0 && (a.D - 2 * a.half) % e == 0) return e;
  return 1;
}

// Heads of a thread: as many as leave some 2048 threads a CU, at most 8.
int heads_of_a_thread(const Rotary& a) {
  const long threads = (long)a.B * a.T * a.units;
  const int heads = a.q.heads + a.k.heads;
  int group = 1;
  while (group < 8 && group < heads && threads * fm_ceil_div(heads, 2 * group) >= 256l * 2048) group *= 2;
  return group;
}

}  // namespace

extern "C" {

int fm_rotary(const void* q, long q_batch, long q_row, long q_head, int heads, const void* k, long k_batch, long k_row,
              long k_head, int kv_heads, const double* frequencies, const void* positions, long positions_batch,
              int positions_bytes, long first, int batch, int length, int head_dim, int rotated, int interleaved, float scale,
              int inverse, int dtype, void* q_out, void* k_out, hipStream_t stream) {
  if (batch < 0 || length < 0 || heads < 0 || kv_heads < 0 || head_dim <= 0 || rotated < 0 || rotated > head_dim || rotated % 2 ||
      dtype < DT_F32 || dtype > DT_F16 || (positions && positions_bytes != 4 && positions_bytes != 8) || scale != scale)
    return FM_BAD_ARGUMENT;
  if (head_dim > 512 || (long)batch * length > 1 << 24 || (long)heads + kv_heads > 65535) return FM_UNSUPPORTED;
  if (batch == 0 || length == 0 || heads + kv_heads == 0) return FM_OK;
  if ((heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)) || (rotated && !frequencies)) return FM_BAD_ARGUMENT;
  Rotary a{};
  a.q = Part{q, q_out, q_batch, q_row, q_head, heads}, a.k = Part{k, k_out, k_batch, k_row, k_head, kv_heads};
  a.frequencies = frequencies, a.positions = positions, a.positions_batch = positions_batch, a.first = first;
  a.wide = positions_bytes == 8, a.B = batch, a.T = length, a.D = head_dim, a.half = rotated / 2;
  a.scale = scale, a.sign = inverse ? -scale : scale;
  const int e = pairs(a, dtype == DT_F32 ? 4 : 2);
  a.units = a.half / e + fm_ceil_div(head_dim - rotated, 2 * e);
  a.per_block = 256 / a.units;
  a.by_units = fm_divisor((unsigned)a.units), a.by_length = fm_divisor((unsigned)length);
  a.group = heads_of_a_thread(a);
  if (dtype == DT_F32) {
    e == 4 ? launch<float, 4>(a, interleaved, stream) : launch<float, 1>(a, interleaved, stream);
  } else if (dtype == DT_BF16) {
    e == 8 ? launch<__bf16, 8>(a, interleaved, stream) : e == 4 ? launch<__bf16, 4>(a, interleaved, stream)
                                                                : launch<__bf16, 1>(a, interleaved, stream);
  } else {
    e == 8 ? launch<_Float16, 8>(a, interleaved, stream) : e == 4 ? launch<_Float16, 4>(a, interleaved, stream)
                                                                  : launch<_Float16, 1>(a, interleaved, stream);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
