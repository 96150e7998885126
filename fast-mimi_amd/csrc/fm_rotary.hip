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
// read.  Each element is read and written once, which is what bounds it: 8 x 4095 positions,
// 16 + 4 heads of 128, bfloat16, 336 MB in 64 us (5.2 TB/s; a large copy reaches 4.9); 64 single
// tokens 4.3 us, by latency.

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
  long positions_batch, first, start;  // start: of this launch's positions
  int wide, B, T, D, half, turns, units, per_block, group, groups;  // units of a position: the first `turns` turn pairs
  float scale, sign;
  FmDivisor by_units, by_length, by_groups;
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
template <bool PAST, typename T, int E>
FM_DEVICE void any_store(T* at, typename Vec<T, E>::type v) {
  auto to = reinterpret_cast<typename AnyVec<T, E>::type*>(at);
  if constexpr (PAST && E > 1) __builtin_nontemporal_store(v, to);
  else *to = v;
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

// A unit is a thread's two vectors within a head, neighbouring threads' side by side in
// memory.  Pairs apart: one vector of the first partners and one of the second, or two that
// are copied.  Pairs side by side (whole pairs in a vector): two vectors half a head
// apart, each turned or copied.  PAST: results go past the L2.
template <typename T, int E, bool INTERLEAVED, bool PAST>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary a) {
  constexpr bool WITHIN = INTERLEAVED && E > 1;
  const int local = (int)fm_div(threadIdx.x, a.by_units), unit = threadIdx.x - local * a.units;
  // Neighbouring blocks take the heads of the same positions: whole rows are read at a time.
  const int block = (int)fm_div(blockIdx.x, a.by_groups), h0 = (blockIdx.x - block * a.groups) * a.group;
  const long n = a.start + (long)block * a.per_block + local;
  if (local >= a.per_block || n >= (long)a.B * a.T) return;
  const int b = (int)fm_div((unsigned)n, a.by_length), t = (int)(n - (long)b * a.T);
  const bool turns = WITHIN || unit < a.turns;
  int first = unit * E, second = first + a.units * E;
  if constexpr (!WITHIN) {
    if (!turns) first = 2 * a.half + (unit - a.turns) * E, second = first + (a.units - a.turns) * E;
    else if (INTERLEAVED) first = 2 * unit, second = first + 1;
    else second = a.half + first;
  }
  const bool both = second < a.D;
  float sine[E], cosine[E];
  if (turns) {
    double position = (double)(a.first + t);
    if (a.positions) {
      const long at = b * a.positions_batch + t;
      position = a.wide ? (double)static_cast<const long*>(a.positions)[at] : (double)static_cast<const int*>(a.positions)[at];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int pair = !WITHIN ? unit * E + e : 2 * e < E ? first / 2 + e : second / 2 + e - E / 2;
      if (WITHIN && pair >= a.half) sine[e] = 0.0f, cosine[e] = 1.0f;  // copied, below
      else turn(position, a.frequencies[pair], sine[e], cosine[e]), sine[e] *= a.sign, cosine[e] *= a.scale;
    }
  }
  const int heads = a.q.heads + a.k.heads;
  for (int h = h0; h < min(h0 + a.group, heads); ++h) {
    const bool key = h >= a.q.heads;
    const Part& p = key ? a.k : a.q;
    const int head = key ? h - a.q.heads : h;
    const T* x = static_cast<const T*>(p.x) + b * p.batch + t * p.row + head * p.head;
    T* y = static_cast<T*>(p.y) + (n * p.heads + head) * a.D;
    typename Vec<T, E>::type u = any_load<T, E>(x + first), v{}, ou = u, ov;
    if (both) v = any_load<T, E>(x + second);
    ov = v;
    if constexpr (WITHIN) {
      auto turned = [&](const auto& from, auto& to, int e0) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const float x0 = (float)from[2 * e], x1 = (float)from[2 * e + 1];
          to[2 * e] = (T)(x0 * cosine[e0 + e] - x1 * sine[e0 + e]);
          to[2 * e + 1] = (T)(x1 * cosine[e0 + e] + x0 * sine[e0 + e]);
        }
      };
      if (first < 2 * a.half) turned(u, ou, 0);
      if (second < 2 * a.half) turned(v, ov, E / 2);
    } else if (turns) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x0 = (float)u[e], x1 = (float)v[e];
        ou[e] = (T)(x0 * cosine[e] - x1 * sine[e]);
        ov[e] = (T)(x1 * cosine[e] + x0 * sine[e]);
      }
    }
    any_store<PAST, T, E>(y + first, ou);
    if (both) any_store<PAST, T, E>(y + second, ov);
  }
}

template <typename T, int E>
void launch(Rotary a, int interleaved, hipStream_t stream) {
  const long positions = (long)a.B * a.T;
  const int heads = a.q.heads + a.k.heads;
  // A grid has fewer than 2^32 threads.
  const long most = std::max(1, ((1 << 24) - 1) / a.groups) * (long)a.per_block;
  // Results of 128 MB or more, half of the last-level cache, go past the L2, where neighbouring
  // threads' stores fill 64 bytes at a time (16-bit, caches / past: 8 x 4095 positions, 20 heads of 128,
  // 168 MB 78 / 52 us; 32 x 2500, 24 of 64, 246 MB 122 / 92; 16 x 2500, 123 MB 41 / 48; 20 of 80, 102 MB 26 / 50).
  const int side_by_side = (interleaved ? a.units : a.units > a.turns ? std::min(a.turns, a.units - a.turns) : a.turns) * E;
  const bool past = E > 1 && positions * heads * a.D * (long)sizeof(T) >= 128l << 20 && side_by_side * sizeof(T) % 64 == 0;
  for (; a.start < positions; a.start += most) {
    const dim3 grid(fm_ceil_div(std::min(most, positions - a.start), a.per_block) * a.groups);
    if (past && interleaved) hipLaunchKernelGGL((rotary_kernel<T, E, true, true>), grid, dim3(256), 0, stream, a);
    else if (past) hipLaunchKernelGGL((rotary_kernel<T, E, false, true>), grid, dim3(256), 0, stream, a);
    else if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, E, true, false>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<T, E, false, false>), grid, dim3(256), 0, stream, a);
  }
}

// Elements of a vector: 16 bytes where turned and copied channels are whole vectors (and
// whole pairs), 8, or one.
int elements(const Rotary& a, int size, bool interleaved) {
  const int turned = interleaved ? 2 * a.half : a.half;
  for (int e : {16 / size, 4})
    if (turned % e == 0 && (a.D - 2 * a.half) % e == 0) return e;
  return 1;
}

// Heads of a thread: two share its sines and cosines, where some 2048 threads a CU remain
// (8 x 4095 positions, 20 heads of 128, one / two / four / eight: 56 / 52 / 53 / 54 us; 250, one / two: 3.7 / 4.0).
int heads_of_a_thread(const Rotary& a) {
  return (long)a.B * a.T * a.units * fm_ceil_div(a.q.heads + a.k.heads, 2) >= 256l * 2048 ? 2 : 1;
}

}  // namespace

extern "C" {

int fm_rotary(const void* q, long q_batch, long q_row, long q_head, int heads, const void* k, long k_batch, long k_row,
              long k_head, int kv_heads, const double* frequencies, const void* positions, long positions_batch,
              int positions_bytes, long first, int batch, int length, int head_dim, int rotated, int interleaved, float scale,
              int inverse, int dtype, void* q_out, void* k_out, hipStream_t stream) {
  if (batch < 0 || length < 0 || heads < 0 || kv_heads < 0 || head_dim <= 0 || rotated < 0 || rotated > head_dim || rotated % 2 ||
      dtype < DT_F32 || dtype > DT_F16 || (positions && positions_bytes != 4 && positions_bytes != 8) || !std::isfinite(scale))
    return FM_BAD_ARGUMENT;
  if (head_dim > 512 || (long)batch * length > 1 << 24 || (long)heads + kv_heads > 65535) return FM_UNSUPPORTED;
  if (batch == 0 || length == 0 || heads + kv_heads == 0) return FM_OK;
  if ((heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)) || (rotated && !frequencies)) return FM_BAD_ARGUMENT;
  Rotary a{};
  a.q = Part{q, q_out, q_batch, q_row, q_head, heads}, a.k = Part{k, k_out, k_batch, k_row, k_head, kv_heads};
  a.frequencies = frequencies, a.positions = positions, a.positions_batch = positions_batch, a.first = first;
  a.wide = positions_bytes == 8, a.B = batch, a.T = length, a.D = head_dim, a.half = rotated / 2;
  a.scale = scale, a.sign = inverse ? -scale : scale;
  const int e = elements(a, dtype == DT_F32 ? 4 : 2, interleaved != 0);
  a.turns = a.half / e, a.units = a.turns + fm_ceil_div(head_dim - rotated, 2 * e);
  if (interleaved && e > 1) a.units = fm_ceil_div(head_dim, 2 * e);
  a.per_block = 256 / a.units;
  a.by_units = fm_divisor((unsigned)a.units), a.by_length = fm_divisor((unsigned)length);
  a.group = heads_of_a_thread(a), a.groups = fm_ceil_div(heads + kv_heads, a.group);
  a.by_groups = fm_divisor((unsigned)a.groups);
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
