// Codebook embedding for training: out[b][t] = scale * sum_q table[q][codes[b][q][t]],
// and its gradient by sorted codes, without atomics on values:
// dtable[q][e] = scale * (sum of dout[b][t] over the (b, t) whose code q is e,
// in ascending order of b, t).
//
// The gradient counts and places the rows of each codebook by code (a stable
// counting sort, one block a codebook), then one wave per entry gathers its
// rows and writes the entry once, zeros included.  Entries that own a large
// share of the rows (silence) would leave one wave with all of them, so whole
// runs of RUN sorted rows of one code are summed beforehand by waves of their
// own; the entry's wave adds those sums in their order.  Sums are FP32.

#include "fm_common.h"

namespace {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

constexpr int HISTOGRAMS = 32768;  // of LDS, in counters: waves x entries at most

struct Embed {
  const int64_t* codes;
  const void* table;
  const void* dout;
  void *out, *dtable;
  int *order, *start;  // [Q][rows], [Q][entries + 1]
  float* run;          // [Q][runs][D]: sums of whole runs of one code
  long codes_batch, codes_book, ld_dout;
  long rows;
  int frames, books, entries, D, run_rows, runs;
  FmDivisor by_frames;
  float scale;
};

template <typename T, int E>
struct Vec {
  typedef T type __attribute__((ext_vector_type(E)));
};
template <typename T>
struct Vec<T, 1> {
  struct type {
    T v;
    FM_DEVICE T& operator[](int) { return v; }
    FM_DEVICE const T& operator[](int) const { return v; }
  };
};

// One thread per E columns of an output row.  Code -1 is absent; any other
// code outside the table gives NaN.
template <typename T, int E>
__global__ __launch_bounds__(256) void embed_forward_kernel(Embed a) {
  typedef typename Vec<T, E>::type VT;
  const int n = a.D / E;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.rows * n) return;
  const long row = i / n;
  const int c = (int)(i - row * n);
  const int b = (int)fm_div((unsigned)row, a.by_frames), t = (int)(row - (long)b * a.frames);
  const int64_t* codes = a.codes + b * a.codes_batch + t;
  const VT* table = static_cast<const VT*>(a.table) + c;
  float s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.0f;
  constexpr int AHEAD = 8;  // codes, then entries, in flight together
  for (int q0 = 0; q0 < a.books; q0 += AHEAD) {
    int64_t code[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) code[u] = q0 + u < a.books ? codes[(q0 + u) * a.codes_book] : -1;
    VT v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      v[u] = VT{};
      if (code[u] >= 0 && code[u] < a.entries) v[u] = table[((long)(q0 + u) * a.entries + code[u]) * n];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const float bad = code[u] < -1 || code[u] >= a.entries ? NAN : 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] += (float)v[u][e] + bad;
    }
  }
  VT o;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = (T)(s[e] * a.scale);
  static_cast<VT*>(a.out)[i] = o;
}

// Stable counting sort of a codebook's rows by code.  The block's waves own
// consecutive shares of the rows and keep a histogram each (count[wave][e] in
// LDS); with the exclusive sums over (entry, wave) in its place, each wave
// walks its share 64 rows at a time, a row's place being its wave's next place
// of that entry plus the number of lower lanes with the same code.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void embed_sort_kernel(Embed a) {
  __shared__ int count[HISTOGRAMS];  // [WAVES][entries]
  __shared__ int totals[64 * WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, book = blockIdx.x;
  const int share = ((int)((a.rows + WAVES - 1) / WAVES) + 63) & ~63;
  const long first = (long)wave * share, last = min(a.rows, first + share);
  for (int i = tid; i < WAVES * a.entries; i += 64 * WAVES) count[i] = 0;
  __syncthreads();
  auto code_of = [&](long row) -> int {
    if (row >= last) return -1;
    const int b = (int)fm_div((unsigned)row, a.by_frames);
    const int64_t c = a.codes[b * a.codes_batch + book * a.codes_book + (row - (long)b * a.frames)];
    return c >= 0 && c < a.entries ? (int)c : -1;
  };
  int* mine = count + wave * a.entries;
  for (long r = first; r < last; r += 64) {
    const int c = code_of(r + lane);
    if (c >= 0) atomicAdd(&mine[c], 1);
  }
  __syncthreads();
  // Exclusive sums: each thread takes a run of entries, all waves of each.
  const int per = (a.entries + 64 * WAVES - 1) / (64 * WAVES);
  const int e0 = min(tid * per, a.entries), e1 = min(e0 + per, a.entries);
  int sum = 0;
  for (int e = e0; e < e1; ++e)
    for (int w = 0; w < WAVES; ++w) sum += count[w * a.entries + e];
  totals[tid] = sum;
  __syncthreads();
  for (int o = 1; o < 64 * WAVES; o <<= 1) {
    const int v = tid >= o ? totals[tid - o] : 0;
    __syncthreads();
    totals[tid] += v;
    __syncthreads();
  }
  int at = totals[tid] - sum;
  int* start = a.start + (long)book * (a.entries + 1);
  for (int e = e0; e < e1; ++e) {
    start[e] = at;
    for (int w = 0; w < WAVES; ++w) {
      const int v = count[w * a.entries + e];
      count[w * a.entries + e] = at;
      at += v;
    }
  }
  if (tid == 64 * WAVES - 1) start[a.entries] = totals[tid];
  __syncthreads();
  int* order = a.order + (long)book * a.rows;
  int bits = 0;
  while ((1 << bits) < a.entries) ++bits;
  for (long r = first; r < last; r += 64) {
    const int c = code_of(r + lane);
    // Lanes with the same code (absent ones form a group that is dropped).
    unsigned long long same = __ballot(c >= 0);
    same = c >= 0 ? same : ~same;
    for (int k = 0; k < bits; ++k) {
      const unsigned long long set = __ballot((c >> k) & 1);
      same &= (c >> k) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (c >= 0) {
      const int place = mine[c] + rank;
      order[place] = (int)(r + lane);
    }
    wave_lds_fence();
    if (c >= 0 && rank == 0) mine[c] += __popcll(same);
    wave_lds_fence();
  }
}

// The sum of n sorted rows of dout in order, E columns a lane.
template <typename T, int E>
FM_DEVICE void gather(const Embed& a, const int* order, int n, int c, bool live, int lane, float (&s)[E]) {
  typedef typename Vec<T, E>::type VT;
  constexpr int AHEAD = 8;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int mine = i0 + lane < n ? order[i0 + lane] : 0, m = min(64, n - i0);
    for (int i = 0; i < m; i += AHEAD) {
      VT v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        v[u] = VT{};
        const long row = __builtin_amdgcn_readlane(mine, min(i + u, m - 1));
        if (live && i + u < m) v[u] = reinterpret_cast<const VT*>(static_cast<const T*>(a.dout) + row * a.ld_dout)[c];
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += (float)v[u][e];
    }
  }
}

// Sums of the runs [RUN k, RUN k + RUN) of a codebook's sorted rows that lie
// within one entry; the others are left to the entry's own wave.
template <typename T, int E>
__global__ __launch_bounds__(256) void embed_run_kernel(Embed a) {
  const int lane = threadIdx.x & 63, run = blockIdx.x * 4 + (threadIdx.x >> 6), book = blockIdx.y;
  if (run >= a.runs) return;
  const int* start = a.start + (long)book * (a.entries + 1);
  const int first = run * a.run_rows, last = first + a.run_rows;
  if (last > start[a.entries]) return;
  // The entry of the run's first row: the last one that starts at or before it.
  int lo = 0, hi = a.entries;  // start[lo] <= first < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (start[mid] <= first) lo = mid;
    else hi = mid;
  }
  if (last > start[lo + 1]) return;
  const int c = blockIdx.z * 64 + lane, n = a.D / E;
  float s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.0f;
  gather<T, E>(a, a.order + (long)book * a.rows + first, a.run_rows, c, c < n, lane, s);
  if (c >= n) return;
  float* to = a.run + ((long)book * a.runs + run) * a.D + (long)c * E;
#pragma unroll
  for (int e = 0; e < E; ++e) to[e] = s[e];
}

// One wave per entry and 64 * E columns.
template <typename T, int E>
__global__ __launch_bounds__(256) void embed_entry_kernel(Embed a) {
  typedef typename Vec<T, E>::type VT;
  const int lane = threadIdx.x & 63, entry = blockIdx.x * 4 + (threadIdx.x >> 6), book = blockIdx.y;
  if (entry >= a.entries) return;
  const int c = blockIdx.z * 64 + lane, n = a.D / E;
  const int* start = a.start + (long)book * (a.entries + 1);
  const int first = start[entry], last = start[entry + 1];
  const int* order = a.order + (long)book * a.rows;
  float s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.0f;
  int head = last, tail = last;  // whole runs within [first, last): [head, tail)
  if (a.runs) {
    head = min((first + a.run_rows - 1) / a.run_rows * a.run_rows, last);
    tail = max(last / a.run_rows * a.run_rows, head);
  }
  gather<T, E>(a, order + first, head - first, c, c < n, lane, s);
  if (c < n)
    for (int r = head; r < tail; r += a.run_rows) {
      const float* from = a.run + ((long)book * a.runs + r / a.run_rows) * a.D + (long)c * E;
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] += from[e];
    }
  gather<T, E>(a, order + tail, last - tail, c, c < n, lane, s);
  if (c >= n) return;
  VT o;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = (T)(s[e] * a.scale);
  static_cast<VT*>(a.dtable)[((long)book * a.entries + entry) * n + c] = o;
}

int embed_check(const Embed& a, int batch, int dtype) {
  if (batch < 0 || a.frames < 0 || a.books <= 0 || a.entries <= 0 || a.D <= 0 || dtype < DT_F32 || dtype > DT_F16 ||
      a.codes_batch < 0 || a.codes_book < 0 || a.ld_dout < 0 || !(a.scale == a.scale))
    return FM_BAD_ARGUMENT;
  if (a.rows >= INT_MAX / 2 || a.entries > HISTOGRAMS || a.books > 65535) return FM_UNSUPPORTED;
  return FM_OK;
}

Embed embed_sizes(int batch, int books, int frames, int entries, int dim, float scale) {
  Embed a{};
  a.rows = (long)batch * frames;
  a.frames = frames, a.books = books, a.entries = entries, a.D = dim, a.scale = scale;
  a.by_frames = fm_divisor((unsigned)std::max(frames, 1));
  // Runs of about sqrt(rows): a code that owns every row is then as many run
  // sums as a run has rows.
  a.run_rows = 64;
  while ((long)a.run_rows * a.run_rows < a.rows) a.run_rows *= 2;
  a.runs = a.rows > 4 * a.run_rows ? (int)(a.rows / a.run_rows) : 0;
  return a;
}

struct Parts {
  size_t order, start, run, total;  // byte offsets
};
Parts parts(const Embed& a) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  Parts p{};
  p.start = up((size_t)a.books * a.rows * sizeof(int));
  p.run = p.start + up((size_t)a.books * (a.entries + 1) * sizeof(int));
  p.total = p.run + (size_t)a.books * a.runs * a.D * sizeof(float);
  return p;
}

bool aligned16(const Embed& a, int size) {
  uintptr_t u = 0;
  for (const void* p : {a.table, a.dout, (const void*)a.out, (const void*)a.dtable}) u |= reinterpret_cast<uintptr_t>(p);
  return (u & 15) == 0 && (a.D * size) % 16 == 0 && a.ld_dout * size % 16 == 0;
}

template <typename T, int E>
int embed_forward(const Embed& a, hipStream_t stream) {
  const long threads = a.rows * (a.D / E);
  if ((threads + 255) / 256 >= INT_MAX) return FM_UNSUPPORTED;
  hipLaunchKernelGGL((embed_forward_kernel<T, E>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int E>
int embed_backward(const Embed& a, hipStream_t stream) {
  // As many waves as histograms fit.
  if (a.entries <= HISTOGRAMS / 16)
    hipLaunchKernelGGL(embed_sort_kernel<16>, dim3(a.books), dim3(1024), 0, stream, a);
  else if (a.entries <= HISTOGRAMS / 4)
    hipLaunchKernelGGL(embed_sort_kernel<4>, dim3(a.books), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(embed_sort_kernel<1>, dim3(a.books), dim3(64), 0, stream, a);
  const unsigned slices = fm_ceil_div(a.D / E, 64);
  if (a.runs)
    hipLaunchKernelGGL((embed_run_kernel<T, E>), dim3(fm_ceil_div(a.runs, 4), a.books, slices), dim3(256), 0, stream, a);
  hipLaunchKernelGGL((embed_entry_kernel<T, E>), dim3(fm_ceil_div(a.entries, 4), a.books, slices), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

#define FM_EMBED_TYPES(run)                                                                       \
  (dtype == DT_F32    ? (aligned16(a, 4) ? run<float, 4>(a, stream) : run<float, 1>(a, stream))    \
   : dtype == DT_BF16 ? (aligned16(a, 2) ? run<__bf16, 8>(a, stream) : run<__bf16, 1>(a, stream))  \
                      : (aligned16(a, 2) ? run<_Float16, 8>(a, stream) : run<_Float16, 1>(a, stream)))

}  // namespace

extern "C" {

int fm_code_embedding(const int64_t* codes, long codes_batch, long codes_book, int batch, int books, int frames,
                      const void* table, int entries, int dim, float scale, int dtype, void* out, hipStream_t stream) {
  Embed a = embed_sizes(batch, books, frames, entries, dim, scale);
  a.codes = codes, a.codes_batch = codes_batch, a.codes_book = codes_book, a.table = table, a.out = out;
  if (const int status = embed_check(a, batch, dtype)) return status;
  if (a.rows == 0) return FM_OK;
  if (!codes || !table || !out) return FM_BAD_ARGUMENT;
  return FM_EMBED_TYPES(embed_forward);
}

size_t fm_code_embedding_backward_workspace_bytes(int batch, int books, int frames, int entries, int dim) {
  const Embed a = embed_sizes(batch, books, frames, entries, dim, 1.0f);
  return embed_check(a, batch, DT_F32) == FM_OK ? parts(a).total : 0;
}

int fm_code_embedding_backward(const void* dout, long ld_dout, const int64_t* codes, long codes_batch, long codes_book,
                               int batch, int books, int frames, int entries, int dim, float scale, int dtype, void* dtable,
                               void* workspace, size_t workspace_bytes, hipStream_t stream) {
  Embed a = embed_sizes(batch, books, frames, entries, dim, scale);
  a.codes = codes, a.codes_batch = codes_batch, a.codes_book = codes_book;
  a.dout = dout, a.ld_dout = ld_dout, a.dtable = dtable;
  if (const int status = embed_check(a, batch, dtype)) return status;
  if (!dtable || (a.rows > 0 && (!dout || !codes))) return FM_BAD_ARGUMENT;
  const Parts p = parts(a);
  if (!workspace || workspace_bytes < p.total) return FM_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return FM_UNSUPPORTED;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  a.order = reinterpret_cast<int*>(ws), a.start = reinterpret_cast<int*>(ws + p.start);
  a.run = reinterpret_cast<float*>(ws + p.run);
  return FM_EMBED_TYPES(embed_backward);
}

}  // extern "C"
