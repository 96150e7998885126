// Codebook embedding for training: out[b][t] = scale * sum_q table[q][codes[b][q][t]],
// and its gradient by sorted codes, without atomics on values:
// dtable[q][e] = scale * (sum of dout[b][t] over the (b, t) whose code q is e,
// in ascending order of b, t).
//
// The gradient sorts the rows of each codebook by code (a stable counting sort,
// by several blocks where there are many rows), then each entry's rows are
// gathered in order and the entry is written once, zeros included.  An entry that
// owns a large share of the rows (silence) is the sum of parts that others have
// summed.  Sums are FP32.

#include "fm_common.h"

namespace {

constexpr int HISTOGRAMS = 32768;  // of LDS, in counters: waves x entries at most

struct Embed {
  const int64_t* codes;
  const void* table;
  const void* dout;
  void *out, *dtable;
  int *order, *start;  // [Q][rows], [Q][entries + 1]
  int* counts;         // [Q][chunks][entries]: occurrences, where there are several chunks
  float* run;          // [Q][runs][2][D]: what each run holds of long entries
  long codes_batch, codes_book, ld_dout;
  long rows;
  int frames, books, entries, D, run_rows, runs, chunk_rows, chunks;
  FmDivisor by_frames;
  float scale;
};

// Work is cut into slices of 128 bytes of columns (8 lanes of 16 bytes), the
// slice being the fastest block index: blocks go to the eight XCDs in turn, so
// each XCD keeps to its own columns and its L2 holds what they are gathered from
// (a frame's entries by every codebook, an entry's frames) instead of an eighth
// of all of it.  64 x 125 frames x 32 codebooks of 2048 x 256 FP32, whole rows a
// wave against slices: forward 39 -> 30 us, gradient 64 -> 51 us.
constexpr int SLICE = 8;  // lanes

// SLICE lanes per output row and slice.  Code -1 is absent; any other code
// outside the table gives NaN.
template <typename T, int E>
__global__ __launch_bounds__(256) void embed_forward_kernel(Embed a) {
  typedef typename Vec<T, E>::type VT;
  const int n = a.D / E, c = blockIdx.x * SLICE + threadIdx.x % SLICE;
  const long row = (long)blockIdx.y * (256 / SLICE) + threadIdx.x / SLICE;
  if (row >= a.rows || c >= n) return;
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
  static_cast<VT*>(a.out)[row * n + c] = o;
}

// Row r's code of a book, or -1 where it names no entry.
FM_DEVICE int code_of(const Embed& a, int book, long row, long last) {
  if (row >= last) return -1;
  const int b = (int)fm_div((unsigned)row, a.by_frames);
  const int64_t c = a.codes[b * a.codes_batch + book * a.codes_book + (row - (long)b * a.frames)];
  return c >= 0 && c < a.entries ? (int)c : -1;
}

// How often each code occurs in a chunk of a book's rows.  Bound by latency, as the
// sort is: 64 x 125 frames x 32 codebooks, 4 us, the sort 13.
__global__ __launch_bounds__(1024) void embed_count_kernel(Embed a) {
  __shared__ int count[HISTOGRAMS];
  const int book = blockIdx.x, chunk = blockIdx.y;
  const long first = (long)chunk * a.chunk_rows, last = min(a.rows, first + a.chunk_rows);
  for (int e = threadIdx.x; e < a.entries; e += 1024) count[e] = 0;
  __syncthreads();
  for (long r = first; r < last; r += 4096) {
    int c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = code_of(a, book, r + 1024 * u + threadIdx.x, last);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c[u] >= 0) atomicAdd(&count[c[u]], 1);
  }
  __syncthreads();
  int* to = a.counts + ((long)book * a.chunks + chunk) * a.entries;
  for (int e = threadIdx.x; e < a.entries; e += 1024) to[e] = count[e];
}

// Stable counting sort of a chunk of a codebook's rows by code (all of them, or
// with the chunks' counts the chunk's own places).  The block's waves own
// consecutive shares of the rows and keep a histogram each (count[wave][e] in
// LDS); with the exclusive sums over (entry, chunk, wave) in its place, each wave
// walks its share 64 rows at a time, a row's place being its wave's next place
// of that entry plus the number of lower lanes with the same code.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void embed_sort_kernel(Embed a) {
  __shared__ int count[HISTOGRAMS];  // [WAVES][entries]
  __shared__ int totals[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, book = blockIdx.x, chunk = blockIdx.y;
  const long chunk_first = (long)chunk * a.chunk_rows, chunk_last = min(a.rows, chunk_first + a.chunk_rows);
  const long rows = chunk_last - chunk_first;
  // Shares of at least 128 rows: a histogram costs more than a few rows.
  const int share = max(128, ((int)((rows + WAVES - 1) / WAVES) + 63) & ~63);
  const int shares = (int)max(1l, (rows + share - 1) / share);
  const long first = chunk_first + (long)wave * share, last = min(chunk_last, first + share);
  for (int i = tid; i < shares * a.entries; i += 64 * WAVES) count[i] = 0;
  __syncthreads();
  int* mine = count + wave * a.entries;
  constexpr int AHEAD = 8;  // steps of 64 rows whose codes are in flight together
  for (long r = first; r < last; r += 64 * AHEAD) {
    int c[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) c[u] = code_of(a, book, r + 64 * u + lane, last);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (c[u] >= 0) atomicAdd(&mine[c[u]], 1);
  }
  __syncthreads();
  // Exclusive sums: each thread takes a run of entries, all chunks and waves of each.
  const int per = (a.entries + 64 * WAVES - 1) / (64 * WAVES);
  const int e0 = min(tid * per, a.entries), e1 = min(e0 + per, a.entries);
  const int* counts = a.counts + (long)book * a.chunks * a.entries;
  int sum = 0;
  for (int e = e0; e < e1; ++e)
    if (a.chunks > 1)
      for (int k = 0; k < a.chunks; ++k) sum += counts[k * a.entries + e];
    else
      for (int w = 0; w < shares; ++w) sum += count[w * a.entries + e];
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o, 64);
    if (lane >= o) upto += v;
  }
  if (lane == 63) totals[wave] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < wave; ++w) at += totals[w];
  int* start = a.start + (long)book * (a.entries + 1);
  if (chunk == 0 && tid == 64 * WAVES - 1) start[a.entries] = at + sum;
  for (int e = e0; e < e1; ++e) {
    if (chunk == 0) start[e] = at;
    int after = 0;
    if (a.chunks > 1)
      for (int k = 0; k < a.chunks; ++k) {
        const int v = counts[k * a.entries + e];
        if (k < chunk) at += v;
        else if (k > chunk) after += v;
      }
    for (int w = 0; w < shares; ++w) {
      const int v = count[w * a.entries + e];
      count[w * a.entries + e] = at;
      at += v;
    }
    at += after;
  }
  __syncthreads();
  int* order = a.order + (long)book * a.rows;
  int bits = 0;
  while ((1 << bits) < a.entries) ++bits;
  for (long r = first; r < last; r += 64 * AHEAD) {
    int c[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) c[u] = code_of(a, book, r + 64 * u + lane, last);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (r + 64 * u >= last) break;
      // Lanes with the same code (absent ones form a group that is dropped).
      unsigned long long same = __ballot(c[u] >= 0);
      same = c[u] >= 0 ? same : ~same;
      for (int k = 0; k < bits; ++k) {
        const unsigned long long set = __ballot((c[u] >> k) & 1);
        same &= (c[u] >> k) & 1 ? set : ~set;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1));
      if (c[u] >= 0) order[mine[c[u]] + rank] = (int)(r + 64 * u + lane);
      wave_lds_fence();
      if (c[u] >= 0 && rank == 0) mine[c[u]] += __popcll(same);
      wave_lds_fence();
    }
  }
}

// s += n sorted rows of dout in order, E columns a lane.  The next rows' places
// are read while these rows are on their way.
template <typename T, int E>
FM_DEVICE void gather(const Embed& a, const int* order, int n, int c, float (&s)[E]) {
  typedef typename Vec<T, E>::type VT;
  constexpr int AHEAD = 16;
  int next[AHEAD];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) next[u] = order[min(i + u, n - 1)];
  };
  if (n > 0) load(0);
  for (int i = 0; i < n; i += AHEAD) {
    VT v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      v[u] = VT{};
      if (i + u < n) v[u] = reinterpret_cast<const VT*>(static_cast<const T*>(a.dout) + (long)next[u] * a.ld_dout)[c];
    }
    if (i + AHEAD < n) load(i + AHEAD);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] += (float)v[u][e];
  }
}

// What run k, the sorted rows [k run_rows, (k + 1) run_rows), holds of entries
// with at least run_rows rows (which reach past a run on some side): of the one
// that its first row belongs to (part 0) and of one that begins in it and reaches
// its end (part 1).  A long entry is then the sum of its runs' parts, in order.
// 16 x 1500 frames x 8 codebooks of 1024 columns, bfloat16, a third of the frames
// with one code: 28 us, and 45 for the entries (393 MB gathered, 5.4 TB/s in all).
template <typename T, int E>
__global__ __launch_bounds__(256) void embed_run_kernel(Embed a) {
  const int c = blockIdx.x * SLICE + threadIdx.x % SLICE, book = blockIdx.z;
  const int run = blockIdx.y * (256 / SLICE) + threadIdx.x / SLICE;
  if (run >= a.runs || c >= a.D / E) return;
  const int* start = a.start + (long)book * (a.entries + 1);
  const int first = run * a.run_rows, last = min(first + a.run_rows, start[a.entries]);
  if (first >= last) return;
  const int* order = a.order + (long)book * a.rows;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const int lo = code_of(a, book, order[part ? last - 1 : first], a.rows);
    const int from = max(start[lo], first), to = min(start[lo + 1], last);
    if (start[lo + 1] - start[lo] < a.run_rows || (part && start[lo] <= first)) continue;
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
    gather<T, E>(a, order + from, to - from, c, s);
    float* out = a.run + (((long)book * a.runs + run) * 2 + part) * a.D + (long)c * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = s[e];
  }
}

// SLICE lanes per ENTRIES consecutive entries and slice.  Their sorted rows are
// one range, gathered with the next rows' places in flight: taken one entry at a
// time (four rows on average in the example above) each would wait for its start,
// its places and its rows in turn.  An entry of run_rows rows or more comes from its runs' parts.
template <typename T, int E, int ENTRIES>
__global__ __launch_bounds__(256) void embed_entry_kernel(Embed a) {
  typedef typename Vec<T, E>::type VT;
  const int n = a.D / E, c = blockIdx.x * SLICE + threadIdx.x % SLICE, book = blockIdx.z;
  int entry = (blockIdx.y * (256 / SLICE) + threadIdx.x / SLICE) * ENTRIES;
  if (entry >= a.entries || c >= n) return;
  const int end = min(entry + ENTRIES, a.entries);
  const int* start = a.start + (long)book * (a.entries + 1);
  const int* order = a.order + (long)book * a.rows;
  int bound[ENTRIES + 1];
#pragma unroll
  for (int u = 0; u <= ENTRIES; ++u) bound[u] = start[min(entry + u, end)];
  const int first = bound[0], last = bound[ENTRIES];
  float s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.0f;
  auto store = [&]() {
    VT o;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = (T)(s[e] * a.scale), s[e] = 0.0f;
    static_cast<VT*>(a.dtable)[((long)book * a.entries + entry) * n + c] = o;
  };
  constexpr int AHEAD = 8;
  if (a.runs && last - first >= a.run_rows) {
    for (; entry < end; ++entry) {
      const int lo = start[entry], hi = start[entry + 1];
      if (hi - lo < a.run_rows) {
        gather<T, E>(a, order + lo, hi - lo, c, s);
      } else {
        const int k0 = lo / a.run_rows, k1 = (hi - 1) / a.run_rows;
        const float* from = a.run + (long)book * a.runs * 2 * a.D + (long)c * E;
        for (int k = k0; k <= k1; k += AHEAD) {
          float v[AHEAD][E];
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) {
            const int at = 2 * min(k + u, k1) + (k + u == k0 && lo % a.run_rows ? 1 : 0);
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = k + u <= k1 ? from[(long)at * a.D + e] : 0.0f;
          }
#pragma unroll
          for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] += v[u][e];
        }
      }
      store();
    }
    return;
  }
  int next[AHEAD];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) next[u] = order[min(i + u, last - 1)];
  };
  if (first < last) load(first);
  for (int i = first; i < last; i += AHEAD) {
    VT v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      v[u] = VT{};
      if (i + u < last) v[u] = reinterpret_cast<const VT*>(static_cast<const T*>(a.dout) + (long)next[u] * a.ld_dout)[c];
    }
    if (i + AHEAD < last) load(i + AHEAD);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (i + u >= last) break;
      while (i + u >= bound[1]) {
        store();
        ++entry;
#pragma unroll
        for (int k = 1; k < ENTRIES; ++k) bound[k] = bound[k + 1];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] += (float)v[u][e];
    }
  }
  for (; entry < end; ++entry) store();
}

int embed_check(const Embed& a, int batch, int dtype) {
  if (batch < 0 || a.frames < 0 || a.books <= 0 || a.entries <= 0 || a.D <= 0 || dtype < DT_F32 || dtype > DT_F16 ||
      a.codes_batch < 0 || a.codes_book < 0 || a.ld_dout < 0 || !(a.scale == a.scale))
    return FM_BAD_ARGUMENT;
  // The grids' second and third dimensions hold 65535 blocks.
  if (a.rows > (256l / SLICE) * 65535 || a.entries > HISTOGRAMS || a.books > 65535) return FM_UNSUPPORTED;
  return FM_OK;
}

Embed embed_sizes(int batch, int books, int frames, int entries, int dim, float scale) {
  Embed a{};
  a.rows = (long)batch * frames;
  a.frames = frames, a.books = books, a.entries = entries, a.D = dim, a.scale = scale;
  a.by_frames = fm_divisor((unsigned)std::max(frames, 1));
  // Runs of at least sqrt(rows) / 2 rows: a code that owns every row is then at
  // most four times as many parts as a run has rows.
  const long rows = std::min(a.rows, 1l << 30);  // more are refused
  a.run_rows = 64;
  while (4l * a.run_rows * a.run_rows < rows) a.run_rows *= 2;
  a.runs = a.rows >= a.run_rows ? (int)((a.rows + a.run_rows - 1) / a.run_rows) : 0;
  // The sort's chunks: 4096 rows are a block's time; more than 16 would make
  // their counts the larger part.
  a.chunk_rows = 4096;
  while (16l * a.chunk_rows < rows) a.chunk_rows *= 2;
  a.chunks = (int)std::max<long>(1, (a.rows + a.chunk_rows - 1) / a.chunk_rows);
  return a;
}

struct Parts {
  size_t start, counts, run, total;  // byte offsets
};
Parts parts(const Embed& a) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  Parts p{};
  p.start = up((size_t)a.books * a.rows * sizeof(int));
  p.counts = p.start + up((size_t)a.books * (a.entries + 1) * sizeof(int));
  p.run = p.counts + (a.chunks > 1 ? up((size_t)a.books * a.chunks * a.entries * sizeof(int)) : 0);
  p.total = p.run + (size_t)a.books * a.runs * 2 * a.D * sizeof(float);
  return p;
}

bool aligned16(const Embed& a, int size) {
  uintptr_t u = 0;
  for (const void* p : {a.table, a.dout, (const void*)a.out, (const void*)a.dtable}) u |= reinterpret_cast<uintptr_t>(p);
  return (u & 15) == 0 && (a.D * size) % 16 == 0 && a.ld_dout * size % 16 == 0;
}

template <typename T, int E>
int embed_forward(const Embed& a, hipStream_t stream) {
  const dim3 grid(fm_ceil_div(a.D / E, SLICE), fm_ceil_div(a.rows, 256 / SLICE));
  hipLaunchKernelGGL((embed_forward_kernel<T, E>), grid, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int E>
int embed_backward(const Embed& a, hipStream_t stream) {
  const dim3 sort(a.books, a.chunks);
  if (a.chunks > 1) hipLaunchKernelGGL(embed_count_kernel, sort, dim3(1024), 0, stream, a);
  // As many waves as histograms fit.
  if (a.entries <= HISTOGRAMS / 16)
    hipLaunchKernelGGL(embed_sort_kernel<16>, sort, dim3(1024), 0, stream, a);
  else if (a.entries <= HISTOGRAMS / 4)
    hipLaunchKernelGGL(embed_sort_kernel<4>, sort, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(embed_sort_kernel<1>, sort, dim3(64), 0, stream, a);
  const unsigned slices = fm_ceil_div(a.D / E, SLICE), per = 256 / SLICE;
  if (a.runs)
    hipLaunchKernelGGL((embed_run_kernel<T, E>), dim3(slices, fm_ceil_div(a.runs, per), a.books), dim3(256), 0, stream, a);
  // One entry at a time where that alone does not fill the chip.  Gradients with one /
  // four, codes even and a third of them one, in us: 16384 units (4 x 512 entries of 256)
  // 20 / 33 and 33 / 40; 65536 (4 x 1024 of 512, 24000 rows) 45 / 49 and 58 / 69; 131072 (8
  // x 2048 of 256, 2000 rows) 23 / 22 and 33 / 33, 125 rows 18 / 16 and 21 / 22; 524288 (32
  // x 2048 of 256, 8000 rows) 59 / 53 and 81 / 78.
  if ((long)a.books * a.entries * slices >= 32768)
    hipLaunchKernelGGL((embed_entry_kernel<T, E, 4>), dim3(slices, fm_ceil_div(a.entries, 4 * per), a.books), dim3(256), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((embed_entry_kernel<T, E, 1>), dim3(slices, fm_ceil_div(a.entries, per), a.books), dim3(256), 0, stream,
                       a);
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
  a.counts = reinterpret_cast<int*>(ws + p.counts), a.run = reinterpret_cast<float*>(ws + p.run);
  return FM_EMBED_TYPES(embed_backward);
}

}  // extern "C"
