// Rows moved by key: the layout of routed rows sorted by expert, their way there and back (with weights), the rows of an
// embedding table and the table's gradient by sorted tokens.
//
// All of it is bound by memory: every kernel touches each row it needs once, in 16-byte vectors where rows allow it, a warp per part
// of a row or a block per token, sums in 32 bits in a fixed order (no floating-point atomics, so reruns give the same bits).
// Measured against a copy's 6.47 TB/s (bf16): 8192 tokens to 8 of 128 experts, width 2048, 56 us there (57 us of memory), 53 us back (47),
// 92 us for the gradients of rows and weights (98); 16384 tokens of a text from a table of 4096 columns 30 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "api.h"
#include "host_utils.h"

namespace rb {
namespace rows {

constexpr int kWarps = 32, kThreads = 32 * kWarps;      // of the sorting kernels
constexpr int kMaxBins = 2048;                          // 32 warps x 2048 counters of 16 bits: 128 KB of shared memory

// ----------------------------------------------------------------------------- elements
__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half down<__half>(float v) { return __float2half(v); }

// N consecutive elements: 16 bytes, or one element for rows of odd size or alignment (and eight floats: the sums of 16 bytes).
// 16-bit elements stay packed until they are used: unpacked, a vector takes twice the registers.
template <typename T, int N> struct alignas(N * sizeof(T)) Pack {
  T v[N];
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = up(v[i]);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = down<T>(f[i]);
  }
};
template <> struct alignas(16) Pack<__nv_bfloat16, 8> {
  uint32_t v[4];
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <> struct alignas(16) Pack<__half, 8> {
  uint32_t v[4];
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      f[2 * i] = h.x, f[2 * i + 1] = h.y;
    }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> zeros() {
  Pack<T, N> p;
  const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  p.set(z);
  return p;
}

// ----------------------------------------------------------------------------- stable counting sort
// One pass puts rows in the order of a key with few values ("bins"), rows of a bin in their old order.  In place_kernel every warp of
// a block has a run of rows and a counter per bin; 32 rows at a time find their equals, which gives their rank in the warp and
// moves the counter.  Counters of warps in front, and of blocks in front (count_kernel's), are added then.
// Up to kOneBlock rows take place_kernel alone.

constexpr int kOutside = 4;      // status word: an id lies outside a table that is whole
__device__ __forceinline__ void note_outside(int* err) {
  if (err != nullptr) *err = kOutside;      // (all that write it write the same)
}

struct ExpertKeys {      // expert ids; others than 0 .. bins - 1 live elsewhere and take no part (where nobody else has experts: noted)
  const void* ids;
  int wide, bins;
  int* err;
  __device__ __forceinline__ int digit(int i) const {
    const long long e = wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
    if (e >= 0 && e < bins) return static_cast<int>(e);
    note_outside(err);
    return -1;
  }
};
struct TokenKeys {      // first pass over token ids: a row's key is its table row, or `rows` (behind all) for tokens of other shards
  const void* ids;
  int wide, rows, shift, mask;
  long long start;
  __device__ __forceinline__ int key(int i) const {
    const long long a = (wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i]) - start;
    return a >= 0 && a < rows ? static_cast<int>(a) : rows;
  }
  __device__ __forceinline__ int pos(int i) const { return i; }
  __device__ __forceinline__ int digit(int i) const { return (key(i) >> shift) & mask; }
};
struct PairKeys {      // later passes over the sorted pairs of the pass in front
  const int2* pairs;
  int shift, mask;
  __device__ __forceinline__ int key(int i) const { return pairs[i].x; }
  __device__ __forceinline__ int pos(int i) const { return pairs[i].y; }
  __device__ __forceinline__ int digit(int i) const { return (key(i) >> shift) & mask; }
};

struct ExpertOut {
  int* dest;          // [n] buffer row of every routed row, -1: elsewhere
  int* source;        // [cap] routed row of every buffer row, -1: padding
  int* tile_expert;   // [cap / align] expert of every tile, -1: unused; null when align == 1
  int* bounds;        // [bins + 1] first buffer row of every expert
  int cap, tiles;
};
struct PairOut {
  int2* pairs;      // (key, row) in order
};

// What a launch fills beside the sort: `near` with -1 (entries that the sort fills in part: by the blocks that sort, before they do),
// and a share of `far` with zeros (a gradient that waits for the sorted rows: by blocks of its own on SMs that would be idle)
struct Fill {
  int* near;
  long long n_near;
  uint4* far;
  long long lo, hi;
  unsigned char* rest;      // the bytes behind the last whole vector
  int n_rest;
  int* counter;             // two counters set to zero, for a kernel behind the sort
};
__device__ __forceinline__ void fill_near(const Fill& f, int blocks) {
  const long long t = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x, all = static_cast<long long>(blocks) * kThreads;
  for (long long i = t; i < f.n_near; i += all) f.near[i] = -1;
}
constexpr int kFillRun = 8;      // vectors of a thread: a block fills 128 KB in one piece (6.9 TB/s; a stride of the whole grid: 5.1)
__device__ __forceinline__ void fill_far(const Fill& f, int blocks) {
  const long long b = blockIdx.x - blocks, v0 = f.lo + b * (kThreads * kFillRun) + threadIdx.x;
  const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < kFillRun; ++u)
    if (v0 + u * kThreads < f.hi) f.far[v0 + u * kThreads] = z;
  if (b == 0 && static_cast<int>(threadIdx.x) < f.n_rest) f.rest[threadIdx.x] = 0;
}

template <typename Src>
__global__ void __launch_bounds__(kThreads) count_kernel(Src src, int n, int chunk, int bins, int blocks, int* __restrict__ hist, Fill fill) {
  extern __shared__ int cnt[];
  if (static_cast<int>(blockIdx.x) >= blocks) return fill_far(fill, blocks);
  for (int b = threadIdx.x; b < bins; b += kThreads) cnt[b] = 0;
  fill_near(fill, blocks);
  __syncthreads();
  const int lo = blockIdx.x * chunk, hi = min(n, lo + chunk);
  for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
    const int d = src.digit(i);
    if (d >= 0) atomicAdd(&cnt[d], 1);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads) hist[static_cast<size_t>(blockIdx.x) * bins + b] = cnt[b];
}

// `sum` of all threads in front of this one, in `all` that of the block; `part`: kWarps ints of shared memory
__device__ __forceinline__ int scan_block(int sum, int* part, int* all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) part[w] = scan;
  __syncthreads();
  int mine = part[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, mine, o);
    if (lane >= o) mine += v;
  }
  *all = __shfl_sync(0xffffffffu, mine, 31);
  const int before = __shfl_sync(0xffffffffu, mine, (w + 31) & 31);
  return scan - sum + (w > 0 ? before : 0);
}
// The rank of this lane's digit among those of its warp so far; the warp's counters move on (digit -1: none).  (Equals found with a
// ballot per bit instead: as fast for a text, slower where most digits are equal.)
__device__ __forceinline__ int rank_in_warp(uint16_t* mine, int d) {
  const unsigned lane = threadIdx.x & 31, same = __match_any_sync(0xffffffffu, d);
  const int c = d >= 0 ? mine[d] : 0;
  __syncwarp();
  if (d >= 0 && static_cast<int>(lane) == __ffs(same) - 1) mine[d] = static_cast<uint16_t>(c + __popc(same));
  __syncwarp();
  return c + __popc(same & ((1u << lane) - 1));
}
// a bin's counters of `warps` warps become those of the warps in front; returns their sum
__device__ __forceinline__ int scan_warps(uint16_t* cnt, int bins, int b, int warps) {
  int run = 0;
#pragma unroll
  for (int k0 = 0; k0 < kWarps; k0 += 8) {
    if (k0 >= warps) break;
    int c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = k0 + k < warps ? cnt[(k0 + k) * bins + b] : 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k0 + k < warps) cnt[(k0 + k) * bins + b] = static_cast<uint16_t>(run);
      run += c[k];
    }
  }
  return run;
}

// kSteps x 1024 rows per block
template <typename Src, typename Out, int kSteps>
__global__ void __launch_bounds__(kThreads) place_kernel(Src src, Out out, int n, int bins, int align, int blocks, const int* __restrict__ hist, Fill fill) {
  constexpr bool kExperts = std::is_same<Out, ExpertOut>::value;
  extern __shared__ int sm[];
  __shared__ int part[kWarps];
  if (static_cast<int>(blockIdx.x) >= blocks) return fill_far(fill, blocks);
  const int t = threadIdx.x, w = t >> 5, lane = t & 31;
  constexpr int kPer = 32 * kSteps;      // rows of a warp
  const int first = blockIdx.x * (kSteps * kThreads), here = min(n - first, kSteps * kThreads), warps = (here + kPer - 1) / kPer;
  int* start = sm;                       // [bins] first output row of the bin (of this block's rows of it)
  int* total = sm + bins;                // [bins] rows of the bin
  int* first_row = total + bins;         // [bins] first output row of the bin
  uint16_t* cnt = reinterpret_cast<uint16_t*>(first_row + bins);      // [warps][bins]
  for (int i = t; i < warps * bins; i += kThreads) cnt[i] = 0;
  if (blockIdx.x == 0 && t == 0 && fill.counter != nullptr) fill.counter[0] = fill.counter[1] = 0;
  int at[kSteps];      // digits, then digits and ranks
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = first + w * kPer + s * 32 + lane;
    at[s] = i < n ? src.digit(i) : -1;
  }
  if (blocks == 1) fill_near(fill, 1);
  __syncthreads();
  uint16_t* mine = cnt + w * bins;
  if (w < warps) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int rank = rank_in_warp(mine, at[s]);
      at[s] = at[s] < 0 ? -1 : at[s] << 16 | rank;      // (ranks of a warp's 512 rows)
    }
  }
  __syncthreads();
  // first output row of every bin: running sum of the (padded) counts; a thread looks after a run of bins
  const int each = (bins + kThreads - 1) / kThreads, b0 = min(bins, t * each), b1 = min(bins, b0 + each);
  int sum = 0, end;
  for (int b = b0; b < b1; ++b) {
    int before = 0, all = 0;
    if (blocks > 1) {
#pragma unroll 16
      for (int k = 0; k < blocks; ++k) {
        const int h = hist[static_cast<size_t>(k) * bins + b];
        all += h;
        before += k < static_cast<int>(blockIdx.x) ? h : 0;
      }
    }
    const int own = scan_warps(cnt, bins, b, warps);
    start[b] = before;
    total[b] = blocks > 1 ? all : own;
    sum += (total[b] + align - 1) / align * align;
  }
  int base = scan_block(sum, part, &end);
  for (int b = b0; b < b1; ++b) {
    const int rows = (total[b] + align - 1) / align * align;
    if constexpr (kExperts) {
      if (b % blocks == static_cast<int>(blockIdx.x)) out.bounds[b] = base;      // (every block knows all bounds)
      if (b == bins - 1 && blockIdx.x == 0) out.bounds[bins] = end;
      first_row[b] = base;
    }
    start[b] += base;
    base += rows;
  }
  __syncthreads();
  if constexpr (kExperts) {
    for (int q = blockIdx.x * kThreads + t; q < out.tiles; q += blocks * kThreads) {      // the last expert that begins at or in front of the tile
      int b = 0;
      for (int step = 1 << (31 - __clz(bins)); step > 0; step >>= 1)
        if (b + step < bins && first_row[b + step] <= q * align) b += step;
      out.tile_expert[q] = q * align < end && q * align < first_row[b] + (total[b] + align - 1) / align * align ? b : -1;
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = first + w * kPer + s * 32 + lane;
    if (i >= n) break;
    const int d = at[s] >> 16, to = at[s] < 0 ? -1 : start[d] + mine[d] + (at[s] & 0xffff);
    if constexpr (kExperts) {
      out.dest[i] = to;
      if (to >= 0) out.source[to] = i;
    } else {
      out.pairs[to] = make_int2(src.key(i), src.pos(i));
    }
  }
}

// Tokens sorted by table row in one launch: (key, position) in 32 bits, all passes in the shared memory of one block, the other blocks
// fill the gradient meanwhile (16384 tokens of a text 45 us, hidden behind a fill of 1.2 GB that takes 166 us; 300 tokens 4 us).
template <int kSteps>
__global__ void __launch_bounds__(kThreads) pack_sort_kernel(TokenKeys src, int2* __restrict__ pairs, int n, int pos_bits, int passes, int each, Fill fill) {
  extern __shared__ int sm[];
  __shared__ int part[kWarps];
  if (blockIdx.x > 0) return fill_far(fill, 1);
  const int t = threadIdx.x, w = t >> 5, lane = t & 31, bins = 1 << each;
  constexpr int kPer = 32 * kSteps;
  const int warps = (n + kPer - 1) / kPer;
  unsigned* a = reinterpret_cast<unsigned*>(sm);                       // [n] (between two barriers all of them are in registers)
  int* start = sm + n;                                                 // [bins]
  uint16_t* cnt = reinterpret_cast<uint16_t*>(start + bins);           // [warps][bins]
  if (t == 0) fill.counter[0] = fill.counter[1] = 0;
  unsigned v[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = w * kPer + s * 32 + lane;
    v[s] = i < n ? static_cast<unsigned>(src.key(i)) << pos_bits | i : 0;
  }
  uint16_t* mine = cnt + w * bins;
  for (int p = 0; p < passes; ++p) {
    const int shift = pos_bits + p * each;
    for (int i = t; i < warps * bins; i += kThreads) cnt[i] = 0;
    if (p > 0) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int i = w * kPer + s * 32 + lane;
        v[s] = i < n ? a[i] : 0;
      }
    }
    __syncthreads();
    int rank[kSteps];
    if (w < warps) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int i = w * kPer + s * 32 + lane;
        rank[s] = rank_in_warp(mine, i < n ? static_cast<int>(v[s] >> shift) & (bins - 1) : -1);
      }
    }
    __syncthreads();
    const int own = t < bins ? scan_warps(cnt, bins, t, warps) : 0;      // (bins <= threads)
    int end;
    const int base = scan_block(own, part, &end);
    if (t < bins) start[t] = base;
    __syncthreads();
    if (w < warps) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int i = w * kPer + s * 32 + lane;
        if (i >= n) break;
        const int d = static_cast<int>(v[s] >> shift) & (bins - 1);
        a[start[d] + mine[d] + rank[s]] = v[s];
      }
    }
    __syncthreads();
  }
  for (int i = t; i < n; i += kThreads) pairs[i] = make_int2(static_cast<int>(a[i] >> pos_bits), static_cast<int>(a[i] & ((1u << pos_bits) - 1)));
}

constexpr size_t kMostSmem = 220 * 1024;
constexpr int kMaxSort = 1 << 30;      // rows and keys of a sort (places are 32-bit)
constexpr int kMostSteps = 16;         // counters of a warp's rows have 16 bits, and so have all of a block's
constexpr int kOneBlock = 4096;        // rows that one block sorts by itself (9003 rows: 18 us, in nine blocks after a count 9 us)
constexpr int kPackSort = 16384;       // ... and that pack_sort_kernel takes, where a key and a position fit 32 bits
// 1024-row steps of a block: enough blocks to spread the work, few enough that reading all their counts is cheap
inline int sort_steps(long long n) {
  const long long want = n <= kOneBlock ? (n + kThreads - 1) / kThreads : (n + 64ll * kThreads - 1) / (64ll * kThreads);
  return want <= 1 ? 1 : want <= 2 ? 2 : want <= 4 ? 4 : want <= 8 ? 8 : kMostSteps;
}
inline int sort_blocks(long long n) {
  const long long c = static_cast<long long>(sort_steps(n)) * kThreads;
  return n <= 0 ? 1 : static_cast<int>((n + c - 1) / c);
}
inline int fill_blocks(const Fill& f, long long vectors) {
  return f.far == nullptr ? 0 : static_cast<int>((vectors + kThreads * kFillRun - 1) / (kThreads * kFillRun)) + 1;
}
// Always the same limit: calls of several threads would lower one another's otherwise.
template <typename K>
int allow_smem(K kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return 0;
  return bytes > kMostSmem ? -4 : static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem)));
}

template <int kSteps, typename Src, typename Out>
int place(const Src& src, const Out& out, int n, int bins, int align, int blocks, int more, const int* hist, const Fill& fill, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(bins) * (12 + 2 * kWarps);
  const int rc = allow_smem(place_kernel<Src, Out, kSteps>, smem);
  if (rc) return rc;
  place_kernel<Src, Out, kSteps><<<blocks + more, kThreads, smem, st>>>(src, out, n, bins, align, blocks, hist, fill);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}

// `launches` of the whole sort share the far fill evenly; `at` counts them
template <typename Src, typename Out>
int sort_pass(const Src& src, const Out& out, int n, int bins, int align, int* hist, const Fill& fill, int launches, int* at, cudaStream_t st) {
  const int nb = sort_blocks(n), steps = sort_steps(n);
  const long long vectors = fill.hi;
  auto share = [&]() {
    Fill f = fill;
    f.lo = vectors * *at / launches;
    f.hi = vectors * (*at + 1) / launches;
    if (*at > 0) f.n_rest = 0;
    ++*at;
    return f;
  };
  if (nb > 1) {
    const Fill f = share();
    count_kernel<Src><<<nb + fill_blocks(f, f.hi - f.lo), kThreads, bins * sizeof(int), st>>>(src, n, steps * kThreads, bins, nb, hist, f);
    rb_note_launch(1);
  }
  const Fill f = share();
  const int more = fill_blocks(f, f.hi - f.lo);
  switch (steps) {
    case 1: return place<1>(src, out, n, bins, align, nb, more, hist, f, st);
    case 2: return place<2>(src, out, n, bins, align, nb, more, hist, f, st);
    case 4: return place<4>(src, out, n, bins, align, nb, more, hist, f, st);
    case 8: return place<8>(src, out, n, bins, align, nb, more, hist, f, st);
    default: return place<kMostSteps>(src, out, n, bins, align, nb, more, hist, f, st);
  }
}

template <int kSteps>
int pack_sort_t(const TokenKeys& src, int2* pairs, int n, int pos_bits, int passes, int each, const Fill& fill, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(n) * 4 + (size_t{1} << each) * (4 + 2 * kWarps);
  const int rc = allow_smem(pack_sort_kernel<kSteps>, smem);
  if (rc) return rc;
  pack_sort_kernel<kSteps><<<1 + fill_blocks(fill, fill.hi), kThreads, smem, st>>>(src, pairs, n, pos_bits, passes, each, fill);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}
int pack_sort(const TokenKeys& src, int2* pairs, int n, int pos_bits, int passes, int each, const Fill& fill, cudaStream_t st) {
  if (n <= 1 * kThreads) return pack_sort_t<1>(src, pairs, n, pos_bits, passes, each, fill, st);
  if (n <= 4 * kThreads) return pack_sort_t<4>(src, pairs, n, pos_bits, passes, each, fill, st);
  if (n <= 8 * kThreads) return pack_sort_t<8>(src, pairs, n, pos_bits, passes, each, fill, st);
  return pack_sort_t<16>(src, pairs, n, pos_bits, passes, each, fill, st);
}

// ----------------------------------------------------------------------------- copies of rows
struct SourceRow {      // buffer row r <- row source[r] / k of the input
  const int* source;
  int k;
  __device__ __forceinline__ long long row(long long r) const {
    const int s = source[r];
    return s < 0 ? -1 : s / k;
  }
};
struct TokenRow {      // row r <- table row of its token
  const void* ids;
  int wide, rows;
  long long start;
  int* err;
  __device__ __forceinline__ long long row(long long r) const {
    const long long a = (wide ? static_cast<const long long*>(ids)[r] : static_cast<const int*>(ids)[r]) - start;
    if (a >= 0 && a < rows) return a;
    note_outside(err);
    return -1;
  }
};

template <int N> constexpr int kMove = N == 1 ? 8 : 4;      // vectors of a lane in flight
// A vector that leaves the L2 first: what is read again and again (a token's row by its experts) stays there meanwhile.
template <typename T, int N>
__device__ __forceinline__ void put_away(Pack<T, N>* o, const Pack<T, N>& p) {
  if constexpr (sizeof(p) == 16) __stcs(reinterpret_cast<uint4*>(o), *reinterpret_cast<const uint4*>(&p));
  else *o = p;
}
// out[r] = scale * in[row(r)], zeros where there is no such row; a warp takes 32 x kMove vectors of a row
template <typename T, int N, bool kScale, typename Row>
__global__ void __launch_bounds__(256) move_kernel(const T* __restrict__ in, long long ld, Row src, T* __restrict__ out, long long n, int cols, int parts,
                                                   float scale) {
  const long long unit = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const long long r = unit / parts;
  if (r >= n) return;
  const int lane = threadIdx.x & 31, vecs = cols / N;
  const int v0 = static_cast<int>(unit - r * parts) * (32 * kMove<N>) + lane;
  const long long s = src.row(r);
  const Pack<T, N>* a = reinterpret_cast<const Pack<T, N>*>(in + (s < 0 ? 0 : s) * ld);
  Pack<T, N>* o = reinterpret_cast<Pack<T, N>*>(out + r * cols);
  Pack<T, N> p[kMove<N>];
#pragma unroll
  for (int u = 0; u < kMove<N>; ++u) {
    const int v = v0 + u * 32;
    p[u] = zeros<T, N>();
    if (s >= 0 && v < vecs) p[u] = a[v];
  }
#pragma unroll
  for (int u = 0; u < kMove<N>; ++u) {
    const int v = v0 + u * 32;
    if (v >= vecs) break;
    if constexpr (kScale) {
      float f[N];
      p[u].get(f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= scale;
      p[u].set(f);
    }
    put_away(o + v, p[u]);
  }
}

// The same for rows that would leave many of those lanes idle: vectors of the output one after the other, over the ends of rows.
template <typename T, int N, bool kScale, typename Row>
__global__ void __launch_bounds__(256) move_flat_kernel(const T* __restrict__ in, long long ld, Row src, T* __restrict__ out, unsigned all, unsigned vecs,
                                                        float scale) {
  const unsigned q0 = (blockIdx.x * 8u + (threadIdx.x >> 5)) * (32 * kMove<N>) + (threadIdx.x & 31);
  Pack<T, N> p[kMove<N>];
#pragma unroll
  for (int u = 0; u < kMove<N>; ++u) {
    const unsigned q = q0 + u * 32, r = q / vecs;
    p[u] = zeros<T, N>();
    if (q >= all) break;
    const long long s = src.row(r);
    if (s >= 0) p[u] = reinterpret_cast<const Pack<T, N>*>(in + s * ld)[q - r * vecs];
  }
#pragma unroll
  for (int u = 0; u < kMove<N>; ++u) {
    const unsigned q = q0 + u * 32;
    if (q >= all) break;
    if constexpr (kScale) {
      float f[N];
      p[u].get(f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= scale;
      p[u].set(f);
    }
    put_away(reinterpret_cast<Pack<T, N>*>(out) + q, p[u]);
  }
}

// out[dest[t, j]] = in[t]: a warp reads its part of a row once and puts it down wherever it goes; warps behind the rows write the zeros of padding.
template <typename T, int N>
__global__ void __launch_bounds__(256) spread_kernel(const T* __restrict__ in, long long ld, const int* __restrict__ source, const int* __restrict__ dest,
                                                     T* __restrict__ out, long long cap, long long n, int k, int cols, int parts) {
  const long long unit = blockIdx.x * 8ll + (threadIdx.x >> 5), empty_unit = unit - n * parts;
  const int lane = threadIdx.x & 31, vecs = cols / N;
  Pack<T, N> p[kMove<N>];
  if (empty_unit >= 0) {      // a part of 32 rows far from one another: padding rows lie together
    const long long units = (cap + 31) / 32, e = empty_unit / parts, r = e + lane * units;
    const int v0 = static_cast<int>(empty_unit - e * parts) * (32 * kMove<N>) + lane;
    unsigned empty = __ballot_sync(0xffffffffu, e < units && r < cap && source[r < cap ? r : 0] < 0);
    for (; empty; empty &= empty - 1) {
      Pack<T, N>* o = reinterpret_cast<Pack<T, N>*>(out + (e + (__ffs(empty) - 1) * units) * cols);
#pragma unroll
      for (int u = 0; u < kMove<N>; ++u)
        if (v0 + u * 32 < vecs) put_away(o + v0 + u * 32, zeros<T, N>());
    }
    return;
  }
  const long long row = unit / parts;
  const int v0 = static_cast<int>(unit - row * parts) * (32 * kMove<N>) + lane;
  const Pack<T, N>* a = reinterpret_cast<const Pack<T, N>*>(in + row * ld);
#pragma unroll
  for (int u = 0; u < kMove<N>; ++u)
    if (v0 + u * 32 < vecs) p[u] = a[v0 + u * 32];
  for (int j0 = 0; j0 < k; j0 += 32) {
    const int mine = j0 + lane < k ? dest[row * k + j0 + lane] : -1;
    for (int j = 0; j < 32 && j0 + j < k; ++j) {
      const long long d = __shfl_sync(0xffffffffu, mine, j);
      if (d < 0) continue;
      Pack<T, N>* o = reinterpret_cast<Pack<T, N>*>(out + d * cols);
#pragma unroll
      for (int u = 0; u < kMove<N>; ++u)
        if (v0 + u * 32 < vecs) put_away(o + v0 + u * 32, p[u]);
    }
  }
}

constexpr int kSingleThreads = 128;      // of a block that works on a row of single elements
// out[t] = sum_j w[t, j] in[dest[t, j]] in 32 bits, j ascending.  A block per token: its places are read once, and the rows that follow
// from them in vectors of all threads, eight rows in flight (single elements: four rows, four elements of a thread).  Measured for
// 65536 rows of 4 KB, 47 us of memory: 54 us; a warp per part of a row, which waits for its places as long as for the rows, 61 us; blocks
// that fetch the places of their next token meanwhile, but wait for one another between tokens, 63 us.
template <typename T, int N, bool kWeight, typename OutT>
__global__ void __launch_bounds__(N == 1 ? kSingleThreads : 256) sum_kernel(const T* __restrict__ in, long long ld, const int* __restrict__ dest, const float* __restrict__ weight,
                                                  OutT* __restrict__ out, int k, int cols) {
  const long long row = blockIdx.x;
  constexpr int S = N == 1 ? 4 : 1, J = N == 1 ? 4 : 8;      // vectors of a thread at a time, rows in flight
  const int vecs = cols / N, step = N == 1 ? kSingleThreads : blockDim.x;
  for (int v = threadIdx.x; v < vecs; v += S * step) {
    float acc[S][N];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[s][i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += J) {
      int d[J];
      float w[J];
      Pack<T, N> p[J][S];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        d[j] = j0 + j < k ? dest[row * k + j0 + j] : -1;
        w[j] = kWeight && d[j] >= 0 ? weight[row * k + j0 + j] : 1.f;
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (d[j] >= 0 && v + s * step < vecs) p[j][s] = reinterpret_cast<const Pack<T, N>*>(in + d[j] * ld)[v + s * step];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (d[j] >= 0 && v + s * step < vecs) {
            float f[N];
            p[j][s].get(f);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[s][i] = kWeight ? fmaf(w[j], f[i], acc[s][i]) : acc[s][i] + f[i];
          }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (v + s * step >= vecs) break;
      Pack<OutT, N> o;
      o.set(acc[s]);
      reinterpret_cast<Pack<OutT, N>*>(out + row * cols)[v + s * step] = o;
    }
  }
}

// buffer rows that a warp looks at for padding: long ones take their time, short ones would be more warps than tokens
__host__ __device__ inline int padding_rows(int vecs) { return vecs >= 128 ? 8 : 32; }

// Backward of the weighted sum: d_y[dest] = w d_out[t] and d_w = <d_out[t], y[dest]>.  A block per token holds its row of d_out (in the
// type of the sum: fp32 for a sum kept in 32 bits) while it walks over the token's rows of y, so that all of them pass once; blocks behind
// the tokens write the zeros of padding rows.  Where rows do not learn (kRows false) nothing is written to the buffer, where weights are
// fixed (kWeights false) y is not read, and need not be there.  (Null pointers asked about in here, 8192
// tokens to 8 of 128 experts, width 2048, cold L2: 125 us instead of 104.)
template <typename T, int N, typename G, bool kRows, bool kWeights>
__global__ void __launch_bounds__(N == 1 ? kSingleThreads : 256) sum_bwd_kernel(const G* __restrict__ d_out, long long ld, const T* __restrict__ y, long long ldy,
                                                      const int* __restrict__ source, const int* __restrict__ dest, const float* __restrict__ weight,
                                                      T* __restrict__ d_y, float* __restrict__ d_w, long long cap, long long n, int k, int cols) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, warps = blockDim.x >> 5, vecs = cols / N;
  const long long row = blockIdx.x;
  if (row >= n) {      // a warp looks at some rows far from one another: padding rows lie together
    const int some = padding_rows(vecs);
    const long long units = (cap + some - 1) / some, unit = (row - n) * warps + w, r = unit + lane * units;
    unsigned empty = __ballot_sync(0xffffffffu, lane < some && unit < units && r < cap && source[r < cap ? r : 0] < 0);
    const Pack<T, N> z = zeros<T, N>();
    for (; empty; empty &= empty - 1) {
      Pack<T, N>* o = reinterpret_cast<Pack<T, N>*>(d_y + (unit + (__ffs(empty) - 1) * units) * cols);
      for (int v = lane; v < vecs; v += 32) o[v] = z;
    }
    return;
  }
  __shared__ float red[8][8];
  constexpr int J = 8;      // rows of y at a time, four of them in flight
  const Pack<G, N>* a = reinterpret_cast<const Pack<G, N>*>(d_out + row * ld);
  for (int j0 = 0; j0 < k; j0 += J) {
    int d[J];
    float wj[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      d[j] = j0 + j < k ? dest[row * k + j0 + j] : -1;
      wj[j] = d[j] >= 0 ? weight[row * k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    if constexpr (N == 1) {      // four elements of a thread at a time, four rows in flight
      constexpr int S = 4;
      for (int v = t; v < vecs; v += S * kSingleThreads) {
        float f[S];
        const G* av = d_out + row * ld + v;
#pragma unroll
        for (int s = 0; s < S; ++s) f[s] = v + s * kSingleThreads < vecs ? up(av[s * kSingleThreads]) : 0.f;
#pragma unroll
        for (int h = 0; h < J; h += 4) {
          if (j0 + h >= k) continue;
          T q[4][S];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const T* b = y + (d[h + j] < 0 ? 0 : d[h + j]) * ldy + v;
#pragma unroll
            for (int s = 0; s < S; ++s)
              if (kWeights && d[h + j] >= 0 && v + s * kSingleThreads < vecs) q[j][s] = b[s * kSingleThreads];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            T* o = d_y + static_cast<long long>(d[h + j] < 0 ? 0 : d[h + j]) * cols + v;
#pragma unroll
            for (int s = 0; s < S; ++s)
              if (d[h + j] >= 0 && v + s * kSingleThreads < vecs) {
                if (kWeights) dot[h + j] = fmaf(f[s], up(q[j][s]), dot[h + j]);
                if (kRows) o[s * kSingleThreads] = down<T>(f[s] * wj[h + j]);
              }
          }
        }
      }
    } else {
      for (int v = t; v < vecs; v += blockDim.x) {
        float f[N];
        a[v].get(f);
#pragma unroll
        for (int h = 0; h < J; h += 4) {
          Pack<T, N> q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (kWeights && d[h + j] >= 0) q[j] = reinterpret_cast<const Pack<T, N>*>(y + d[h + j] * ldy)[v];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d[h + j] >= 0) {
              float b[N];
              if constexpr (kWeights) {
                q[j].get(b);
#pragma unroll
                for (int i = 0; i < N; ++i) dot[h + j] = fmaf(f[i], b[i], dot[h + j]);
              }
              if constexpr (kRows) {
                Pack<T, N> o;
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = f[i] * wj[h + j];
                o.set(b);
                reinterpret_cast<Pack<T, N>*>(d_y + static_cast<long long>(d[h + j]) * cols)[v] = o;
              }
            }
        }
      }
    }
    if constexpr (!kWeights) continue;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
    }
    if (j0 > 0) __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < J; ++j) red[w][j] = dot[j];
    }
    __syncthreads();
    if (t < J && j0 + t < k) {
      float s = red[0][t];
      for (int i = 1; i < warps; ++i) s += red[i][t];
      d_w[row * k + j0 + t] = s;
    }
  }
}

// ----------------------------------------------------------------------------- gradient of a table by sorted rows
// `pairs` holds (table row, input row) in order.  A warp walks 32 of them for 32 vectors of columns and keeps one running sum; a run
// of equal keys that ends inside goes out at once, one that goes on in the next 32 (or came from those in front) leaves a partial
// sum, and merge_kernel adds those of a run.  16384 tokens of a text (7100 different ones), 4096 columns in bf16: 39 us for 30 us of
// memory and 9 us for the merge; added to fp32 rows 69 us for 57 (all different: 116 for 104; by `red` of four 72 and 135).
constexpr int kRun = 32, kLongRun = 16;

template <typename OutT, int N, bool kAdd>
__device__ __forceinline__ void put_sum(OutT* out, long long row, int cols, int v, const float* acc, float scale) {
  if constexpr (kAdd && N % 4 == 0) {      // (rows of 16-byte vectors)
    float4* o = reinterpret_cast<float4*>(out + row * cols + v * N);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      float4 f = o[i];
      f.x += acc[4 * i] * scale;
      f.y += acc[4 * i + 1] * scale;
      f.z += acc[4 * i + 2] * scale;
      f.w += acc[4 * i + 3] * scale;
      o[i] = f;
    }
  } else if constexpr (kAdd) {
    out[row * cols + v] += acc[0] * scale;
  } else {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = acc[i] * scale;
    Pack<OutT, N> p;
    p.set(f);
    reinterpret_cast<Pack<OutT, N>*>(out + row * cols)[v] = p;
  }
}

template <typename T, int N, typename OutT, bool kAdd>
__global__ void __launch_bounds__(256) run_kernel(const T* __restrict__ dy, long long ld, const int2* __restrict__ pairs, OutT* __restrict__ out,
                                                  float* __restrict__ part, int* __restrict__ open, int n, int rows, int cols, int parts, float scale) {
  const long long unit = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int c = static_cast<int>(unit / parts);
  if (static_cast<long long>(c) * kRun >= n) return;
  const int lane = threadIdx.x & 31;
  const int v = static_cast<int>(unit - static_cast<long long>(c) * parts) * 32 + lane;
  const bool there = v < cols / N;
  const int i0 = c * kRun;
  const int2 pr = i0 + lane < n ? pairs[i0 + lane] : make_int2(rows, 0);
  const int prev = i0 > 0 ? pairs[i0 - 1].x : -1, next = i0 + kRun < n ? pairs[i0 + kRun].x : rows;
  int after = __shfl_down_sync(0xffffffffu, pr.x, 1);
  if (lane == 31) after = next;
  const int m = __popc(__ballot_sync(0xffffffffu, pr.x < rows));                          // keys behind the table's rows stand last
  const unsigned ends = __ballot_sync(0xffffffffu, pr.x != after) | 1u << 31;             // a run ends here, or at least its part in this chunk
  const bool from_front = __shfl_sync(0xffffffffu, pr.x, 0) == prev, goes_on = __shfl_sync(0xffffffffu, pr.x, 31) == next;
  const bool copies = std::is_same<T, OutT>::value && !kAdd && scale == 1.f;              // runs of one row go out as they are
  if (lane == 0 && unit == static_cast<long long>(c) * parts && m == kRun && goes_on && !(from_front && ends == 1u << 31)) {
    // a run that begins here goes on
    const long long far = (static_cast<long long>(c) + kLongRun) * kRun, chunks = (static_cast<long long>(n) + kRun - 1) / kRun;
    if (far < n && pairs[far].x == next) open[1 + chunks - atomicAdd(open + 1, 1)] = c;
    else open[2 + atomicAdd(open, 1)] = c;
  }
  float acc[N];
  bool fresh = true, head = true;      // nothing in `acc`; no run has ended in here yet
  constexpr int U = 8;
  for (int j0 = 0; j0 < m; j0 += U) {
    Pack<T, N> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long pos = __shfl_sync(0xffffffffu, pr.y, j0 + u);
      if (j0 + u < m && there) p[u] = reinterpret_cast<const Pack<T, N>*>(dy + pos * ld)[v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j >= m) break;
      const bool end = (ends >> j) & 1, before = head && from_front, behind = j == kRun - 1 && goes_on;
      const bool whole = end && !before && !behind;
      const long long key = __shfl_sync(0xffffffffu, pr.x, j);
      if (copies && whole && fresh) {
        if constexpr (std::is_same<T, OutT>::value) {
          if (there) reinterpret_cast<Pack<T, N>*>(out + key * cols)[v] = p[u];
        }
        head = false;
        continue;
      }
      float f[N];
      p[u].get(f);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = fresh ? f[i] : acc[i] + f[i];
      fresh = end;
      if (!end) continue;
      head = false;
      if (!there) continue;
      if (whole) put_sum<OutT, N, kAdd>(out, key, cols, v, acc, scale);
      else {
        Pack<float, N> q;
        q.set(acc);
        *reinterpret_cast<Pack<float, N>*>(part + (static_cast<long long>(c) * 2 + (before ? 0 : 1)) * cols + v * N) = q;
      }
    }
  }
}

// acc += the partial sums d0 .. d1 - 1 of a run that begins in chunk c: the end of that chunk, the beginnings of the others
template <int N>
__device__ __forceinline__ void add_parts(const float* __restrict__ part, long long c, long long d0, long long d1, int cols, int v, float* acc) {
  for (long long d = d0; d < d1; d += 8) {
    Pack<float, N> p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (d + u < d1) p[u] = *reinterpret_cast<const Pack<float, N>*>(part + ((d + u) * 2 + (d + u == c)) * cols + v * N);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (d + u < d1) {
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += p[u].v[i];
      }
  }
}

// the chunk behind the last of a run that begins in chunk c: 32 chunks side by side, then 32 at equal distances in what is left
__device__ __forceinline__ long long run_end(const int2* __restrict__ pairs, int key, long long c, long long chunks) {
  long long lo = c + 1, hi = chunks, step = 1;      // chunk lo begins with this key, chunk hi does not
  for (;;) {
    const long long x = lo + (threadIdx.x & 31) * step;
    const int yes = __popc(__ballot_sync(0xffffffffu, x < hi && pairs[(x < hi ? x : lo) * kRun].x == key));
    const long long next = lo + yes * step;
    if (yes < 32 && next < hi) hi = next;
    lo += (yes - 1) * step;
    if (hi - lo <= 1) return hi;
    step = (hi - lo + 31) / 32;
  }
}

// Runs over several chunks; `open`: the number of those of up to kLongRun more chunks and of the others, then the chunks where they
// begin, from the front and from the back, in no order.  A warp takes a part of the columns of a short run; of a long one a block
// does, every warp a stretch, and the stretches are added from left to right.
template <int N, typename OutT, bool kAdd>
__global__ void __launch_bounds__(256) merge_kernel(const int2* __restrict__ pairs, const float* __restrict__ part, const int* __restrict__ open,
                                                    OutT* __restrict__ out, int n, int cols, int parts, float scale) {
  __shared__ Pack<float, N> sums[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long chunks = (static_cast<long long>(n) + kRun - 1) / kRun, items = static_cast<long long>(open[0]) * parts;
  float acc[N];
  for (long long item = blockIdx.x * 8ll + w; item < items; item += gridDim.x * 8ll) {
    const long long c = open[2 + item / parts];
    const int key = pairs[c * kRun + kRun - 1].x, v = static_cast<int>(item % parts) * 32 + lane;
    const long long hi = run_end(pairs, key, c, chunks);
    if (v >= cols / N) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    add_parts<N>(part, c, c, hi, cols, v, acc);
    put_sum<OutT, N, kAdd>(out, key, cols, v, acc, scale);
  }
  const long long longs = static_cast<long long>(open[1]) * parts;
  for (long long item = gridDim.x - 1 - blockIdx.x; item < longs; item += gridDim.x) {      // (the last blocks have the fewest short ones)
    const long long c = open[1 + chunks - item / parts];
    const int key = pairs[c * kRun + kRun - 1].x, v = static_cast<int>(item % parts) * 32 + lane;
    const bool there = v < cols / N;
    const long long hi = run_end(pairs, key, c, chunks), each = (hi - c + 7) / 8, d0 = c + w * each, d1 = d0 + each < hi ? d0 + each : hi;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    if (there) add_parts<N>(part, c, d0, d1, cols, v, acc);
    sums[w][lane].set(acc);
    __syncthreads();
    if (w == 0 && there) {
#pragma unroll
      for (int j = 1; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += sums[j][lane].v[i];
      put_sum<OutT, N, kAdd>(out, key, cols, v, acc, scale);
    }
    __syncthreads();
  }
}

// ----------------------------------------------------------------------------- host
inline bool wide_rows(const void* p, long long ld, int cols, int size) {      // rows that split into aligned 16-byte vectors
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * size) % 16 == 0 && (static_cast<long long>(cols) * size) % 16 == 0;
}
inline long long grid_of(long long units) { return (units + 7) / 8; }
constexpr long long kMaxGrid = 2147483647ll;

template <typename T, typename Row>
int move_t(const void* in, long long ld, const Row& src, void* out, long long n, int cols, float scale, cudaStream_t st) {
  constexpr int NV = 16 / sizeof(T);
  const bool wide = wide_rows(in, ld, cols, sizeof(T)) && wide_rows(out, cols, cols, sizeof(T));
  const int per = wide ? 32 * kMove<NV> * NV : 32 * kMove<1>, parts = (cols + per - 1) / per;
  const long long grid = grid_of(n * parts);
  if (grid > kMaxGrid) return -3;
  const T* a = static_cast<const T*>(in);
  T* o = static_cast<T*>(out);
  const int g = static_cast<int>(grid);
  const long long vecs = cols / NV, all = n * vecs;
  if (wide && parts * 128ll * 8 > vecs * 9 && all < 1ll << 31) {
    const int blocks = static_cast<int>((all + 8 * 32 * kMove<NV> - 1) / (8 * 32 * kMove<NV>));
    if (scale == 1.f) move_flat_kernel<T, NV, false><<<blocks, 256, 0, st>>>(a, ld, src, o, static_cast<unsigned>(all), static_cast<unsigned>(vecs), scale);
    else move_flat_kernel<T, NV, true><<<blocks, 256, 0, st>>>(a, ld, src, o, static_cast<unsigned>(all), static_cast<unsigned>(vecs), scale);
  } else if (wide && scale == 1.f) move_kernel<T, NV, false><<<g, 256, 0, st>>>(a, ld, src, o, n, cols, parts, scale);
  else if (wide) move_kernel<T, NV, true><<<g, 256, 0, st>>>(a, ld, src, o, n, cols, parts, scale);
  else if (scale == 1.f) move_kernel<T, 1, false><<<g, 256, 0, st>>>(a, ld, src, o, n, cols, parts, scale);
  else move_kernel<T, 1, true><<<g, 256, 0, st>>>(a, ld, src, o, n, cols, parts, scale);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}

template <typename Row>
int move_any(const void* in, long long ld, const Row& src, void* out, long long n, int cols, float scale, int dtype, cudaStream_t st) {
  if (n == 0 || cols == 0) return 0;
  switch (dtype) {
    case 0: return move_t<__nv_bfloat16>(in, ld, src, out, n, cols, scale, st);
    case 1: return move_t<__half>(in, ld, src, out, n, cols, scale, st);
    case 2: return move_t<float>(in, ld, src, out, n, cols, scale, st);
  }
  return -1;
}

// threads of a block that works on one row: up to two vectors each
inline int row_threads(int vecs, bool single) {
  if (single) return kSingleThreads;
  return vecs <= 32 ? 32 : vecs <= 64 ? 64 : vecs <= 256 ? 128 : 256;
}

template <typename T, int N, typename OutT>
int sum_t(const void* in, long long ld, const int* dest, const float* weight, void* out, int n, int k, int cols, cudaStream_t st) {
  const T* a = static_cast<const T*>(in);
  OutT* o = static_cast<OutT*>(out);
  const int threads = row_threads(cols / N, N == 1);
  if (weight) sum_kernel<T, N, true, OutT><<<n, threads, 0, st>>>(a, ld, dest, weight, o, k, cols);
  else sum_kernel<T, N, false, OutT><<<n, threads, 0, st>>>(a, ld, dest, weight, o, k, cols);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}
template <typename T, typename OutT>
int sum_any(const void* in, long long ld, const int* dest, const float* weight, void* out, int n, int k, int cols, cudaStream_t st) {
  return wide_rows(in, ld, cols, sizeof(T)) && reinterpret_cast<uintptr_t>(out) % 32 == 0
             ? sum_t<T, 16 / sizeof(T), OutT>(in, ld, dest, weight, out, n, k, cols, st)
             : sum_t<T, 1, OutT>(in, ld, dest, weight, out, n, k, cols, st);
}

template <typename T, typename G>
int sum_bwd_t(const void* d_out, long long ld, const void* y, long long ldy, const int* source, const int* dest, const float* weight, void* d_y, float* d_w,
              long long cap, long long n, int k, int cols, cudaStream_t st) {
  constexpr int NV = 16 / sizeof(T);
  const bool wide = wide_rows(y, ldy, cols, sizeof(T)) && wide_rows(d_y, cols, cols, sizeof(T)) && reinterpret_cast<uintptr_t>(d_out) % (NV * sizeof(G)) == 0 &&
                    ld % NV == 0;      // (so many elements of a row of d_out are one vector, too)
  const int threads = row_threads(cols / (wide ? NV : 1), !wide);
  const long long warps = threads / 32, some = padding_rows(cols / (wide ? NV : 1)), grid = n + (d_y ? ((cap + some - 1) / some + warps - 1) / warps : 0);
  if (grid > kMaxGrid) return -3;
  const G* a = static_cast<const G*>(d_out);
  const T* b = static_cast<const T*>(y);
  T* o = static_cast<T*>(d_y);
  const int g = static_cast<int>(grid);
  auto launch = [&](auto rows, auto weights) {
    constexpr bool kR = decltype(rows)::value, kW = decltype(weights)::value;
    if (wide) sum_bwd_kernel<T, NV, G, kR, kW><<<g, threads, 0, st>>>(a, ld, b, ldy, source, dest, weight, o, d_w, cap, n, k, cols);
    else sum_bwd_kernel<T, 1, G, kR, kW><<<g, threads, 0, st>>>(a, ld, b, ldy, source, dest, weight, o, d_w, cap, n, k, cols);
  };
  if (d_y && d_w) launch(std::true_type{}, std::true_type{});
  else if (d_y) launch(std::true_type{}, std::false_type{});
  else launch(std::false_type{}, std::true_type{});
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int N, typename OutT, bool kAdd>
int runs_t(const void* dy, long long ld, const int2* pairs, void* out, float* part, int* open, int n, int rows, int cols, float scale, cudaStream_t st) {
  const int per = 32 * N, parts = (cols + per - 1) / per;
  const long long chunks = (n + kRun - 1) / kRun, grid = grid_of(chunks * parts);
  if (grid > kMaxGrid) return -3;
  run_kernel<T, N, OutT, kAdd><<<static_cast<int>(grid), 256, 0, st>>>(static_cast<const T*>(dy), ld, pairs, static_cast<OutT*>(out), part, open, n, rows,
                                                                       cols, parts, scale);
  rb_note_launch(1);
  if (chunks > 1) {
    const long long most = 8ll * num_sms(), blocks = (chunks / 2 + 1) * parts < most ? (chunks / 2 + 1) * parts : most;
    merge_kernel<N, OutT, kAdd><<<static_cast<int>(blocks), 256, 0, st>>>(pairs, part, open, static_cast<OutT*>(out), n, cols, parts, scale);
    rb_note_launch(1);
  }
  return static_cast<int>(cudaGetLastError());
}
template <typename T>
int runs_any(const void* dy, long long ld, const int2* pairs, void* out, float* part, int* open, int n, int rows, int cols, float scale, int add, cudaStream_t st) {
  constexpr int NV = 16 / sizeof(T);
  const bool wide = wide_rows(dy, ld, cols, sizeof(T)) && wide_rows(out, cols, cols, add ? 4 : sizeof(T)) && wide_rows(part, cols, cols, 4);
  if (add) return wide ? runs_t<T, NV, float, true>(dy, ld, pairs, out, part, open, n, rows, cols, scale, st)
                       : runs_t<T, 1, float, true>(dy, ld, pairs, out, part, open, n, rows, cols, scale, st);
  return wide ? runs_t<T, NV, T, false>(dy, ld, pairs, out, part, open, n, rows, cols, scale, st)
              : runs_t<T, 1, T, false>(dy, ld, pairs, out, part, open, n, rows, cols, scale, st);
}

inline int key_bits(int rows) {      // of the keys 0 .. rows
  int b = 1;
  while (b < 31 && (rows >> b) != 0) ++b;
  return b;
}
constexpr int kPassBits = 10;
static_assert((1 << kPassBits) <= kThreads && (1 << kPassBits) <= kMaxBins, "pack_sort_kernel gives every bin a thread");

}  // namespace rows
}  // namespace rb

using namespace rb;
using namespace rb::rows;

extern "C" int rb_sort_counters(long long n, int bins) { return n > 0 && sort_blocks(n) > 1 ? sort_blocks(n) * bins : 1; }

// err (or null, where other ranks hold experts): a word that becomes 4 where an id is none of 0 .. experts - 1
extern "C" int rb_expert_layout(const void* ids, int wide, int n, int experts, int align, int cap, int* dest, int* source, int* tile_expert, int* bounds,
                                int* hist, int* err, cudaStream_t st) {
  if (n < 0 || n > kMaxSort || experts < 1 || experts > kMaxBins || align < 1 || cap < 0 || cap % align) return -1;
  const int tiles = align > 1 ? cap / align : 0;
  int at = 0;
  return sort_pass(ExpertKeys{ids, wide, experts, err}, ExpertOut{dest, source, align > 1 ? tile_expert : nullptr, bounds, cap, tiles}, n, experts, align, hist,
                   Fill{source, cap, nullptr, 0, 0, nullptr, 0, nullptr}, 1, &at, st);
}

template <typename T>
int spread_t(const void* in, long long ld, const int* source, const int* dest, void* out, long long cap, long long n, int k, int cols, cudaStream_t st) {
  constexpr int NV = 16 / sizeof(T);
  const int parts = (cols / NV + 32 * kMove<NV> - 1) / (32 * kMove<NV>);
  const long long grid = grid_of((n + (cap + 31) / 32) * parts);
  if (grid > kMaxGrid) return -3;
  spread_kernel<T, NV><<<static_cast<int>(grid), 256, 0, st>>>(static_cast<const T*>(in), ld, source, dest, static_cast<T*>(out), cap, n, k, cols, parts);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int rb_expert_dispatch(const void* x, long long ld, const int* source, const int* dest, void* out, int cap, int n, int k, int cols, int dtype,
                                  cudaStream_t st) {
  if (k < 1 || cap < 0 || n < 0 || cols < 0 || dtype < 0 || dtype > 2) return -1;
  if (cap == 0 || cols == 0) return 0;
  const int size = dtype == 2 ? 4 : 2;
  // Rows of many tokens fall out of the L2 between their experts: each is read once and put down k times (8 of 128 experts, width 2048:
  // 8192 tokens 55 us against 57 by buffer rows, 16384 104 against 130, 32768 195 against 287; fewer tokens are too few warps: 4096 34 against 30).
  if (k >= 2 && static_cast<long long>(n) * cols * size >= 24ll << 20 && wide_rows(x, ld, cols, size) && wide_rows(out, cols, cols, size)) {
    if (dtype == 0) return spread_t<__nv_bfloat16>(x, ld, source, dest, out, cap, n, k, cols, st);
    if (dtype == 1) return spread_t<__half>(x, ld, source, dest, out, cap, n, k, cols, st);
    return spread_t<float>(x, ld, source, dest, out, cap, n, k, cols, st);
  }
  return move_any(x, ld, SourceRow{source, k}, out, cap, cols, 1.f, dtype, st);
}

extern "C" int rb_expert_combine(const void* y, long long ld, const int* dest, const float* weight, void* out, int n, int k, int cols, int dtype,
                                 int out_fp32, cudaStream_t st) {
  if (k < 1 || n < 0 || cols < 0) return -1;
  if (n == 0 || cols == 0) return 0;
  switch (dtype) {
    case 0:
      return out_fp32 ? sum_any<__nv_bfloat16, float>(y, ld, dest, weight, out, n, k, cols, st)
                      : sum_any<__nv_bfloat16, __nv_bfloat16>(y, ld, dest, weight, out, n, k, cols, st);
    case 1: return out_fp32 ? sum_any<__half, float>(y, ld, dest, weight, out, n, k, cols, st) : sum_any<__half, __half>(y, ld, dest, weight, out, n, k, cols, st);
    case 2: return sum_any<float, float>(y, ld, dest, weight, out, n, k, cols, st);
  }
  return -1;
}

// out_fp32: d_out is in fp32, whatever the type of y.  d_y and d_w may be null: that gradient is not asked for; y is null where d_w is.
extern "C" int rb_expert_combine_bwd(const void* d_out, long long ld, const void* y, long long ldy, const int* source, const int* dest, const float* weight,
                                     void* d_y, float* d_w, int cap, int n, int k, int cols, int dtype, int out_fp32, cudaStream_t st) {
  if (k < 1 || n < 0 || cap < 0 || cols < 0) return -1;
  if ((cap == 0 && n == 0) || (!d_y && (!d_w || n == 0))) return 0;
  switch (dtype) {
    case 0:
      return out_fp32 ? sum_bwd_t<__nv_bfloat16, float>(d_out, ld, y, ldy, source, dest, weight, d_y, d_w, cap, n, k, cols, st)
                      : sum_bwd_t<__nv_bfloat16, __nv_bfloat16>(d_out, ld, y, ldy, source, dest, weight, d_y, d_w, cap, n, k, cols, st);
    case 1:
      return out_fp32 ? sum_bwd_t<__half, float>(d_out, ld, y, ldy, source, dest, weight, d_y, d_w, cap, n, k, cols, st)
                      : sum_bwd_t<__half, __half>(d_out, ld, y, ldy, source, dest, weight, d_y, d_w, cap, n, k, cols, st);
    case 2: return sum_bwd_t<float, float>(d_out, ld, y, ldy, source, dest, weight, d_y, d_w, cap, n, k, cols, st);
  }
  return -1;
}

// err (or null, for a shard): a word that becomes 4 where a token lies outside the table
extern "C" int rb_embedding(const void* ids, int wide, long long start, const void* table, long long ld, int rows, void* out, int n, int cols, float scale,
                            int dtype, int* err, cudaStream_t st) {
  if (n < 0 || cols < 0 || rows < 0) return -1;
  return move_any(table, ld, TokenRow{ids, wide, rows, start, err}, out, n, cols, scale, dtype, st);
}

extern "C" int rb_embedding_bwd_bins(int rows) {      // counters of one block in every pass
  const int bits = key_bits(rows), passes = (bits + kPassBits - 1) / kPassBits;
  return 1 << ((bits + passes - 1) / passes);
}

extern "C" int rb_embedding_bwd(const void* ids, int wide, long long start, const void* dy, long long ld, void* out, int add, int2* pairs, int* hist,
                                float* part, int* open, int n, int rows, int cols, float scale, int dtype, cudaStream_t st) {
  if (n < 0 || n > kMaxSort || rows < 0 || rows > kMaxSort || cols < 0) return -1;
  if (rows == 0 || cols == 0) return 0;
  const size_t bytes = static_cast<size_t>(rows) * cols * (dtype == 2 ? 4 : 2);
  if (n == 0) return add ? 0 : static_cast<int>(cudaMemsetAsync(out, 0, bytes, st));
  const int bits = key_bits(rows), passes = (bits + kPassBits - 1) / kPassBits, each = (bits + passes - 1) / passes;
  const int bins = 1 << each, mask = bins - 1;
  Fill fill{};
  fill.counter = open;
  if (!add) {
    if (reinterpret_cast<uintptr_t>(out) % 16) return -4;
    fill.far = static_cast<uint4*>(out);
    fill.hi = static_cast<long long>(bytes / 16);
    fill.rest = static_cast<unsigned char*>(out) + bytes / 16 * 16;
    fill.n_rest = static_cast<int>(bytes % 16);
  }
  int pos_bits = 1;
  while (pos_bits < 31 && ((n - 1) >> pos_bits) != 0) ++pos_bits;
  int2* to = pairs;
  int2* from = pairs + n;
  // one launch: few tokens, or a fill that takes longer than one block's sort (16384 tokens: 45 us, in four launches 18 us)
  const bool one = n <= kOneBlock || (n <= kPackSort && !add && bytes >= static_cast<size_t>(n) * 20000);
  if (one && pos_bits + bits <= 32) {
    const int rc = pack_sort(TokenKeys{ids, wide, rows, 0, mask, start}, from, n, pos_bits, passes, each, fill, st);
    if (rc) return rc;
  } else {
    const int launches = passes * (sort_blocks(n) > 1 ? 2 : 1);
    int at = 0;
    for (int p = 0; p < passes; ++p) {
      int rc;
      if (p == 0) rc = sort_pass(TokenKeys{ids, wide, rows, 0, mask, start}, PairOut{to}, n, bins, 1, hist, fill, launches, &at, st);
      else rc = sort_pass(PairKeys{from, p * each, mask}, PairOut{to}, n, bins, 1, hist, fill, launches, &at, st);
      if (rc) return rc;
      int2* s = to;
      to = from;
      from = s;
    }
  }
  switch (dtype) {
    case 0: return runs_any<__nv_bfloat16>(dy, ld, from, out, part, open, n, rows, cols, scale, add, st);
    case 1: return runs_any<__half>(dy, ld, from, out, part, open, n, rows, cols, scale, add, st);
    case 2: return runs_any<float>(dy, ld, from, out, part, open, n, rows, cols, scale, add, st);
  }
  return -1;
}
