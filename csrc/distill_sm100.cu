// Divergence of a student from a teacher known on K token ids per row, and the gradient of the student's logits.
//
//   s_i = z_i / T - log sum_v exp(z_v / T) on the K ids (the student), t_i given (the teacher), P = exp(s), Q = exp(t)
//   reverse  sum P (s - t),  forward  sum Q (t - s),  mixed  (1 - a) sum P (s - m) + a sum Q (t - m)  with exp(m) = (1 - a) P + a Q,
//   low variance  sum exp(t - s) - 1 + s - t;   over the K ids as they are, over the K ids renormalised, or over the K ids and one
//   bin with all other mass (no less than 1 - exp(-1e-7) of it).
//   d z_v = g / T (sum_i c_i [v = id_i] - P_v sum_i c_i)  with  c_i = dD / ds_i
//
// Both directions are bound by memory: the forward pass reads the logits once (maximum and sum together, the sum rescaled when the
// maximum grows), the backward pass reads them once more and writes the gradient; everything about the K ids is a few values per
// row.  The mass outside the ids is summed by itself - the ids are marked in a bitmap and left out - because 1 - sum P loses all
// digits where the ids hold nearly everything.  The forward pass is two kernels: one that streams the rows (several blocks per row
// where there are few of them) and a small one with the 64-bit arithmetic, which would cost the first its occupancy.
// Arithmetic: 32-bit exponentials (the instruction is off by 1.5e-7 at most, 5e-8 on average), 64 of them added in 32 bits, the rest of
// the sum and everything about the ids in 64.
// Measured (copy: 6.47 TB/s): 2048 rows of 151936 in bf16 124 us forward, where memory (96 us) and the exponentials (69 us) meet, and
// 174 us backward (193 us of a copy); 4096 rows in fp32 369 us (385) and 733 us (770); the ids 10 to 24 us.  A polynomial on the multiply-add
// pipe for a quarter of the exponentials made the first 6 us slower: instructions are no less scarce.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "api.h"
#include "host_utils.h"

namespace rb {
namespace distill {

constexpr int kThreads = 256, kHalfThreads = 128, kFewThreads = 64;      // of a block that streams a row or a part of it; of smaller ones
constexpr int kMaxIds = 1024, kMine = kMaxIds / kThreads;      // ids of a row; of a thread of a streaming block
constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxParts = 32;      // blocks of a row
constexpr int kStats = 4;      // per row: log2 reference, 1 / sum, sum of the slopes, power of two of a far row's sum and a half (or 0)
constexpr double kLn2 = 0.6931471805599453, kLog2e = 1.4426950408889634;
constexpr double kLeastRest = 9.9999995e-08;      // 1 - exp(-1e-7)

enum Kl { kReverse = 0, kForward = 1, kMixed = 2, kLowVar = 3 };
enum Norm { kTail = 0, kNorm = 1, kTrunc = 2 };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows are summed against a whole number near their largest z log2(e) / T.  As far as kFar, 32 bits in two parts tell z log2(e) / T from it;
// rows (and steps) whose largest logit is further away - masks of -1e9, say, that leave nothing - are taken in 64 bits.  Beyond kBeyond, where
// neighbouring 32-bit numbers lie 512 apart, a logit is what its 32-bit product is, and the products end at kLow: a type's lowest value would
// pass it.  A row of nothing but one such value is uniform, and beside other logits it has no mass either way.
constexpr float kFar = 1048576.f, kBeyond = 4294967296.f, kLow = -3.4e38f;
__device__ __noinline__ double far_mass(float z, double scale, float c2, float ref) {      // 2^(z scale - ref), NaN stays
  if (z == -INFINITY) return 0.0;
  const float x = z * c2;
  if (fabsf(ref) > kBeyond) return static_cast<double>(ex2((x < kLow ? kLow : x) - ref));
  return exp2(static_cast<double>(z) * scale - static_cast<double>(ref));      // (2^512 at most)
}
// s 2^d for a whole number d, at most 0 (from 2^-1022 on there is nothing left of sums that begin at 2^512)
__device__ __forceinline__ double moved(double s, float d) {
  return s * __hiloint2double((1023 + static_cast<int>(fmaxf(d, -1022.f))) << 20, 0);
}

// the whole number at or above z log2(e) / T
__device__ __forceinline__ float whole_ref(float z, float c2) {
  const float x = z * c2;
  return z == -INFINITY ? z : ceilf(x < kLow ? kLow : x);      // (NaN stays)
}
__device__ __forceinline__ float max_nan(float a, float b) {      // (fmaxf would drop a NaN)
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// two 32-bit operations at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}

// eight consecutive elements, aligned to their size
template <typename T> struct Eight;
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ float max() const {
    return max_nan(max_nan(max_nan(a.x, a.y), max_nan(a.z, a.w)), max_nan(max_nan(b.x, b.y), max_nan(b.z, b.w)));
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ static void store(float* p, const float* f) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <> struct Eight<__nv_bfloat16> {
  __nv_bfloat162 h[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ float max() const {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __bfloat1622float2(h[i]);
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  __device__ __forceinline__ static void store(__nv_bfloat16* p, const float* f) {
    uint4 u;
    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  }
};
template <> struct Eight<__half> {
  __half2 h[4];
  __device__ __forceinline__ void load(const __half* p) { *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ float max() const {
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(h[i]);
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  __device__ __forceinline__ static void store(__half* p, const float* f) {
    uint4 u;
    __half2* o = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  }
};
__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half(v); }

struct Params {
  const void* z;               // [rows, vocab] logits, pitch ld
  long long ld;
  const long long* ids;        // [rows, k]; outside 0 .. vocab - 1: no id
  const float* teacher;        // [rows, k] log-probs
  float* loss;                 // [rows]
  float* coef;                 // [rows, k] logits of the ids (from one kernel to the other), then d D / d z of the ids, times T
  float* stats;                // [rows, kStats]
  float* log_probs;            // [rows, k] or null
  double2* sums;               // [rows, parts] (reference, sum) of the parts of a row
  int vocab, k, kl, norm, parts;
  float c2, c2_low;            // log2(e) / T and what 32 bits leave of it
  double scale;                // log2(e) / T
  double alpha, clamp;         // weight of the teacher; least log-prob
};

// (reference, sum): the sum of 2^(z c2) is sum 2^reference.  References are whole numbers, so that moving a sum to another one is exact
// (each move by an approximate power took 5e-8 off the sum, 2.5e-7 in all).
struct Sum {
  float ref;
  double sum;
  __device__ __forceinline__ void add(float r, double s) {      // nothing yet: ref -inf, sum 0
    const float m = fmaxf(ref, r), at = m == -INFINITY ? 0.f : m;
    sum = moved(sum, ref - at) + moved(s, r - at);
    ref = m;
  }
};

constexpr int kIdThreads = 128, kIdWarps = kIdThreads / 32;      // most of the kernel that looks at a row's ids
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double (*sm)[kIdWarps]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) sm[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0;
    for (int w = 0; w < warps; ++w) v[i] += sm[i][w];
  }
}

template <int N>
__device__ __forceinline__ void block_max(double (&v)[N], double (*sm)[kIdWarps]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] = fmax(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) sm[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int w = 0; w < warps; ++w) v[i] = fmax(v[i], sm[i][w]);
}

__device__ __forceinline__ double least(double x, double c) { return x < c ? c : x; }      // (NaN stays)
// 0 log 0 = 0: a term whose weight is nothing counts nothing
__device__ __forceinline__ double weighted(double w, double x) { return w == 0.0 ? 0.0 : w * x; }
struct Term {
  double d, slope;      // D's term and its derivative by P
};
// p, q the masses and l = log(p / q).  The mixture's logs come from l: log(p / m) = -log(1 + a (q / p - 1)) keeps its digits where p
// and q are near each other, and the like from the side of q where q is the larger.
__device__ __forceinline__ Term term_of(int kl, double a, double p, double q, double l) {
  Term r;
  if (kl == kReverse) {
    r.d = weighted(p, l);
    r.slope = l + 1.0;
  } else if (kl == kForward) {
    r.d = weighted(q, -l);
    r.slope = -q / p;
  } else {
    double pm, qm;      // log(p / m), log(q / m)
    if (l >= 0.0) {
      pm = -log1p(a * expm1(-l));
      qm = pm - l;
    } else {
      qm = -log1p((1.0 - a) * expm1(l));
      pm = l + qm;
    }
    r.d = (1.0 - a) * weighted(p, pm) + a * weighted(q, qm);
    r.slope = (1.0 - a) * pm;
  }
  return r;
}

// Sums over the vocabulary, `parts` blocks per row.  The row counts from the last address in front of it that is a multiple of eight
// elements, so that all but its first and last group of eight are whole; groups are shared out to the blocks in runs.
template <typename T, int kBlock>
__global__ void __launch_bounds__(kBlock, 1024 / kBlock) sum_kernel(Params p) {
  const long long row = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x - row * p.parts), t = threadIdx.x;
  extern __shared__ unsigned marks[];      // a bit per element of this block's groups
  __shared__ Sum warp_sum[kBlock / 32];
  const T* z = static_cast<const T*>(p.z) + row * p.ld;
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(z) / sizeof(T)) & 7);      // elements in front of the row in its first group
  const T* origin = z - skip;
  const int groups = (skip + p.vocab + 7) >> 3, each = (groups + p.parts - 1) / p.parts;
  const int g0 = min(groups, part * each), g1 = min(groups, g0 + each);
  const int w0 = g0 == 0 && skip ? 1 : g0, w1 = (g1 == groups && ((skip + p.vocab) & 7)) ? g1 - 1 : g1;      // whole groups

  for (int i = t; i < (each + 3) / 4; i += kBlock) marks[i] = 0;
  __syncthreads();
  // logits of this part's ids, for the kernel behind this one: fetched here, where other blocks keep the memory busy meanwhile (K
  // scattered reads per row by themselves took 116 us for 4096 rows of 128), and put down at the end
  float at_id[kMine];
  unsigned here = 0;
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int i = t + j * kBlock;
    if (i >= p.k) break;
    const long long v = p.ids[row * p.k + i], b = v + skip - 8ll * g0;
    if (v >= 0 && v < p.vocab && b >= 0 && b < 8ll * (g1 - g0)) {
      here |= 1u << j;
      at_id[j] = up(z[v]);
      atomicOr(&marks[b >> 5], 1u << (b & 31));
    }
  }
  __syncthreads();
  const unsigned char* mark = reinterpret_cast<const unsigned char*>(marks);

  Sum s{-INFINITY, 0.0};
  unsigned far = 0;      // steps left out: 1 below, 2 above
  constexpr int U = sizeof(T) == 4 ? 4 : 8;      // groups of a thread in one step: 128 bytes of it under way
  // U groups from g on, in strides of the block; the last step (kAll false) holds what is left
  auto step = [&](int g, auto all) {
    constexpr bool kAll = decltype(all)::value;
    Eight<T> e[U];
    unsigned m[U];
    float big = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kAll || g + u * kBlock < w1) e[u].load(origin + 8ll * (g + u * kBlock));
#pragma unroll
    for (int u = 0; u < U; ++u) m[u] = kAll || g + u * kBlock < w1 ? mark[g + u * kBlock - g0] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kAll || g + u * kBlock < w1) big = max_nan(big, e[u].max());
    big = whole_ref(big, p.c2);
    if (fabsf(big) > kFar) {      // nothing there (-inf), or for the loop behind this one
      far |= big > 0.f ? 2u : big != -INFINITY;
      return;
    }
    if (big > s.ref) {
      s.sum = moved(s.sum, s.ref - big);
      s.ref = big;
    }
    const float at = s.ref == -INFINITY ? 0.f : s.ref;
    const float2 c = make_float2(p.c2, p.c2), l = make_float2(p.c2_low, p.c2_low), o = make_float2(-at, -at);
    float2 add = make_float2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kAll || g + u * kBlock < w1) {
        float f[8];
        e[u].get(f);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 y = make_float2(f[i], f[i + 1]), x = fma2(y, l, fma2(y, c, o));
          f[i] = ex2(x.x), f[i + 1] = ex2(x.y);
        }
        if (m[u]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = (m[u] >> i) & 1 ? 0.f : f[i];
        }
        add = add2(add, add2(add2(make_float2(f[0], f[1]), make_float2(f[2], f[3])), add2(make_float2(f[4], f[5]), make_float2(f[6], f[7]))));
      }
    s.sum += static_cast<double>(add.x + add.y);
  };
  int g = w0 + t;
  for (; g + (U - 1) * kBlock < w1; g += U * kBlock) step(g, std::true_type{});
  if (g < w1) step(g, std::false_type{});
  // steps whose largest logit is far away, once more; those far below are nothing where some other logit is not
  if (__syncthreads_or(s.ref > 4096.f - kFar)) far &= 2;
  if (far) {
#pragma unroll 1
    for (g = w0 + t; g < w1; g += U * kBlock) {
      float big = -INFINITY;
#pragma unroll 1
      for (int q = g; q < w1 && q < g + U * kBlock; q += kBlock)
        for (int i = 0; i < 8; ++i) big = max_nan(big, up(origin[8ll * q + i]));
      big = whole_ref(big, p.c2);
      if (!(fabsf(big) > kFar) || big == -INFINITY || (far == 2 && big < 0.f)) continue;
      Sum some{big, 0.0};
#pragma unroll 1
      for (int q = g; q < w1 && q < g + U * kBlock; q += kBlock)
        for (int i = 0; i < 8; ++i)
          if (!((mark[q - g0] >> i) & 1)) some.sum += far_mass(up(origin[8ll * q + i]), p.scale, p.c2, big);
      s.add(some.ref, some.sum);
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the small kernel may come in and set up its table
  // the row's first and last group, where they are not whole: one element per thread
  if (t < 16) {
    const int g = t < 8 ? 0 : groups - 1, i = t & 7;
    const long long v = 8ll * g + i - skip;
    const bool mine = t < 8 ? (g0 == 0 && skip) : (g1 == groups && ((skip + p.vocab) & 7) && !(groups == 1 && skip));
    if (mine && g0 < g1 && v >= 0 && v < p.vocab) {
      const bool counts = !((mark[g - g0] >> i) & 1);
      const float y = up(z[v]), x = whole_ref(y, p.c2);
      const double own = x == -INFINITY ? 0.0 : fabsf(x) > kFar ? far_mass(y, p.scale, p.c2, x) : static_cast<double>(ex2(fmaf(y, p.c2_low, fmaf(y, p.c2, -x))));
      s.add(x, counts ? own : 0.0);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s.add(__shfl_xor_sync(0xffffffffu, s.ref, o), __shfl_xor_sync(0xffffffffu, s.sum, o));
  if ((t & 31) == 0) warp_sum[t >> 5] = s;
  __syncthreads();
  if (t == 0) {
    Sum b = warp_sum[0];
#pragma unroll
    for (int w = 1; w < kBlock / 32; ++w) b.add(warp_sum[w].ref, warp_sum[w].sum);
    p.sums[blockIdx.x] = make_double2(b.ref, b.sum);
  }
#pragma unroll
  for (int j = 0; j < kMine; ++j)
    if ((here >> j) & 1) p.coef[row * p.k + t + j * kBlock] = at_id[j];
}

// every bit of an id in every bit of its slot: ids at even distances would fill one stretch of the table otherwise
__device__ __forceinline__ unsigned mixed(unsigned x) {
  x = (x ^ (x >> 16)) * 0x9e3779b1u;
  x = (x ^ (x >> 15)) * 0x9e3779b1u;
  return x ^ (x >> 16);
}

// The K ids of a row: the divergence, its slopes, the row's statistics, in 64 bits: where student and teacher are near each other the
// divergence is a small difference of its terms (32-bit masses left it 2e-5 off).  Equal ids are found with a hash table that keeps the first place of every id.
__global__ void __launch_bounds__(kIdThreads) id_kernel(Params p, int slots) {
  const long long row = blockIdx.x;
  const int t = threadIdx.x, threads = blockDim.x;
  extern __shared__ __align__(16) unsigned char dyn[];
  double* lp = reinterpret_cast<double*>(dyn);                // [k] log-probs of the student, then slopes
  double* pm = lp + p.k;                                      // [k] places in the table, then probabilities of the student
  int* id = reinterpret_cast<int*>(pm + p.k);                 // [k] the row's ids, -1: none
  float* tl = reinterpret_cast<float*>(id + p.k);             // [k] log-probs of the teacher
  int* key = reinterpret_cast<int*>(tl + p.k);                // [slots] ids (a power of two, at least 2 k)
  int* place = key + slots;                                   // [slots] where they stand first
  __shared__ double red[4][kIdWarps];
  const bool tail = p.norm == kTail && p.kl != kLowVar, renorm = p.norm == kNorm && p.kl != kLowVar;
  for (int i = t; i < slots; i += threads) key[i] = -1, place[i] = p.k;
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the streaming kernel is done, and what it wrote can be seen
  Sum all{-INFINITY, 0.0};
  for (int r = 0; r < p.parts; ++r) {
    const double2 s = p.sums[row * p.parts + r];
    all.add(static_cast<float>(s.x), s.y);
  }
  const double ref = all.ref == -INFINITY ? 0.0 : static_cast<double>(all.ref), rest_sum = all.sum;
  const bool beyond = fabs(ref) > kBeyond;
  bool some = false;
  __syncthreads();
  for (int i0 = t; i0 < p.k; i0 += 4 * threads) {      // four ids at a time: they wait for memory
    int v[4];
    float z[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * threads;
      const long long w = i < p.k ? p.ids[row * p.k + i] : -1;
      v[u] = w >= 0 && w < p.vocab ? static_cast<int>(w) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * threads;
      if (i < p.k) tl[i] = p.teacher[row * p.k + i];
      z[u] = v[u] >= 0 ? p.coef[row * p.k + i] : 0.f;      // (its logit, for now)
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * threads;
      if (i >= p.k) break;
      id[i] = v[u];
      if (v[u] < 0) continue;
      some = true;
      const float x = z[u] * p.c2;
      const double y = beyond ? static_cast<double>(x < kLow && z[u] != -INFINITY ? kLow : x) : static_cast<double>(z[u]) * p.scale;
      lp[i] = (y - ref) * kLn2;      // z - reference in units of ln
      unsigned h = mixed(v[u]);
      for (;; ++h) {      // (ends: no more than half the slots are taken)
        const int was = atomicCAS(&key[h & (slots - 1)], -1, v[u]);
        if (was == -1 || was == v[u]) break;
      }
      atomicMin(&place[h & (slots - 1)], i);
      pm[i] = static_cast<double>(h & (slots - 1));
    }
  }
  if (!__syncthreads_or(some)) {      // no ids: nothing to compare, whatever the logits are
    for (int i = t; i < p.k; i += threads) {
      p.coef[row * p.k + i] = 0.f;
      if (p.log_probs) p.log_probs[row * p.k + i] = -INFINITY;
    }
    if (t == 0) p.loss[row] = 0.f, *reinterpret_cast<float4*>(p.stats + row * kStats) = make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  double one[1] = {0.0};
  unsigned firsts = 0, moving = 0;      // a bit for each of this thread's ids
  for (int i = t, n = 0; i < p.k; i += threads, ++n) {
    if (id[i] < 0) continue;
    const bool first = place[static_cast<int>(pm[i])] == i;
    firsts |= static_cast<unsigned>(first) << n;
    pm[i] = exp(lp[i]);
    if (first) one[0] += pm[i];
  }
  block_sums(one, red);      // the sum over the vocabulary left the ids out
  const double total = rest_sum + one[0], log_total = log(total), inv_total = 1.0 / total;

  // masses of the ids (renormalised), what the rest lacks (equal ids and clamped ones count as written), ids in all
  double mass[4] = {0.0, 0.0, 0.0, 0.0}, most[2] = {-INFINITY, -INFINITY};
  bool twice = false;
  for (int i = t, n = 0; i < p.k; i += threads, ++n) {
    if (id[i] < 0) continue;
    const bool first = (firsts >> n) & 1;
    twice |= !first;
    lp[i] -= log_total;
    pm[i] *= inv_total;
    if (p.log_probs) p.log_probs[row * p.k + i] = static_cast<float>(lp[i]);
    if (!tail && !renorm) continue;
    const double used = least(lp[i], p.clamp), t_i = least(static_cast<double>(tl[i]), p.clamp);
    if (tail) {
      const double pu = used == lp[i] ? pm[i] : exp(used);
      mass[1] += exp(t_i);
      mass[2] += pu - (first ? pm[i] : 0.0);
    } else {
      most[0] = used > most[0] ? used : most[0];
      most[1] = t_i > most[1] ? t_i : most[1];
    }
  }
  double* pn = reinterpret_cast<double*>(key);      // [k] renormalised masses of the student (the table is no longer needed)
  if (renorm) {      // against the largest of them: ids far behind the others would have no mass left to renormalise
    block_max(most, red);
    for (int i = t; i < p.k; i += threads) {
      if (id[i] < 0) continue;
      pn[i] = exp(least(lp[i], p.clamp) - most[0]);
      mass[0] += pn[i];
      mass[1] += exp(least(static_cast<double>(tl[i]), p.clamp) - most[1]);
      mass[3] += pn[i] == 1.0 ? 1.0 : 2.0;
    }
  }
  if (tail || renorm) block_sums(mass, red);
  double rest_slope = 0.0, rest = 0.0;
  if (tail) {
    const double free = rest_sum / total - mass[2];      // (exactly one where there are no ids)
    const double pr = least(free, kLeastRest), qr = least(1.0 - mass[1], kLeastRest);
    const Term r = term_of(p.kl, p.alpha, pr, qr, log(pr / qr));
    rest = r.d;
    rest_slope = free >= kLeastRest ? r.slope : 0.0;
  }
  const bool alone = renorm && mass[3] == 1.0 && mass[1] == 1.0;      // all mass is this id's, on both sides
  const double ls = renorm ? log(mass[0] / mass[1]) : 0.0, np = renorm ? 1.0 / mass[0] : 1.0, nq = renorm ? 1.0 / mass[1] : 1.0;
  double sums[4] = {0.0, 0.0, 0.0, 0.0};      // the divergence; slopes of all ids; slopes and masses of those that move
  for (int i = t, n = 0; i < p.k; i += threads, ++n) {
    if (id[i] < 0) {
      if (p.log_probs) p.log_probs[row * p.k + i] = -INFINITY;
      continue;
    }
    const double s_i = lp[i], t_i = least(static_cast<double>(tl[i]), p.clamp), used = least(s_i, p.clamp);
    const bool moves = !(s_i < p.clamp);      // clamped ids do not
    double c, pp = 0.0;
    if (p.kl == kLowVar) {
      const double r = used - t_i, x = exp(-r);
      sums[0] += x - 1.0 + r;
      c = 1.0 - x;
    } else {
      const double qq = renorm ? exp(t_i - most[1]) * nq : exp(t_i);
      pp = renorm ? pn[i] * np : moves ? pm[i] : exp(used);
      const Term r = term_of(p.kl, p.alpha, pp, qq, alone ? 0.0 : renorm ? (used - most[0]) - (t_i - most[1]) - ls : used - t_i);
      sums[0] += r.d;
      c = (p.kl == kForward ? -qq : weighted(pp, r.slope)) - weighted(pp, rest_slope);
    }
    sums[1] += c;
    if (moves) {
      sums[2] += c;
      sums[3] += pp;
      moving |= 1u << n;
    }
    lp[i] = moves ? c : 0.0;
  }
  block_sums(sums, red);
  double move = sums[2];
  if (renorm) {      // c_i - P_i sum c
    move -= sums[1] * sums[3];
    for (int i = t, n = 0; i < p.k; i += threads, ++n)
      if ((moving >> n) & 1) lp[i] -= pn[i] * np * sums[1];
  }
  // what the logit of an id gets, its share of the sum of the slopes with it; equal ids move together
  const bool sum_equals = __syncthreads_or(twice);
  for (int i = t; i < p.k; i += threads) {
    double c = 0.0;
    if (id[i] >= 0) {
      c = lp[i];
      if (sum_equals) {
        c = 0.0;
        for (int j = 0; j < p.k; ++j) c += id[j] == id[i] ? lp[j] : 0.0;
      }
      c -= move * pm[i];
    }
    p.coef[row * p.k + i] = static_cast<float>(c);
  }
  if (t == 0) {
    p.loss[row] = static_cast<float>(sums[0] + rest);
    // the sum's power of two goes to the reference: 1 / sum is no less than a half.  Far references have no place for it.
    const int e = total > 0.0 && total < INFINITY ? ilogb(total) : 0;
    const bool far = fabs(ref) > kFar;
    *reinterpret_cast<float4*>(p.stats + row * kStats) =
        make_float4(static_cast<float>(far ? ref : ref + e), static_cast<float>(ldexp(inv_total, e)), static_cast<float>(move), far ? e + 0.5f : 0.f);
  }
}

struct BwdParams {
  const void* z;
  long long ld;
  const long long* ids;
  const float* coef;
  const float* stats;
  const float* g;          // [rows] gradient of the divergence
  void* dz;                // [rows, vocab] dense (may be z itself where types agree)
  int vocab, k, parts;
  float c2, c2_low, inv_t;
  double scale;
};

// A block per part of a row: -g / T (sum c) P over its elements, then the K ids of that part in place of what stands there.
template <typename T, typename O, bool kWhole, int kBlock>
__global__ void __launch_bounds__(kBlock) bwd_kernel(BwdParams p) {
  const long long row = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x - row * p.parts), t = threadIdx.x;
  const T* z = static_cast<const T*>(p.z) + row * p.ld;
  O* d = static_cast<O*>(p.dz) + row * p.vocab;
  const float g = p.g[row] * p.inv_t;
  const float ref = p.stats[row * kStats], inv = p.stats[row * kStats + 1], csum = p.stats[row * kStats + 2];
  const float f = g == 0.f ? 0.f : -g * csum * inv, power = p.stats[row * kStats + 3];
  const bool far = power != 0.f;
  const int skip = kWhole ? static_cast<int>((reinterpret_cast<uintptr_t>(z) / sizeof(T)) & 7) : 0;
  const int groups = (skip + p.vocab + 7) >> 3, each = (groups + p.parts - 1) / p.parts;
  const int g0 = min(groups, part * each), g1 = min(groups, g0 + each);
  const long long lo = max(0ll, 8ll * g0 - skip), hi = min(static_cast<long long>(p.vocab), 8ll * g1 - skip);
  if (lo >= hi) return;
  auto mass = [&](float x) { return ex2(fmaf(x, p.c2_low, fmaf(x, p.c2, -ref))); };
  auto one = [&](long long v) {
    put(d + v, f == 0.f ? 0.f : far ? static_cast<float>(f * ldexp(far_mass(up(z[v]), p.scale, p.c2, ref), -static_cast<int>(floorf(power)))) : f * mass(up(z[v])));
  };
  if (!kWhole || (far && f != 0.f)) {
    for (long long v = lo + t; v < hi; v += kBlock) one(v);
  } else {
    const int w0 = g0 == 0 && skip ? 1 : g0, w1 = (g1 == groups && ((skip + p.vocab) & 7)) ? g1 - 1 : g1;
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    for (int q = w0 + t; q < w1; q += kBlock * U) {
      Eight<T> e[U];
      if (f != 0.f) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (q + u * kBlock < w1) e[u].load(z + (8ll * (q + u * kBlock) - skip));
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * kBlock < w1) {
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (f != 0.f) {
            e[u].get(x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = f * mass(x[i]);
          }
          Eight<O>::store(d + (8ll * (q + u * kBlock) - skip), x);
        }
    }
    if (t < 16) {
      const int q = t < 8 ? 0 : groups - 1;
      const long long v = 8ll * q + (t & 7) - skip;
      const bool mine = t < 8 ? (g0 == 0 && skip) : (g1 == groups && ((skip + p.vocab) & 7) && !(groups == 1 && skip));
      if (mine && v >= 0 && v < p.vocab) one(v);
    }
  }
  if (g == 0.f) return;
  __syncthreads();
  for (int i = t; i < p.k; i += kBlock) {
    const long long v = p.ids[row * p.k + i];
    if (v >= lo && v < hi) put(d + v, g * p.coef[row * p.k + i]);
  }
}

// Blocks of a row for kernels of `slots` blocks at a time: the number with the shortest waves, where a block costs as much as `fixed`
// groups of eight beside its own.  (2048 rows of 151936, while a block's own part of the work was smaller: two parts in 7 waves 108 us;
// one part in 4 waves, the last of them less than half full, 115 us; four parts 127 us.)
inline int parts_of(long long rows, int vocab, long long slots, int fixed) {
  const long long groups = (vocab + 7) / 8;
  int best = 1;
  long long cost = 0;
  for (int p = 1; p <= kMaxParts && (p == 1 || groups / p >= 512); ++p) {
    const long long c = (rows * p + slots - 1) / slots * (groups / p + fixed);
    if (p == 1 || c < cost) best = p, cost = c;
  }
  return best;
}
// log2(e) / T in two 32-bit numbers.  Both are above zero: a logit of -inf stays -inf in z c2 + z c2_low.
inline void two_floats(double scale, float& c2, float& c2_low) {
  c2 = static_cast<float>(scale);
  if (static_cast<double>(c2) > scale) c2 = nextafterf(c2, 0.f);
  c2_low = fmaxf(static_cast<float>(scale - c2), FLT_MIN);
}

template <typename T, int kBlock>
int sums_t(const Params& p, long long rows, cudaStream_t st) {
  const int each = ((p.vocab + 14) / 8 + p.parts - 1) / p.parts + 1;
  const size_t smem = (each + 3) / 4 * 4 + 16;
  constexpr size_t kMostSmem = 200 * 1024;      // (always the same limit: calls of several threads would lower one another's)
  if (smem > kMostSmem) return -4;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(sum_kernel<T, kBlock>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  sum_kernel<T, kBlock><<<static_cast<unsigned>(rows * p.parts), kBlock, smem, st>>>(p);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}
// Rows that take more than one wave of large blocks but one of blocks half their size: the second wave is mostly empty (777 rows of 32003 in
// bf16, ids included: 30 us against 39 with large blocks; of 151936 68 against 72; fp32: 777 rows of 4099 17.4 against 19.5, of 32003 39 against
// 42, of 50000 48.6 against 52, of 65536 57 against 59; 1000 and 1184 rows of 32003 to 65536 within one in a hundred; of 151936 106 against 100).
inline bool one_wave_of_halves(long long rows, int vocab, int size) {
  return rows > 4ll * num_sms() && rows <= 8ll * num_sms() && vocab <= (size == 2 ? 200000 : 65536);      // (eight bitmaps fit shared memory)
}
// Many short rows: small blocks, so that more rows are under way and wait for their ids and their sums side by side (8192 rows of 4096 in
// bf16, ids included: 50 us against 91 with large blocks; of 12000: 81 against 108; of 32000: 134 against 149, but 204 against 189 in fp32).
template <typename T>
int sums_of(const Params& p, long long rows, cudaStream_t st) {
  if (p.vocab <= 16384 && rows >= 8ll * num_sms() && p.parts == 1 && p.k <= kMine * kFewThreads) return sums_t<T, kFewThreads>(p, rows, st);
  if (one_wave_of_halves(rows, p.vocab, sizeof(T)) && p.k <= kMine * kHalfThreads) return sums_t<T, kHalfThreads>(p, rows, st);
  return sums_t<T, kThreads>(p, rows, st);
}

template <typename T, typename O>
int bwd_t(BwdParams p, long long rows, cudaStream_t st) {
  // blocks of at least 24576 elements where rows are long (2048 rows of 151936 in bf16: six parts 201 us, one 221, sixteen 240)
  const int most = p.vocab / 24576 < kMaxParts ? p.vocab / 24576 : kMaxParts;
  p.parts = parts_of(rows, p.vocab, 5ll * num_sms(), 500);
  p.parts = p.parts > most ? p.parts : most;
  if (rows * p.parts > 2147483647ll) return -3;
  // groups of eight line up in both where rows keep their distance and begin alike
  const uintptr_t a = reinterpret_cast<uintptr_t>(p.z) / sizeof(T), b = reinterpret_cast<uintptr_t>(p.dz) / sizeof(O);
  const bool whole = (a - b) % 8 == 0 && (rows == 1 || (p.ld - p.vocab) % 8 == 0);
  const int grid = static_cast<int>(rows * p.parts);
  // many short rows: small blocks (8192 rows of 1024 in bf16 19 us against 33, of 4096 31 against 41, in fp32 53 both; of 12000 fp32 152 against 130)
  const bool few = p.vocab <= 4096 && rows >= 8ll * num_sms();
  if (whole && few) bwd_kernel<T, O, true, kFewThreads><<<grid, kFewThreads, 0, st>>>(p);
  else if (whole) bwd_kernel<T, O, true, kThreads><<<grid, kThreads, 0, st>>>(p);
  else bwd_kernel<T, O, false, kThreads><<<grid, kThreads, 0, st>>>(p);
  rb_note_launch(1);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace distill
}  // namespace rb

using namespace rb;
using namespace rb::distill;

// Blocks per row, and so pairs of doubles per row that rb_topk_distill takes as workspace.  size: bytes of a logit.
extern "C" int rb_topk_distill_parts(long long rows, int vocab, int k, int size) {
  // More ids than small blocks hold leave large blocks: parts pay where rows are long (700 rows, 600 ids: of 151936 in bf16 87 us against 91 of
  // whole rows, of 65536 in fp32 68 against 75), not where every part's own look at the ids costs more (32003 in bf16 52 against 48, in fp32 54
  // against 53; 65536 in bf16 63 against 60; 100000 in bf16 75 both).
  if (one_wave_of_halves(rows, vocab, size) && (k <= kMine * kHalfThreads || static_cast<long long>(vocab) * size <= 200000)) return 1;
  const int parts = parts_of(rows, vocab, 4ll * num_sms(), 1000);      // (a fixed 2 us of 4 blocks per SM)
  return vocab / parts > (1 << 20) ? kMaxParts : parts;                 // the bitmap of a part fits shared memory
}

// dtype: 0 bf16, 1 fp16, 2 fp32.  kl: reverse, forward, mixed, low variance; norm: tail bin, renormalised, as they are.
extern "C" int rb_topk_distill(const void* z, long long ld, const long long* ids, const float* teacher, float* loss, float* coef, float* stats,
                               float* log_probs, double2* sums, long long rows, int vocab, int k, int kl, int norm, double alpha, double clamp,
                               double inv_temp, int dtype, cudaStream_t st) {
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab || k < 0 || k > kMaxIds || kl < 0 || kl > 3 || norm < 0 || norm > 2 || !(inv_temp > 0.0)) return -1;
  if (rows == 0) return 0;
  const int parts = rb_topk_distill_parts(rows, vocab, k, dtype == 2 ? 4 : 2);
  if (rows * parts > 2147483647ll) return -3;
  const double scale = inv_temp * kLog2e;
  float c2, c2_low;
  two_floats(scale, c2, c2_low);
  const Params p{z, ld, ids, teacher, loss, coef, stats, log_probs, sums, vocab, k, kl, norm, parts, c2, c2_low, scale, alpha, clamp};
  int rc = -1;
  switch (dtype) {
    case 0: rc = sums_of<__nv_bfloat16>(p, rows, st); break;
    case 1: rc = sums_of<__half>(p, rows, st); break;
    case 2: rc = sums_of<float>(p, rows, st); break;
  }
  if (rc) return rc;
  // many rows: a warp each, which spends the fewest instructions (8192 rows of 4096 and 128 ids, streaming included: 112 us, a thread per id
  // 157); few: a thread per id, for the shortest way (the same time up to 64 ids)
  int threads = rows >= 8ll * num_sms() ? 32 : (k + 31) / 32 * 32, slots = 32;
  threads = threads < 32 ? 32 : threads > kIdThreads ? kIdThreads : threads;
  while (slots < 2 * k) slots *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(k) * 24 + slots * 8;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, id_kernel, p, slots);
  rb_note_launch(1);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// out_dtype: that of the logits, or 0 (bf16) for logits in fp32
extern "C" int rb_topk_distill_bwd(const void* z, long long ld, const long long* ids, const float* coef, const float* stats, const float* g, void* dz,
                                   long long rows, int vocab, int k, double inv_temp, int dtype, int out_dtype, cudaStream_t st) {
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab || k < 0 || k > kMaxIds || !(inv_temp > 0.0)) return -1;
  if (rows == 0) return 0;
  const double scale = inv_temp * kLog2e;
  float c2, c2_low;
  two_floats(scale, c2, c2_low);
  const BwdParams p{z, ld, ids, coef, stats, g, dz, vocab, k, 1, c2, c2_low, static_cast<float>(inv_temp), scale};
  if (dtype == 0 && out_dtype == 0) return bwd_t<__nv_bfloat16, __nv_bfloat16>(p, rows, st);
  if (dtype == 1 && out_dtype == 1) return bwd_t<__half, __half>(p, rows, st);
  if (dtype == 2 && out_dtype == 2) return bwd_t<float, float>(p, rows, st);
  if (dtype == 2 && out_dtype == 0) return bwd_t<float, __nv_bfloat16>(p, rows, st);
  return -1;
}
