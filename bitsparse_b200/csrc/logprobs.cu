// Log probabilities of given tokens, with entropy and top alternatives, and
// the gradient of the logits.
//
//   z_j = (x_j - m) / temperature, m = max x;  S = sum e^z_j
//   logprob = z_t - log S;  H = log S - (sum e^z_j z_j) / S
//   dx_j = (gl (delta_jt - p_j) - gh p_j (log p_j + H)) / temperature
//
// Forward: one pass over the logits.  A thread keeps the running maximum, sum
// and weighted sum of its columns in fp32 and rescales them when a vector of
// 16 bytes brings a larger maximum; thread, warp, block and (for few rows) the
// CTAs of a cluster are then joined by the same rescaling.  Where the maximum
// has most of the probability, log S = log(1 + R), and R, the sum without the
// maximum, would have lost its digits beside the 1: then R is summed apart (the
// columns of the one thread that holds the maximum are read again; 8192 x 50304
// bf16, every row such a one: 143 us where others take 137).  NaN travels in the
// maximum (a NaN-propagating maximum), a row with +inf has no distribution
// (NaN), a row of nothing but -inf has log probability -inf and entropy 0.
//
// Top alternatives (k at most 64) cost no second pass: a thread's maximum and
// the vector that it came from are a key (value, then lowest index); the k-th
// largest of the threads' keys bounds the k-th largest value from below, so only
// the k threads whose own maximum reaches it have their columns read again
// (from L2), and the values that reach it are listed and ranked by counting.  Rows built so that
// the list overflows are done by k searches over the row.
#include "common.cuh"

#include <mutex>

namespace bs {
namespace {

// Threads of a forward CTA.  A thread's join with the others costs as much as
// some 30 columns: 256 threads, each with twice the columns, rather than 512.
constexpr int kThreadsL = 256, kWarpsL = kThreadsL / 32;
constexpr int kMaxTop = 64;
constexpr int kListCap = 1024;
// Differences to the maximum are cut off here: e^z is 0 long before, and 0
// times the cut value is 0, where 0 times -inf (a masked logit) would be NaN.
constexpr float kFloor = -1e20f;
constexpr uint32_t kFloorBf16x2 = 0xE0ADE0ADu;  // -9.97e19, twice
// Below this sum R is summed apart (above it, log S has lost 2 bits at most).
constexpr float kPeaked = 1.5f;
constexpr float kLog2e = 1.44269504088896340736f;

struct LogprobParams {
  const void *x;
  const int64_t *target;
  int64_t rows, V, ld, ignore;
  float rcp_t;            // 1 / temperature
  int top;
  float *logprob, *entropy, *top_lp;
  int64_t *top_ix;
  float *stats;           // [rows][2]: m, log S (natural, of z); for the backward
  int32_t *status;
  // backward
  const float *gl, *gh, *ent;
  // Differences to the maximum are cut off here: p is 0 already, and b times the
  // cut is finite at the smallest temperatures too (b is up to 1e20 then; 0 times
  // an infinite product would be NaN).
  float cut;
  void *dx;
  int64_t ldd;
};

template <class T> struct Vec;  // a 16-byte vector of logits
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float get(const float *p) { return *p; }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ void put(float *p, float f) { *p = f; }
};
template <> struct Vec<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float get(const uint16_t *p) { return bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(bf16x2_from_f32(f[0], f[1]), bf16x2_from_f32(f[2], f[3]),
                      bf16x2_from_f32(f[4], f[5]), bf16x2_from_f32(f[6], f[7]));
  }
  static __device__ __forceinline__ void put(uint16_t *p, float f) {
    *p = (uint16_t)f32_to_bf16_bits(f);
  }
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The largest value (NaN if there is one) of U vectors.
template <int U>
__device__ __forceinline__ float vec_max(const uint4 (&v)[U], const uint16_t *) {
  uint32_t m = v[0].x;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u) m = max_nan_bf16x2(m, v[u].x);
    m = max_nan_bf16x2(m, max_nan_bf16x2(v[u].y, max_nan_bf16x2(v[u].z, v[u].w)));
  }
  return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
}
template <int U>
__device__ __forceinline__ float vec_max(const uint4 (&v)[U], const float *) {
  float m = __uint_as_float(v[0].x);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u) m = max_nan(m, __uint_as_float(v[u].x));
    m = max_nan(m, __uint_as_float(v[u].y));
    m = max_nan(m, max_nan(__uint_as_float(v[u].z), __uint_as_float(v[u].w)));
  }
  return m;
}
// Two values in one instruction (packed fp32).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// The values of a 16-byte vector as pairs, not below kFloor (bf16: clamped two
// at a time before they are widened).
__device__ __forceinline__ void floored(const uint4 &v, float2 (&f)[4], const uint16_t *) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t c;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(w[i]), "r"(kFloorBf16x2));
    f[i] = make_float2(__uint_as_float(c << 16), __uint_as_float(c & 0xFFFF0000u));
  }
}
__device__ __forceinline__ void floored(const uint4 &v, float2 (&f)[2], const float *) {
  f[0] = make_float2(fmaxf(__uint_as_float(v.x), kFloor), fmaxf(__uint_as_float(v.y), kFloor));
  f[1] = make_float2(fmaxf(__uint_as_float(v.z), kFloor), fmaxf(__uint_as_float(v.w), kFloor));
}

// Order of the alternatives: value (NaN above +inf, -0 equal to +0), then the
// lowest index.  The key of a value at column `ix` is larger the better it
// is, and never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u)
                          : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ unsigned long long key_of(float x, int ix) {
  return ((unsigned long long)order_of(x) << 32) | (0xFFFFFFFFu - (uint32_t)ix);
}
__device__ __forceinline__ int64_t index_of(unsigned long long key) {
  return (int64_t)(0xFFFFFFFFu - (uint32_t)key);
}

// Running maximum, sum of e^z and of e^z (x - m); k = log2(e) / temperature.
struct Running {
  float m, S, W;
  // to a larger (or NaN) maximum
  __device__ __forceinline__ void raise(float n, float k) {
    const float d = fmaxf(m - n, kFloor), f = ex2(d * k);
    W = f * fmaf(S, d, W);
    S *= f;
    m = n;
  }
};
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// Joins the first `lanes` lanes of a warp (a power of two).
template <int LANES>
__device__ __forceinline__ void join_warp(Running &a, float k) {
  float n = a.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) n = max_nan(n, __shfl_xor_sync(0xFFFFFFFFu, n, o));
  a.raise(n, k);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    a.S += __shfl_xor_sync(0xFFFFFFFFu, a.S, o);
    a.W += __shfl_xor_sync(0xFFFFFFFFu, a.W, o);
  }
}

// The columns of a segment [c0, c1) of a row, as one thread walks them: at
// most one column before the first 16-byte boundary, vectors kThreadsL apart,
// at most one column after the last whole vector.
template <class T>
struct Walk {
  static constexpr int N = Vec<T>::N;
  const T *row;
  int c0, vec0, nvec, tail0, head, tail;
  __device__ __forceinline__ Walk(const T *r, int a, int b) : row(r), c0(a) {
    const int len = b - a;
    const int skew = (int)((reinterpret_cast<uintptr_t>(r + a) & 15) / sizeof(T));
    const int h = (N - skew) % N;
    head = h < len ? h : len;
    vec0 = a + head;
    nvec = (len - head) / N;
    tail0 = vec0 + nvec * N;
    tail = b - tail0;
  }
  __device__ __forceinline__ int column(int v) const { return vec0 + v * N; }
  __device__ __forceinline__ uint4 load(int v) const {
    return ld_nc_v4(reinterpret_cast<const uint4 *>(row + vec0) + v);
  }
  // f(value, column) of all of thread t's columns
  template <class F>
  __device__ __forceinline__ void each(int t, F f) const {
    if (t < head) f(Vec<T>::get(row + c0 + t), c0 + t);
    for (int v = t; v < nvec; v += kThreadsL) {
      float x[N];
      Vec<T>::unpack(load(v), x);
#pragma unroll
      for (int j = 0; j < N; ++j) f(x[j], column(v) + j);
    }
    if (t < tail) f(Vec<T>::get(row + tail0 + t), tail0 + t);
  }
};

struct LogprobShared {
  float m[kWarpsL], S[kWarpsL], W[kWarpsL];
  Running cta;                                 // read by the cluster's first CTA
  float rest;                                  // cta.S - 1, the same
  unsigned long long group[kWarpsL * 32];
  unsigned long long bound;
  unsigned long long list[kListCap];
  unsigned long long best[kMaxTop];            // this CTA's alternatives, best first
  unsigned long long found;
  int qualify[kThreadsL];
  int nqual, nlist;
};

__device__ __forceinline__ unsigned long long shfl_xor_max(unsigned long long v, int o) {
  const unsigned long long w = __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v > w ? v : w;
}

// sh.best[0 .. top) = the `top` largest keys of sh.list[0 .. n), best first, 0
// where there are fewer.  Keys are distinct; every thread of the block calls.
__device__ __forceinline__ void rank_list(LogprobShared &sh, int n, int top) {
  for (int i = threadIdx.x; i < top; i += kThreadsL) sh.best[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreadsL) {
    const unsigned long long mine = sh.list[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += sh.list[j] > mine;
    if (mine != 0 && above < top) sh.best[above] = mine;
  }
  __syncthreads();
}

// This CTA's `top` best keys of its columns into sh.best; `mine` is the
// thread's best vector's key (0: it has no columns).
template <class T>
__device__ __forceinline__ void find_top(LogprobShared &sh, const Walk<T> &walk,
                                         unsigned long long mine, int top) {
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  // The top-th largest of the threads' keys: each warp sorts its own (largest
  // first), then a key's rank is its place plus what the other warps' lists hold
  // above it, found by halving.
  unsigned long long key = mine;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) {
      const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, key, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
      key = (other > key) == larger ? other : key;
    }
  sh.group[t] = key;
  if (t == 0) {
    sh.nqual = sh.nlist = 0;
    sh.bound = 0;  // fewer than `top` threads have columns: all of them qualify
  }
  __syncthreads();
  // (the first `span` >= min(top, 32) places of a list decide; the lists are
  // searched side by side)
  int span = 1;
  while (span < top && span < 32) span *= 2;
  int above[kWarpsL - 1], place = lane;
#pragma unroll
  for (int w = 0; w < kWarpsL - 1; ++w) above[w] = 0;
  for (int half = span / 2; half > 0; half /= 2)
#pragma unroll
    for (int w = 0; w < kWarpsL - 1; ++w)
      if (sh.group[((warp + w + 1) & (kWarpsL - 1)) * 32 + above[w] + half - 1] > key)
        above[w] += half;
#pragma unroll
  for (int w = 0; w < kWarpsL - 1; ++w)  // above[w] is span - 1 at most here
    place += above[w] +
             (sh.group[((warp + w + 1) & (kWarpsL - 1)) * 32 + above[w]] > key ? 1 : 0);
  if (key != 0 && place == top - 1) sh.bound = key;
  __syncthreads();
  const unsigned long long bound = sh.bound;
  if (mine != 0 && mine >= bound) sh.qualify[atomicAdd(&sh.nqual, 1)] = t;
  __syncthreads();
  const int nqual = sh.nqual;
  auto offer = [&](float x, int ix, int start) {
    if (key_of(x, start) >= bound) {
      const int at = atomicAdd(&sh.nlist, 1);
      if (at < kListCap) sh.list[at] = key_of(x, ix);
    }
  };
  // the qualified threads' columns, spread over all threads: one vector each,
  // and one more place for their columns before and after the vectors
  const int per = (walk.nvec + kThreadsL - 1) / kThreadsL + 1;
  for (int who = 0, i = t; who < nqual; i += kThreadsL) {
    who = i / per;
    if (who >= nqual) break;
    const int q = sh.qualify[who], step = i - who * per;
    if (step == 0) {
      if (q < walk.head)
        offer(Vec<T>::get(walk.row + walk.c0 + q), walk.c0 + q, walk.c0 + q);
      if (q < walk.tail)
        offer(Vec<T>::get(walk.row + walk.tail0 + q), walk.tail0 + q, walk.tail0 + q);
      continue;
    }
    const int v = q + (step - 1) * kThreadsL;
    if (v < walk.nvec) {
      const uint4 raw[1] = {walk.load(v)};
      if (key_of(vec_max<1>(raw, (const T *)nullptr), walk.column(v)) < bound) continue;
      float x[Vec<T>::N];
      Vec<T>::unpack(raw[0], x);
#pragma unroll
      for (int j = 0; j < Vec<T>::N; ++j) offer(x[j], walk.column(v) + j, walk.column(v));
    }
  }
  __syncthreads();
  const int nlist = sh.nlist;
  if (nlist <= kListCap) {
    rank_list(sh, nlist, top);
    return;
  }
  unsigned long long before = ~0ull;
  for (int r = 0; r < top; ++r) {  // the list overflowed: one search for each place
    unsigned long long best = 0;
    walk.each(t, [&](float x, int ix) {
      const unsigned long long k = key_of(x, ix);
      if (k < before && k > best) best = k;
    });
    for (int o = 16; o > 0; o >>= 1) best = shfl_xor_max(best, o);
    if (lane == 0) sh.group[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarpsL; ++w) best = sh.group[w] > best ? sh.group[w] : best;
    if (t == 0) sh.best[r] = best;
    before = best;
    __syncthreads();
  }
}

__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_f32(const float *p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long peer_u64(const unsigned long long *p,
                                                       uint32_t rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(p, rank)) : "memory");
  return v;
}

template <int N>
struct Count {
  static constexpr int value = N;
};

// One row per cluster of C CTAs, each with a segment of its columns.
template <class T, int C, bool TOP>
__global__ void __launch_bounds__(kThreadsL) logprobs_fwd_kernel(const LogprobParams P) {
  __shared__ LogprobShared sh;
  constexpr int N = Vec<T>::N, U = 4;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int64_t row = (int64_t)blockIdx.x / C;
  const uint32_t rank = C > 1 ? ctarank() : 0;
  const int64_t target = P.target[row];
  if (target == P.ignore) {  // the whole cluster leaves
    if (rank == 0) {
      if (t == 0) {
        P.logprob[row] = P.entropy[row] = 0.f;
        if (P.stats) P.stats[2 * row] = P.stats[2 * row + 1] = 0.f;
      }
      if constexpr (TOP)
        for (int i = t; i < P.top; i += kThreadsL) {
          P.top_lp[row * P.top + i] = 0.f;
          P.top_ix[row * P.top + i] = -1;
        }
    }
    return;
  }
  const T *x = static_cast<const T *>(P.x) + row * P.ld;
  const int V = (int)P.V, seg = ((V + C - 1) / C + 63) & ~63;
  const int c0 = min((int)rank * seg, V), c1 = min(c0 + seg, V);
  const Walk<T> walk(x, c0, c1);
  const float k = P.rcp_t * kLog2e;

  Running a = {-INFINITY, 0.f, 0.f};
  int from = -1;  // the first column of the vector that the maximum came from
  if (t < walk.head) from = c0 + t;
  else if (t < walk.nvec) from = walk.column(t);
  else if (t < walk.tail) from = walk.tail0 + t;
  // Sums of pairs; rescaled with a, joined to it at the end.
  float2 S2 = both(0.f), W2 = both(0.f);
  const float2 k2 = both(k);
  auto fold = [&]() {
    a.S += S2.x + S2.y;
    a.W += W2.x + W2.y;
    S2 = W2 = both(0.f);
  };
  auto add = [&](float v) {
    const float d = fmaxf(v - a.m, kFloor), e = ex2(d * k);
    a.S += e;
    a.W = fmaf(e, d, a.W);
  };
  auto single = [&](int c) {
    const float v = Vec<T>::get(x + c);
    if (!(v <= a.m) && a.m == a.m) {  // a NaN maximum stays
      fold();
      a.raise(v, k);
      from = c;
    }
    add(v);
  };
  // U vectors from vector v on, kThreadsL apart
  auto vecs = [&](auto count, int v) {
    constexpr int U = decltype(count)::value;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = walk.load(v + u * kThreadsL);
    const float top = vec_max<U>(raw, (const T *)nullptr);
    if (!(top <= a.m) && a.m == a.m) {
      fold();
      a.raise(top, k);
      if constexpr (TOP) {  // the first vector with this maximum
#pragma unroll
        for (int u = U - 1; u >= 0; --u) {
          const uint4 one[1] = {raw[u]};
          const float m = vec_max<1>(one, (const T *)nullptr);
          if (m == top || m != m) from = walk.column(v + u * kThreadsL);
        }
      }
    }
    if (a.m < 0.01f * kFloor) {  // so far nothing but masked logits: one by one
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        float f[N];
        Vec<T>::unpack(walk.load(v + u * kThreadsL), f);
#pragma unroll
        for (int j = 0; j < N; ++j) add(f[j]);
      }
      return;
    }
    const float2 minus_m = both(-a.m);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 f[N / 2];
      floored(raw[u], f, (const T *)nullptr);
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const float2 d = __fadd2_rn(f[j], minus_m), z = __fmul2_rn(d, k2);
        const float2 e = make_float2(ex2(z.x), ex2(z.y));
        S2 = __fadd2_rn(S2, e);
        W2 = __ffma2_rn(e, d, W2);
      }
    }
  };
  if (t < walk.head) single(c0 + t);
  int v = t;
  for (; v + (U - 1) * kThreadsL < walk.nvec; v += U * kThreadsL) vecs(Count<U>{}, v);
  for (; v < walk.nvec; v += kThreadsL) vecs(Count<1>{}, v);
  if (t < walk.tail) single(walk.tail0 + t);
  fold();

  const unsigned long long mine = from < 0 ? 0ull : key_of(a.m, from);
  const float own_m = a.m, own_S = a.S;
  join_warp<32>(a, k);
  if (lane == 0) {
    sh.m[warp] = a.m;
    sh.S[warp] = a.S;
    sh.W[warp] = a.W;
  }
  __syncthreads();
  if (warp == 0) {
    a = {-INFINITY, 0.f, 0.f};
    if (lane < kWarpsL) a = {sh.m[lane], sh.S[lane], sh.W[lane]};
    join_warp<kWarpsL>(a, k);
    if (lane == 0) sh.cta = a;
  }
  if constexpr (TOP) find_top<T>(sh, walk, mine, P.top);
  __syncthreads();
  a = sh.cta;
  float rest = a.S - 1.f;
  if (a.S >= 1.f && a.S < kPeaked) {  // (of the whole CTA; one column alone has the maximum)
    const uint32_t holder = __ballot_sync(0xFFFFFFFFu, own_m == a.m);
    rest = own_m == a.m ? 0.f : own_S * ex2(fmaxf(own_m - a.m, kFloor) * k);
    if (holder) {  // the lanes of its warp share its columns
      const int q = warp * 32 + __ffs(holder) - 1;
      auto other = [&](float v) {
        if (v != a.m) rest += ex2(fmaxf(v - a.m, kFloor) * k);
      };
      if (lane == 0 && q < walk.head) other(Vec<T>::get(x + c0 + q));
      if (lane == 1 && q < walk.tail) other(Vec<T>::get(x + walk.tail0 + q));
      for (int v = q + lane * kThreadsL; v < walk.nvec; v += 32 * kThreadsL) {
        float f[N];
        Vec<T>::unpack(walk.load(v), f);
#pragma unroll
        for (int j = 0; j < N; ++j) other(f[j]);
      }
    }
    rest = warp_add(rest);
    if (lane == 0) sh.S[warp] = rest;
    __syncthreads();
    rest = 0.f;
#pragma unroll
    for (int w = 0; w < kWarpsL; ++w) rest += sh.S[w];
  }
  if (C > 1 && t == 0) sh.rest = rest;
  if constexpr (C > 1) {
    cluster_barrier();
    if (rank == 0) {
#pragma unroll
      for (uint32_t r = 1; r < C; ++r) {
        Running b = {peer_f32(&sh.cta.m, r), peer_f32(&sh.cta.S, r), peer_f32(&sh.cta.W, r)};
        const float n = max_nan(a.m, b.m), b_rest = peer_f32(&sh.rest, r);
        const bool above = b.m > a.m;
        a.raise(n, k);
        b.raise(n, k);
        rest = above ? b_rest + a.S : rest + b.S;
        a.S += b.S;
        a.W += b.W;
      }
      if constexpr (TOP) {
        for (int i = t; i < C * P.top; i += kThreadsL)
          sh.list[i] = peer_u64(&sh.best[i % P.top], (uint32_t)(i / P.top));
      }
    }
    cluster_barrier();  // the peers' shared memory is read
    if (rank != 0) return;
    if constexpr (TOP) rank_list(sh, C * P.top, P.top);
  }
  const bool dead = a.m == -INFINITY, none = !(a.m < INFINITY);
  const float nan = __uint_as_float(0x7FC00000u);
  const float log_s = none ? nan : log1pf(rest);
  auto logprob = [&](float v) {
    return dead ? -INFINITY : (v - a.m) * P.rcp_t - log_s;
  };
  if (t == 0) {
    float lp = nan;
    if (target >= 0 && target < P.V) lp = logprob(Vec<T>::get(x + target));
    else status_or(P.status, BS_STATUS_INDEX);
    P.logprob[row] = lp;
    P.entropy[row] = dead ? 0.f : log_s - P.rcp_t * (a.W / a.S);
    if (P.stats) {
      P.stats[2 * row] = none ? nan : a.m;
      P.stats[2 * row + 1] = log_s;
    }
  }
  if constexpr (TOP)
    for (int i = t; i < P.top; i += kThreadsL) {
      const unsigned long long key = sh.best[i];
      P.top_lp[row * P.top + i] = logprob(value_of((uint32_t)(key >> 32)));
      P.top_ix[row * P.top + i] = index_of(key);
    }
}

// ---------------------------------------------------------------------------
// Backward: elementwise over the row from m, log S and H, written once.
// ---------------------------------------------------------------------------
constexpr int kThreadsB = 256, kUnrollB = 4;
template <class T>
__global__ void __launch_bounds__(kThreadsB) logprobs_bwd_kernel(const LogprobParams P) {
  constexpr int N = Vec<T>::N;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int64_t target = P.target[row];
  const T *x = static_cast<const T *>(P.x) + row * P.ld;
  T *dx = static_cast<T *>(P.dx) + row * P.ldd;
  const bool none = target == P.ignore || target < 0 || target >= P.V;
  const float gl = none || !P.gl ? 0.f : P.gl[row], gh = none || !P.gh ? 0.f : P.gh[row];
  const float m = P.stats[2 * row], log_s = P.stats[2 * row + 1];
  const bool dead = m == -INFINITY;
  const float k = P.rcp_t * kLog2e, shift = dead ? 0.f : -log_s * kLog2e;
  // d = p (a + b (x - m)), at the target's column + at
  const float ah = none || dead ? 0.f : -P.rcp_t * (gh * (P.ent[row] - log_s));
  const float b = none || dead ? 0.f : -P.rcp_t * P.rcp_t * gh, at = gl * P.rcp_t;
  const float a = none || dead ? 0.f : ah - at;
  // (a row with NaN has m NaN and with it a; so NaN need not be looked for)
  const float a_ = m == m ? a : m;
  // Where p is near 1, at (1 - p) as at - at p would keep the rounding of p
  // alone (1e-3 of it at log p = -2e-5); -expm1(log p) has the digits of 1 - p.
  // (Only there: few rows wait for it.)  One thread of a row comes here.
  auto at_target = [&]() {
    if (none || dead) return none ? 0.f : at;
    const float d = fmaxf(Vec<T>::get(x + target) - m, P.cut), p = ex2(fmaf(d, k, shift));
    const float logprob = fmaf(d, P.rcp_t, -log_s);
    return fmaf(at, logprob > -0.5f ? -expm1f(logprob) : 1.f - p, p * fmaf(b, d, ah));
  };
  auto grad = [&](float v, int c) {
    const float d = fmaxf(v - m, P.cut);
    if (c == target) return at_target();
    return none || dead ? 0.f : ex2(fmaf(d, k, shift)) * fmaf(b, d, a_);
  };
  const float2 minus_m = both(-m), k2 = both(k), shift2 = both(shift), a2 = both(a_), b2 = both(b);
  const int V = (int)P.V;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool same = (reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(dx) & 15);
  const int head = same ? min((N - skew) % N, V) : V;  // vectors start here
  const int nvec = (V - head) / N, tail0 = head + nvec * N;
  // columns outside the vectors (all of them where x and dx are not aligned alike)
  const int y0 = (int)blockIdx.y * kThreadsB + t, dy = (int)gridDim.y * kThreadsB;
  for (int c = y0; c < head; c += dy) Vec<T>::put(dx + c, grad(Vec<T>::get(x + c), c));
  for (int c = tail0 + y0; c < V; c += dy) Vec<T>::put(dx + c, grad(Vec<T>::get(x + c), c));
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
  uint4 *dv = reinterpret_cast<uint4 *>(dx + head);
  const bool zero = none || dead;
  const int at_vec = target >= head && target < tail0 ? ((int)target - head) / N : -1;
  const int at_pos = at_vec >= 0 ? (int)target - head - at_vec * N : 0;
  auto one = [&](const uint4 &raw, int v) {
    float f[N];
    Vec<T>::unpack(raw, f);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float2 d = __fadd2_rn(make_float2(f[j], f[j + 1]), minus_m);
      d = make_float2(fmaxf(d.x, P.cut), fmaxf(d.y, P.cut));
      const float2 z = __ffma2_rn(d, k2, shift2);
      const float2 g = __fmul2_rn(make_float2(ex2(z.x), ex2(z.y)), __ffma2_rn(b2, d, a2));
      f[j] = zero ? 0.f : g.x;
      f[j + 1] = zero ? 0.f : g.y;
    }
    if (v == at_vec) {
      const float own = at_target();
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j == at_pos) f[j] = own;
    }
    st_v4(dv + v, Vec<T>::pack(f));
  };
  if (none) {  // an ignored row is not read
    for (int v = y0; v < nvec; v += dy) st_v4(dv + v, make_uint4(0, 0, 0, 0));
    return;
  }
  int v = y0;
  for (; v + (kUnrollB - 1) * dy < nvec; v += kUnrollB * dy) {
    uint4 raw[kUnrollB];
#pragma unroll
    for (int u = 0; u < kUnrollB; ++u) raw[u] = ld_nc_v4(xv + v + u * dy);
#pragma unroll
    for (int u = 0; u < kUnrollB; ++u) one(raw[u], v + u * dy);
  }
  for (; v < nvec; v += dy) one(ld_nc_v4(xv + v), v);
}

template <class T, int C>
int launch_fwd(const LogprobParams &P, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(P.rows * C));
  cfg.blockDim = dim3(kThreadsL);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  const cudaError_t e = P.top ? cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, C, true>, P)
                              : cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, C, false>, P);
  return launch_code(e);
}
// Few rows are divided among the CTAs of a cluster, as long as all CTAs find
// an SM and each has some thousand columns.
template <class T>
int fwd_clustered(const LogprobParams &P, cudaStream_t st) {
  if (P.rows <= 18 && P.V >= 16384) return launch_fwd<T, 8>(P, st);
  if (P.rows <= 37 && P.V >= 8192) return launch_fwd<T, 4>(P, st);
  if (P.rows <= 74 && P.V >= 4096) return launch_fwd<T, 2>(P, st);
  return launch_fwd<T, 1>(P, st);
}

int logprob_checks(int dtype, int64_t rows, int64_t V, int64_t ld, const void *x,
                   const void *target, float temperature) {
  if (rows < 0 || V <= 0 || ld < V) return BS_ERR_SHAPE;
  if (rows >= ((int64_t)1 << 28) || V >= ((int64_t)1 << 31) - (1 << 20)) return BS_ERR_TOO_LARGE;
  if (dtype != BS_BF16 && dtype != BS_F32) return BS_ERR_DTYPE;
  if (rows == 0) return BS_OK;
  if (!x || !target || !(temperature > 0.f) || temperature > 1e10f || temperature < 1e-10f)
    return BS_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(x) & (dtype == BS_F32 ? 3 : 1)) ||
      (reinterpret_cast<uintptr_t>(target) & 7))
    return BS_ERR_ALIGN;
  return BS_OK;
}

}  // namespace
}  // namespace bs

using namespace bs;

extern "C" int bs_token_logprobs(const void *logits, int dtype, int64_t rows, int64_t V,
                                 int64_t ld, const int64_t *targets, int64_t ignore_index,
                                 float temperature, int top, float *logprobs, float *entropy,
                                 float *top_logprobs, int64_t *top_indices, float *stats,
                                 int32_t *status, void *stream) {
  const int rc = logprob_checks(dtype, rows, V, ld, logits, targets, temperature);
  if (rc != BS_OK) return rc;
  if (top < 0 || top > kMaxTop || top > V) return BS_ERR_ARG;
  if (rows == 0) return BS_OK;
  if (!logprobs || !entropy || (top && (!top_logprobs || !top_indices))) return BS_ERR_ARG;
  LogprobParams P = {};
  P.x = logits; P.target = targets; P.rows = rows; P.V = V; P.ld = ld; P.ignore = ignore_index;
  P.rcp_t = 1.f / temperature; P.top = top; P.logprob = logprobs; P.entropy = entropy;
  P.top_lp = top_logprobs; P.top_ix = top_indices; P.stats = stats; P.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BS_F32 ? fwd_clustered<float>(P, st) : fwd_clustered<uint16_t>(P, st);
}

extern "C" int bs_token_logprobs_backward(const void *logits, int dtype, int64_t rows, int64_t V,
                                          int64_t ld, const int64_t *targets,
                                          int64_t ignore_index, float temperature,
                                          const float *stats, const float *entropy,
                                          const float *d_logprobs, const float *d_entropy,
                                          void *d_logits, int64_t ldd, void *stream) {
  const int rc = logprob_checks(dtype, rows, V, ld, logits, targets, temperature);
  if (rc != BS_OK) return rc;
  if (ldd < V) return BS_ERR_SHAPE;
  if (rows == 0) return BS_OK;
  if (!stats || !entropy || !d_logits) return BS_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(d_logits) & (dtype == BS_F32 ? 3 : 1)) return BS_ERR_ALIGN;
  LogprobParams P = {};
  P.x = logits; P.target = targets; P.rows = rows; P.V = V; P.ld = ld; P.ignore = ignore_index;
  P.rcp_t = 1.f / temperature; P.stats = const_cast<float *>(stats); P.ent = entropy;
  P.cut = -256.f / (P.rcp_t * kLog2e);
  P.gl = d_logprobs; P.gh = d_entropy; P.dx = d_logits; P.ldd = ldd;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a CTA a row (its columns' sums of indices are paid once a row), several
  // where there are too few rows to fill the SMs eight CTAs deep
  const int64_t span = (int64_t)kThreadsB * kUnrollB * (dtype == BS_F32 ? 4 : 8);
  int64_t blocks = (8 * 148 + rows - 1) / rows;
  const int64_t most = (V + span - 1) / span;
  if (blocks > most) blocks = most;
  if (blocks > 1024) blocks = 1024;
  const dim3 grid((unsigned)rows, (unsigned)blocks);
  if (dtype == BS_F32) logprobs_bwd_kernel<float><<<grid, kThreadsB, 0, st>>>(P);
  else logprobs_bwd_kernel<uint16_t><<<grid, kThreadsB, 0, st>>>(P);
  return launch_code(cudaGetLastError());
}
