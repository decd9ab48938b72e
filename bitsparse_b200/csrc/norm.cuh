// Residual join and RMSNorm around a block, forward and backward.
//
//   u = post ? y * ry * w_post : y          ry = 1 / sqrt(mean(y^2) + eps)
//   s = skip * x + branch * act(g) * u      (the new residual stream)
//   h = s * r * w                           r  = 1 / sqrt(mean(s^2) + eps)
//
// x and s are the residual stream [T, D] (fp32 or bf16), y and h the block's
// output and the next block's input, g an optional gate with one row for
// every `gate_rows` rows, D columns wide or one.  All arithmetic and both
// statistics are fp32; each output is rounded once (h from the unrounded s).
//
// Backward, from ds, dh, ry, r and the saved s -- or x and y, where a norm or a
// gate on the branch needs y anyway: s is then formed again in fp32, free of
// its rounding, for the same bytes.  One pass over them:
//   xh = s r,  A = ds + r dh w,  S1 = sum dh w xh,  d = A - r (S1 / D) xh
//   dx = skip d,  dz = branch d,  dg = dz u act'(g),  du = dz act(g)
//   dw = sum_rows dh xh,  dw_post = sum_rows du n,  n = y ry
//   dy = post ? ry (du w_post - n mean(du w_post n)) : du
// The last mean needs d, hence S1; since d is linear in S1 it comes from two
// sums taken in the same reduction, S2 = sum q A and S3 = sum q xh with
// q = act(g) w_post n:  sum du w_post n = branch (S2 - r S1 / D S3).  So a
// row costs one block reduction.  The parameter gradients are sums over rows:
// each CTA walks a run of rows with its column sums in registers and writes
// them once; a second kernel adds the CTAs' sums in a fixed order (no
// atomics: the same inputs give the same bits).
#pragma once
#include "common.cuh"

#include <mutex>
#include <type_traits>

namespace bs {

struct NormParams {
  const void *x, *y, *gate, *w, *pw;
  void *s, *h;                 // forward outputs; backward: s (see the entry point) is read
  const void *ds, *dh;         // backward inputs (either may be null: zero)
  void *dx, *dy, *dgate;       // backward outputs (null: not wanted)
  float *r_post, *r_pre;       // [T]
  float *part;                 // column sums: [3][chunks][D] (w, post w, gate)
  float *row_gate;             // [T] gate sums of rows, for a one-column gate of many rows
  int64_t T, ldx, ldy, lds, gate_rows;
  // how the backward divides its rows: groups of `div_rows` (see divide())
  int64_t div_rows, chunks, chunk_rows, chunks_per_group, groups_per_chunk;
  int D, post, w_dt, pw_dt, gate_dt, gate_wide, act;
  float skip, branch, eps, rcp_d;
  int stages;                  // of the staged backward
  int32_t *status;
};

// The staged backward.  How many of its CTAs stay resident decides how the
// rows are divided, and that the workspace's size: both ask plan_bwd().
struct BwdPlan {
  bool staged;
  int mode, threads, stages;
  size_t smem;
  int64_t ctas;
};

namespace {

enum { kActNone = 0, kActSigmoid = 1 };
constexpr int kMaxStages = 4;
constexpr size_t kStagedSmem = 216 * 1024;  // of an SM, for the staged rows


__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_bits_to_f32(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t from_f32<uint16_t>(float v) {
  return (uint16_t)f32_to_bf16_bits(v);
}

// Columns of a thread's value j of vector v.  Vector form: eight neighbouring
// columns (16 or 32 bytes); scalar form (odd widths, unaligned rows): columns
// TPR apart, so that a warp's loads are neighbours.
template <bool VEC>
__device__ __forceinline__ int column(int v, int j, int t, int tpr) {
  return VEC ? (v * tpr + t) * 8 + j : (v * 8 + j) * tpr + t;
}

__device__ __forceinline__ void load_vec(float (&f)[8], const float *p) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  const float4 b = *reinterpret_cast<const float4 *>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load_vec(float (&f)[8], const uint16_t *p) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store_vec(float *p, const float (&f)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store_vec(uint16_t *p, const float (&f)[8]) {
  *reinterpret_cast<uint4 *>(p) =
      make_uint4(bf16x2_from_f32(f[0], f[1]), bf16x2_from_f32(f[2], f[3]),
                 bf16x2_from_f32(f[4], f[5]), bf16x2_from_f32(f[6], f[7]));
}

// Vector v of this thread of a row (zeros past D).
template <bool VEC, class T>
__device__ __forceinline__ void load8(float (&f)[8], const T *row, int v, int t, int tpr, int D) {
  if constexpr (VEC) {
    const int c = column<true>(v, 0, t, tpr);
    if (c < D) {
      load_vec(f, row + c);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else {
    const T *mine = row + t;  // column(): t + (8 v + j) tpr
    const int rest = D - t;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = (v * 8 + j) * tpr < rest ? to_f32(mine[(v * 8 + j) * tpr]) : 0.f;
  }
}
__device__ __forceinline__ void put_scalar(float *mine, const float (&f)[8], int v, int tpr,
                                           int rest) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((v * 8 + j) * tpr < rest) mine[(v * 8 + j) * tpr] = f[j];
}
__device__ __forceinline__ void put_scalar(uint16_t *mine, const float (&f)[8], int v, int tpr,
                                           int rest) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint32_t w = bf16x2_from_f32(f[j], f[j + 1]);
    if ((v * 8 + j) * tpr < rest) mine[(v * 8 + j) * tpr] = (uint16_t)w;
    if ((v * 8 + j + 1) * tpr < rest) mine[(v * 8 + j + 1) * tpr] = (uint16_t)(w >> 16);
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T *row, const float (&f)[8], int v, int t, int tpr, int D) {
  if constexpr (VEC) {
    const int c = column<true>(v, 0, t, tpr);
    if (c < D) store_vec(row + c, f);
  } else {
    T *mine = row + t;
    const int rest = D - t;
    put_scalar(mine, f, v, tpr, rest);
  }
}
// The same for a parameter, whose type is a launch argument (bf16 or fp32).
template <bool VEC>
__device__ __forceinline__ void load_param(float (&f)[8], const void *p, int dt, int64_t at, int v,
                                           int t, int tpr, int D) {
  if (dt == BS_F32) load8<VEC>(f, static_cast<const float *>(p) + at, v, t, tpr, D);
  else load8<VEC>(f, static_cast<const uint16_t *>(p) + at, v, t, tpr, D);
}
template <bool VEC>
__device__ __forceinline__ void store_param(void *p, const float (&f)[8], int dt, int64_t at,
                                            int v, int t, int tpr, int D) {
  if (dt == BS_F32) store8<VEC>(static_cast<float *>(p) + at, f, v, t, tpr, D);
  else store8<VEC>(static_cast<uint16_t *>(p) + at, f, v, t, tpr, D);
}
__device__ __forceinline__ float load_one(const void *p, int dt, int64_t at) {
  return dt == BS_F32 ? static_cast<const float *>(p)[at]
                      : to_f32(static_cast<const uint16_t *>(p)[at]);
}
__device__ __forceinline__ void store_one(void *p, int dt, int64_t at, float v) {
  if (dt == BS_F32) static_cast<float *>(p)[at] = v;
  else static_cast<uint16_t *>(p)[at] = from_f32<uint16_t>(v);
}

// The sigmoid by the hardware's 2^x and reciprocal: within 2^-21 (1 + |g|) of
// its value, at a sixth of the instructions of expf and a division.
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act != kActSigmoid) return g;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}
__device__ __forceinline__ float gate_slope(float a, int act) {
  return act == kActSigmoid ? a * (1.f - a) : 1.f;
}

// Two values in one instruction (the packed fp32 forms; each value is rounded
// as by the scalar instruction).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 gate_act(float2 g, int act) {
  return make_float2(gate_act(g.x, act), gate_act(g.y, act));
}
__device__ __forceinline__ float2 gate_slope(float2 a, int act) {
  return act == kActSigmoid ? fma2(make_float2(-a.x, -a.y), a, a) : both(1.f);
}
// Eight values as pairs.
template <bool VEC, class T>
__device__ __forceinline__ void load8(float2 (&f)[4], const T *row, int v, int t, int tpr, int D) {
  float s[8];
  load8<VEC>(s, row, v, t, tpr, D);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(s[2 * i], s[2 * i + 1]);
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T *row, const float2 (&f)[4], int v, int t, int tpr, int D) {
  const float s[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
  store8<VEC>(row, s, v, t, tpr, D);
}
template <bool VEC>
__device__ __forceinline__ void load_param(float2 (&f)[4], const void *p, int dt, int64_t at, int v,
                                           int t, int tpr, int D) {
  if (dt == BS_F32) load8<VEC>(f, static_cast<const float *>(p) + at, v, t, tpr, D);
  else load8<VEC>(f, static_cast<const uint16_t *>(p) + at, v, t, tpr, D);
}
template <bool VEC>
__device__ __forceinline__ void store_param(void *p, const float2 (&f)[4], int dt, int64_t at,
                                            int v, int t, int tpr, int D) {
  if (dt == BS_F32) store8<VEC>(static_cast<float *>(p) + at, f, v, t, tpr, D);
  else store8<VEC>(static_cast<uint16_t *>(p) + at, f, v, t, tpr, D);
}

// Row of the gate that row `row` of y has (32-bit: rows are fewer than 2^31).
__device__ __forceinline__ int64_t gate_row(int64_t row, int64_t gate_rows) {
  return gate_rows == 1 ? row : (int64_t)((uint32_t)row / (uint32_t)gate_rows);
}

// Sums of N values over the threads of a row, given to all of them.  A row is
// one warp, or the whole block: then the warps' sums go through shared memory,
// in one of two alternating buffers so that a reduction costs one barrier (a
// buffer is written again only after the next reduction's barrier, which
// every thread reaches after its reads).
template <int N, bool BLOCK>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buf)[N][32], int &turn) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
  if constexpr (BLOCK) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float(*b)[32] = buf[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) b[i][warp] = v[i];
    __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = lane < warps ? b[i][lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      v[i] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// Forward: a row per warp (BLOCK false, four rows a CTA) or per CTA, its
// NV * 8 values a thread in registers.
// ---------------------------------------------------------------------------
template <class TX, class TY, int NV, bool VEC, bool BLOCK, bool POST, bool GATE>
__global__ void __launch_bounds__(BLOCK ? 512 : 128, BLOCK && NV <= 2 ? 2 : 1) norm_fwd_kernel(const NormParams P) {
  __shared__ float buf[2][1][32];
  int turn = 0;
  const int tpr = BLOCK ? blockDim.x : 32;
  const int t = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int64_t row = BLOCK ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= P.T) return;  // whole warps, and no block reduction with BLOCK false
  const TX *x = static_cast<const TX *>(P.x) + row * P.ldx;
  float2 xs[NV][4], z[NV][4];
#pragma unroll
  for (int v = 0; v < NV; ++v) load8<VEC>(xs[v], x, v, t, tpr, P.D);
  if (P.y) {
    const TY *y = static_cast<const TY *>(P.y) + row * P.ldy;
#pragma unroll
    for (int v = 0; v < NV; ++v) load8<VEC>(z[v], y, v, t, tpr, P.D);
    float2 ga[GATE ? NV : 1][4];
    float a1 = 1.f;
    if constexpr (GATE) {  // with the others, ahead of the first reduction
      const int64_t g = gate_row(row, P.gate_rows);
      if (P.gate_wide) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          load_param<VEC>(ga[v], P.gate, P.gate_dt, g * P.D, v, t, tpr, P.D);
      } else {
        a1 = gate_act(load_one(P.gate, P.gate_dt, g), P.act);
      }
    }
    float2 scale = both(P.branch);  // of the branch: with a norm or one gate of the row
    if constexpr (POST) {
      float2 sq = both(0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) sq = fma2(z[v][i], z[v][i], sq);
      float sum[1] = {sq.x + sq.y};
      row_sums<1, BLOCK>(sum, buf, turn);
      const float r = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
      if (P.r_post && t == 0) P.r_post[row] = r;
      scale = both(P.branch * r);
      if (P.pw) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float2 pw[4];
          load_param<VEC>(pw, P.pw, P.pw_dt, 0, v, t, tpr, P.D);
#pragma unroll
          for (int i = 0; i < 4; ++i) z[v][i] = mul(z[v][i], pw[i]);
        }
      }
    }
    if constexpr (GATE) {
      if (P.gate_wide) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[v][i] = mul(z[v][i], gate_act(ga[v][i], P.act));
      } else {
        scale = both(scale.x * a1);
      }
    }
    const float2 skip = both(P.skip);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) xs[v][i] = fma2(scale, z[v][i], mul(skip, xs[v][i]));
  }
  float2 sq = both(0.f);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (P.s) store8<VEC>(static_cast<TX *>(P.s) + row * P.D, xs[v], v, t, tpr, P.D);
#pragma unroll
    for (int i = 0; i < 4; ++i) sq = fma2(xs[v][i], xs[v][i], sq);
  }
  float sum[1] = {sq.x + sq.y};
  row_sums<1, BLOCK>(sum, buf, turn);
  const float r = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
  if (P.r_pre && t == 0) P.r_pre[row] = r;
  TY *h = static_cast<TY *>(P.h) + row * P.D;
  const float2 r2 = both(r);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float2 w[4];
    if (P.w) load_param<VEC>(w, P.w, P.w_dt, 0, v, t, tpr, P.D);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      xs[v][i] = P.w ? mul(mul(xs[v][i], r2), w[i]) : mul(xs[v][i], r2);
    store8<VEC>(h, xs[v], v, t, tpr, P.D);
  }
}

// Eight values of a row in shared memory, as stored.
template <class TY> struct Raw8 { uint4 a; };
template <> struct Raw8<float> { uint4 a, b; };
__device__ __forceinline__ void get_raw(Raw8<uint16_t> &r, const uint8_t *p) {
  r.a = *reinterpret_cast<const uint4 *>(p);
}
__device__ __forceinline__ void get_raw(Raw8<float> &r, const uint8_t *p) {
  r.a = *reinterpret_cast<const uint4 *>(p);
  r.b = *reinterpret_cast<const uint4 *>(p + 16);
}
__device__ __forceinline__ void set_raw(Raw8<uint16_t> &r, const uint32_t (&e)[8]) {
  r.a = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}
__device__ __forceinline__ void set_raw(Raw8<float> &r, const uint32_t (&e)[8]) {
  r.a = make_uint4(e[0], e[1], e[2], e[3]);
  r.b = make_uint4(e[4], e[5], e[6], e[7]);
}
__device__ __forceinline__ float2 pair(const Raw8<uint16_t> &r, int i) {
  const uint32_t w = i == 0 ? r.a.x : i == 1 ? r.a.y : i == 2 ? r.a.z : r.a.w;
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 pair(const Raw8<float> &r, int i) {
  const uint4 &v = i < 2 ? r.a : r.b;
  return i & 1 ? make_float2(__uint_as_float(v.z), __uint_as_float(v.w))
               : make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}

// How the staged rows lie:
//   kRowsAligned  every row starts on 16 bytes and D is a multiple of 8;
//   kRowsShifted  contiguous tensors on 16 bytes, any D: row r starts e = r D mod
//                 8 elements into a block of 8 that is aligned in every one of
//                 them, fp32 or bf16.  A CTA takes rows of one r mod 8, so e is
//                 its own: its threads have whole blocks, read and written by
//                 vectors, the first and last of a row with a part masked;
//   kRowsAny      any stride and base: single elements, columns TPR apart.
// (16384 x 1219 bf16 with a norm and an element gate, forward + backward: 98 +
// 352 us by single elements, 64 + 227 shifted; 1216 columns, aligned, 49 + 101.)
enum { kRowsAligned = 0, kRowsShifted = 1, kRowsAny = 2 };

// Forms of the staged kernels by the row's width: 1 (a warp a row, up to 256
// columns), 2 (up to 4096) and 4 (up to 8192) have one, two and two vectors of
// eight columns a thread, the last with up to 512 threads.
__host__ __device__ constexpr int vectors(int W) { return W == 1 ? 1 : 2; }

template <class T> struct Bits { using type = uint16_t; };
template <> struct Bits<float> { using type = uint32_t; };

// A thread's columns: first + 0..7 of vector v (kRowsAny: see column()).
struct Cols {
  int t, tpr, D, e;
  __device__ __forceinline__ int first(int v) const { return (v * tpr + t) * 8 - e; }
};

// The thread's vector v of a row in shared memory (`row`: its block or element
// 0), zeros outside the row.
template <int MODE, class T>
__device__ __forceinline__ void take(Raw8<T> &r, const uint8_t *row, int v, const Cols &c) {
  using E = typename Bits<T>::type;
  if constexpr (MODE == kRowsAny) {
    const E *mine = reinterpret_cast<const E *>(row) + c.t;
    const int rest = c.D - c.t;
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      e[j] = (v * 8 + j) * c.tpr < rest ? mine[(v * 8 + j) * c.tpr] : 0;
    set_raw(r, e);
  } else {
    const int first = c.first(v);
    r = {};
    if (first >= c.D) return;
    get_raw(r, row + (first + c.e) * (int)sizeof(T));
    if (MODE == kRowsShifted && (first < 0 || first + 8 > c.D)) {
      uint32_t e[8];
      const E *mine = reinterpret_cast<const E *>(row) + first + c.e;
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = first + j >= 0 && first + j < c.D ? mine[j] : 0;
      set_raw(r, e);
    }
  }
}
// The thread's vector v of a row of memory, and the other way.
template <int MODE, class T>
__device__ __forceinline__ void get8(float2 (&f)[4], const T *row, int v, const Cols &c) {
  if constexpr (MODE == kRowsShifted) {
    const int first = c.first(v);
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      s[j] = first + j >= 0 && first + j < c.D ? to_f32(row[first + j]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(s[2 * i], s[2 * i + 1]);
  } else {
    load8<MODE == kRowsAligned>(f, row, v, c.t, c.tpr, c.D);
  }
}
// (ALIGNED: the row's block lies on 16 bytes)
template <int MODE, bool ALIGNED, class T>
__device__ __forceinline__ void put8(T *row, const float2 (&f)[4], int v, const Cols &c) {
  if constexpr (MODE == kRowsShifted) {
    const int first = c.first(v);
    const float s[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
    if (ALIGNED && first >= 0 && first + 8 <= c.D) {
      store_vec(row + first, s);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (first + j >= 0 && first + j < c.D) row[first + j] = from_f32<T>(s[j]);
    }
  } else {
    store8<MODE == kRowsAligned>(row, f, v, c.t, c.tpr, c.D);
  }
}
template <int MODE>
__device__ __forceinline__ void get_param(float2 (&f)[4], const void *p, int dt, int64_t at, int v,
                                          const Cols &c) {
  if (dt == BS_F32) get8<MODE>(f, static_cast<const float *>(p) + at, v, c);
  else get8<MODE>(f, static_cast<const uint16_t *>(p) + at, v, c);
}
template <int MODE>
__device__ __forceinline__ void put_param(void *p, const float2 (&f)[4], int dt, int64_t at, int v,
                                          const Cols &c) {
  if (dt == BS_F32) put8<MODE, false>(static_cast<float *>(p) + at, f, v, c);
  else put8<MODE, false>(static_cast<uint16_t *>(p) + at, f, v, c);
}

// Parameters of rows that are not aligned: in shared memory as fp32, in the
// order of the threads' vectors, zero outside the row.
template <int MODE>
__device__ __forceinline__ void keep_param(float *to, const void *p, int dt, const Cols &c, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int col = MODE == kRowsShifted ? i - c.e : i;
    to[i] = col >= 0 && col < c.D ? load_one(p, dt, col) : 0.f;
  }
}
template <int MODE>
__device__ __forceinline__ void take_param(float2 (&f)[4], const float *kept, const void *p, int dt,
                                           int v, const Cols &c) {
  if constexpr (MODE == kRowsShifted) {
    float s[8];
    load_vec(s, kept + (v * c.tpr + c.t) * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(s[2 * i], s[2 * i + 1]);
  } else if constexpr (MODE == kRowsAny) {
    const float *mine = kept + c.t;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = make_float2(mine[(v * 8 + 2 * i) * c.tpr], mine[(v * 8 + 2 * i + 1) * c.tpr]);
  } else {
    load_param<true>(f, p, dt, 0, v, c.t, c.tpr, c.D);
  }
}

// A tensor whose rows are staged, and what of a row a bulk copy brings: the row,
// or the 16-byte blocks (kRowsShifted: blocks of 8 elements) that hold it, but
// none that reaches outside the tensor (a few elements of its first and last
// rows, which the block's threads then fetch).  The row lies `off` bytes into
// its place.
struct Staged {
  const uint8_t *base;  // null: not staged
  int64_t stride;       // bytes from row to row
  uint32_t size, bytes; // of an element, of a row
};
struct Span {
  uint32_t off, lo, n;  // the copy covers [lo, lo + n) of the row's place
};
template <int MODE>
__host__ __device__ __forceinline__ uint32_t stage_bytes(uint32_t D, uint32_t size) {
  if (MODE == kRowsAligned) return D * size;
  if (MODE == kRowsShifted) return (D + 14) / 8 * 8 * size;
  return ((D * size + 15) & ~15u) + 16;
}
template <int MODE>
__device__ __forceinline__ Span span_of(const Staged &a, int64_t row, int64_t rows, int e) {
  if constexpr (MODE == kRowsAligned) return {0, 0, a.bytes};
  const uint8_t *at = a.base + row * a.stride;
  const uint32_t off = MODE == kRowsShifted
                           ? (uint32_t)e * a.size
                           : (uint32_t)(reinterpret_cast<uintptr_t>(at) & 15);
  const uint32_t end = off + a.bytes;
  const uint32_t lo = at - off < a.base ? 16 : 0;
  const bool past = at + ((end + 15) & ~15u) - off > a.base + (rows - 1) * a.stride + a.bytes;
  const uint32_t hi = past ? end & ~15u : (end + 15) & ~15u;
  return {off, lo, hi > lo ? hi - lo : 0};
}
template <int MODE>
__device__ __forceinline__ void copy_row(uint8_t *to, const Staged &a, int64_t row, int64_t rows,
                                         int e, uint64_t *bar) {
  const Span s = span_of<MODE>(a, row, rows, e);
  if (s.n) bulk_load(to + s.lo, a.base + row * a.stride - s.off + s.lo, s.n, bar);
}
// The elements that the copy left out.
template <int MODE>
__device__ __forceinline__ void copy_rest(uint8_t *to, const Staged &a, int64_t row, int64_t rows,
                                          int e) {
  const Span s = span_of<MODE>(a, row, rows, e);
  const uint8_t *from = a.base + row * a.stride - s.off;
  for (uint32_t p = s.off + threadIdx.x * a.size; p < s.off + a.bytes; p += blockDim.x * a.size)
    if (p < s.lo || p >= s.lo + s.n) {
      if (a.size == 2)
        *reinterpret_cast<uint16_t *>(to + p) = *reinterpret_cast<const uint16_t *>(from + p);
      else
        *reinterpret_cast<uint32_t *>(to + p) = *reinterpret_cast<const uint32_t *>(from + p);
    }
}
// Thread 0, where its wait for row `k` of `rows` gave up: the copies of that row
// and of those requested after it are waited for (with the same limit), so that
// none lands after the CTA has left.  (The row waits in shared memory: a register
// for it cost the backward with sigmoid gates 5 to 10 %, 16384 x 4096 bf16 214 ->
// 224 us, on an fp32 stream 370 -> 408.)
__device__ __forceinline__ void drain(uint64_t *full, int k, int rows, int stages) {
  const int end = k + stages < rows ? k + stages : rows;
  for (; k < end; ++k)
    for (uint32_t n = 0; n < kMaxPolls; ++n)
      if (mbar_try_wait(&full[k % stages], (uint32_t)(k / stages) & 1)) break;
}
// Rows near enough to a tensor's ends for that (16 bytes are 8 elements at most).
__device__ __forceinline__ bool near_end(int64_t row, int64_t rows) {
  return row < 8 || row >= rows - 8;
}

// A thread's part of a parameter.  Of type T (void: of either type) it is fetched
// before a reduction, whose wait hides the load.
template <int MODE, int NV, class T>
struct RowParam {
  const void *p;
  const float *kept;
  const int dt;
  Raw8<T> raw[NV];
  __device__ __forceinline__ void fetch(const Cols &c) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      raw[v] = {};  // of a thread past the row's end: its zeros are multiplied by this
      if (p && c.first(v) < c.D)
        get_raw(raw[v], static_cast<const uint8_t *>(p) + c.first(v) * (int)sizeof(T));
    }
  }
  __device__ __forceinline__ void take(float2 (&f)[4], int v, const Cols &) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair(raw[v], i);
  }
};
template <int MODE, int NV>
struct RowParam<MODE, NV, void> {
  const void *p;
  const float *kept;
  const int dt;
  __device__ __forceinline__ void fetch(const Cols &) {}
  __device__ __forceinline__ void take(float2 (&f)[4], int v, const Cols &c) const {
    take_param<MODE>(f, kept, p, dt, v, c);
  }
};

// Forward of many wide rows that can be read by vectors: persistent CTAs, whole
// rows of x, y (and an element gate) arriving in shared memory by bulk copies
// P.stages rows ahead.  One row a CTA and no look-ahead, as above, leaves the
// memory idle through a row's two reductions: 16 x 1024 x 4096 with norm and
// sigmoid gate took 159 us, 4.2 TB/s; this form takes 112, 6.0 TB/s (125 with
// the parameters read after the reductions and a stage refilled after the second).
// GATE: 0 none, 1 an element each, 2 anything else (read directly).
// TW: the parameters' type, where both have one and the rows are aligned, else void.
template <class TX, class TY, class TG, int W, bool POST, int GATE, int MODE, class TW>
__global__ void __launch_bounds__(W == 4 ? 512 : 256, W == 4 ? 1 : 3)
    norm_fwd_staged_kernel(const NormParams P) {
  constexpr int NV = vectors(W);
  constexpr bool NARROW = std::is_same<TW, uint16_t>::value;
  // (fp32 before the first reduction, beside x, y and the gate, has no registers)
  using TPW = typename std::conditional<NARROW, uint16_t, void>::type;
  extern __shared__ uint8_t dyn[];
  __shared__ float buf[2][1][32];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int lost_row;  // of thread 0, if its wait gave up
  int turn = 0;
  const int tpr = blockDim.x, t = threadIdx.x, D = P.D;
  const int rows = (int)((P.T - blockIdx.x + gridDim.x - 1) / gridDim.x);
  // (kRowsShifted: the grid is a multiple of 8)
  const int e = MODE == kRowsShifted ? (int)((int64_t)blockIdx.x * D & 7) : 0;
  const Cols cols = {t, tpr, D, e};
  const Staged ax = {static_cast<const uint8_t *>(P.x), P.ldx * (int64_t)sizeof(TX), sizeof(TX),
                     (uint32_t)D * (uint32_t)sizeof(TX)};
  const Staged ay = {static_cast<const uint8_t *>(P.y), P.ldy * (int64_t)sizeof(TY), sizeof(TY),
                     (uint32_t)D * (uint32_t)sizeof(TY)};
  const Staged ag = {static_cast<const uint8_t *>(P.gate), D * (int64_t)sizeof(TG), sizeof(TG),
                     (uint32_t)D * (uint32_t)sizeof(TG)};
  const uint32_t bx = stage_bytes<MODE>(D, sizeof(TX)), by = stage_bytes<MODE>(D, sizeof(TY));
  const uint32_t bytes = bx + by + (GATE == 1 ? stage_bytes<MODE>(D, sizeof(TG)) : 0);
  float *kept_w = reinterpret_cast<float *>(dyn + (size_t)P.stages * bytes);
  float *kept_pw = kept_w + (P.w ? NV * 8 * tpr : 0);
  if constexpr (MODE != kRowsAligned) {
    if (P.w) keep_param<MODE>(kept_w, P.w, P.w_dt, cols, NV * 8 * tpr);
    if (POST && P.pw) keep_param<MODE>(kept_pw, P.pw, P.pw_dt, cols, NV * 8 * tpr);
  }
  auto request = [&](int k, int stage) {  // thread 0: this CTA's row k
    uint8_t *at = dyn + (size_t)stage * bytes;
    const int64_t row = blockIdx.x + (int64_t)k * gridDim.x;
    uint32_t total = span_of<MODE>(ax, row, P.T, e).n + span_of<MODE>(ay, row, P.T, e).n;
    if (GATE == 1) total += span_of<MODE>(ag, row, P.T, e).n;
    mbar_expect_tx(&full[stage], total);
    copy_row<MODE>(at, ax, row, P.T, e, &full[stage]);
    copy_row<MODE>(at + bx, ay, row, P.T, e, &full[stage]);
    if (GATE == 1) copy_row<MODE>(at + bx + by, ag, row, P.T, e, &full[stage]);
  };
  if (t == 0) {
    for (int i = 0; i < P.stages; ++i) mbar_init(&full[i], 1);
    lost_row = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < P.stages && i < rows; ++i) request(i, i);
  }
  __syncthreads();
  int stage = 0;
  uint32_t phase = 0;
  bool lost = false;  // a wait gave up: go on without waiting or copying (results invalid)
  // After a reduction, when every thread has read this stage: the first one for
  // bf16 parameters.  (For fp32 ones that came out slower, 140 against 125 us.)
  auto refill = [&](int k) {
    if (t == 0 && !lost && k + P.stages < rows) {
      fence_proxy_async_smem();
      request(k + P.stages, stage);
    }
  };
  for (int k = 0; k < rows; ++k) {
    const int64_t row = blockIdx.x + (int64_t)k * gridDim.x;
    if (!lost) {
      uint32_t n = 0;
      while (!mbar_try_wait(&full[stage], phase) && n < kMaxPolls) ++n;
      if (n == kMaxPolls) {
        lost = true;
        if (t == 0) lost_row = k;
        status_or(P.status, BS_STATUS_TIMEOUT);
      }
    }
    uint8_t *at = dyn + (size_t)stage * bytes;
    uint32_t ox = 0, oy = bx, og = bx + by;
    if constexpr (MODE != kRowsAligned) {
      if (near_end(row, P.T)) {
        copy_rest<MODE>(at, ax, row, P.T, e);
        copy_rest<MODE>(at + bx, ay, row, P.T, e);
        if (GATE == 1) copy_rest<MODE>(at + bx + by, ag, row, P.T, e);
        __syncthreads();
      }
    }
    if constexpr (MODE == kRowsAny) {
      ox += span_of<MODE>(ax, row, P.T, e).off;
      oy += span_of<MODE>(ay, row, P.T, e).off;
      if (GATE == 1) og += span_of<MODE>(ag, row, P.T, e).off;
    }
    RowParam<MODE, NV, TW> param_w = {P.w, kept_w, P.w_dt};
    RowParam<MODE, NV, TPW> param_pw = {P.pw, kept_pw, P.pw_dt};
    float2 xs[NV][4], z[NV][4], sq = both(0.f);
    Raw8<TG> gr[GATE == 1 ? NV : 1];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Raw8<TX> xr;
      Raw8<TY> yr;
      take<MODE>(xr, at + ox, v, cols);
      take<MODE>(yr, at + oy, v, cols);
      if constexpr (GATE == 1) take<MODE>(gr[v], at + og, v, cols);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xs[v][i] = pair(xr, i);
        z[v][i] = pair(yr, i);
        if constexpr (POST) sq = fma2(z[v][i], z[v][i], sq);
      }
    }
    float a1 = 1.f;
    float2 ga[GATE == 2 ? NV : 1][4];
    if constexpr (GATE == 2) {
      const int64_t g = gate_row(row, P.gate_rows);
      if (P.gate_wide) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          get_param<MODE>(ga[v], P.gate, P.gate_dt, g * D, v, cols);
      } else {
        a1 = gate_act(load_one(P.gate, P.gate_dt, g), P.act);
      }
    }
    float2 scale = both(P.branch * a1);
    if constexpr (POST) {
      float sum[1] = {sq.x + sq.y};
      param_pw.fetch(cols);
      row_sums<1, true>(sum, buf, turn);
      if (NARROW) refill(k);
      const float r = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
      if (P.r_post && t == 0) P.r_post[row] = r;
      scale = both(P.branch * a1 * r);
    }
    sq = both(0.f);
    const float2 skip = both(P.skip);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (POST && P.pw) {
        float2 pw[4];
        param_pw.take(pw, v, cols);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[v][i] = mul(z[v][i], pw[i]);
      }
      if (GATE == 1 || (GATE == 2 && P.gate_wide)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 g;
          if constexpr (GATE == 1) g = pair(gr[v], i);
          else g = ga[GATE == 2 ? v : 0][i];
          z[v][i] = mul(z[v][i], gate_act(g, P.act));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xs[v][i] = fma2(scale, z[v][i], mul(skip, xs[v][i]));
        sq = fma2(xs[v][i], xs[v][i], sq);
      }
      put8<MODE, true>(static_cast<TX *>(P.s) + row * D, xs[v], v, cols);
    }
    float sum[1] = {sq.x + sq.y};
    param_w.fetch(cols);
    row_sums<1, true>(sum, buf, turn);
    if (!POST || !NARROW) refill(k);
    if (++stage == P.stages) {
      stage = 0;
      phase ^= 1;
    }
    const float r = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
    if (P.r_pre && t == 0) P.r_pre[row] = r;
    const float2 r2 = both(r);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float2 w[4];
      if (P.w) param_w.take(w, v, cols);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        xs[v][i] = P.w ? mul(mul(xs[v][i], r2), w[i]) : mul(xs[v][i], r2);
      put8<MODE, true>(static_cast<TY *>(P.h) + row * D, xs[v], v, cols);
    }
  }
  if (t == 0 && lost_row >= 0) drain(full, lost_row, rows, P.stages);
}

// Rows wider than the registers hold: the row is read once for each
// statistic and once for the outputs (from L2 after the first time).
template <class TX, class TY>
__global__ void __launch_bounds__(512) norm_fwd_wide_kernel(const NormParams P) {
  __shared__ float buf[2][1][32];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const TX *x = static_cast<const TX *>(P.x) + row * P.ldx;
  const TY *y = P.y ? static_cast<const TY *>(P.y) + row * P.ldy : nullptr;
  const int64_t g = P.gate ? gate_row(row, P.gate_rows) : 0;
  const bool post = P.post != 0;
  float ry = 1.f;
  if (y && post) {
    float sum[1] = {0.f};
    for (int c = threadIdx.x; c < P.D; c += blockDim.x) {
      const float v = to_f32(y[c]);
      sum[0] = fmaf(v, v, sum[0]);
    }
    row_sums<1, true>(sum, buf, turn);
    ry = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
    if (P.r_post && threadIdx.x == 0) P.r_post[row] = ry;
  }
  auto joined = [&](int c) {
    float v = to_f32(x[c]);
    if (y) {
      float z = to_f32(y[c]);
      if (post) z *= P.pw ? ry * load_one(P.pw, P.pw_dt, c) : ry;
      if (P.gate)
        z *= gate_act(load_one(P.gate, P.gate_dt, P.gate_wide ? g * P.D + c : g), P.act);
      v = fmaf(P.branch, z, P.skip * v);
    }
    return v;
  };
  float sum[1] = {0.f};
  for (int c = threadIdx.x; c < P.D; c += blockDim.x) {
    const float v = joined(c);
    sum[0] = fmaf(v, v, sum[0]);
  }
  row_sums<1, true>(sum, buf, turn);
  const float r = rsqrtf(fmaf(sum[0], P.rcp_d, P.eps));
  if (P.r_pre && threadIdx.x == 0) P.r_pre[row] = r;
  for (int c = threadIdx.x; c < P.D; c += blockDim.x) {
    const float v = joined(c);
    if (P.s) static_cast<TX *>(P.s)[row * P.D + c] = from_f32<TX>(v);
    static_cast<TY *>(P.h)[row * P.D + c] =
        from_f32<TY>(v * (P.w ? r * load_one(P.w, P.w_dt, c) : r));
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// Rows of chunk `b`: a run of whole gate groups, or a part of one group.
__device__ __forceinline__ void chunk_range(const NormParams &P, int64_t b, int64_t &r0,
                                            int64_t &r1) {
  if (P.groups_per_chunk) {
    r0 = b * P.groups_per_chunk * P.div_rows;
    r1 = r0 + P.groups_per_chunk * P.div_rows;
    if (r1 > P.T) r1 = P.T;
  } else {
    const int64_t g = b / P.chunks_per_group, k = b - g * P.chunks_per_group;
    const int64_t end = (g + 1) * P.div_rows;
    r0 = g * P.div_rows + k * P.chunk_rows;
    r1 = r0 + P.chunk_rows < end ? r0 + P.chunk_rows : end;
  }
}

// Whole rows arrive in shared memory by bulk copies, P.stages rows ahead, so the
// loads in flight do not depend on registers or on where the block stands; a
// row is taken into registers before its reduction, whose barrier therefore
// also frees its stage.  bf16 parameters are fetched before the wait for the
// row, but a norm's on the branch with an element gate, which has no registers
// for them (16 x 1024 x 4096 bf16: 354 us from spills).  Backward and column sums
// with the fetch and without: 16384 x 4096 bf16 with a norm 165 and 175 us, with an
// element gate too 214 and 216, with a channel gate 208 and 228; on an fp32 stream
// 16384 x 2048 105 both, with a norm 116 and 126; 4096 x 6144 bf16 with a norm and a
// channel gate, two vectors a thread, 153 and 161 in spite of its spills.
//
// GATE: 0 none, 1 an element each (in the stage), 4 the same with a sigmoid, 2
// columns shared by rows (in registers while the group lasts, its sums too), 3
// one column.  TW: the type of both parameters (aligned rows), else void.
template <class TX, class TY, class TG, int W, bool POST, int GATE, int MODE, class TW>
__global__ void __launch_bounds__(GATE == 2 || W == 4 ? 512 : 256, GATE == 2 || W == 4 ? 1 : 2)
    norm_bwd_staged_kernel(const NormParams P) {
  constexpr int NV = vectors(W);
  constexpr bool BRANCH = POST || GATE != 0, ELEM = GATE == 1 || GATE == 4;
  constexpr int ACT = GATE == 4 ? kActSigmoid : kActNone;  // of ELEM
  using TPW = typename std::conditional<ELEM, void, TW>::type;
  constexpr int NS = BRANCH ? 3 : 1;
  extern __shared__ uint8_t dyn[];
  __shared__ float buf[2][NS][32];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int lost_row;  // of thread 0, if its wait gave up
  int turn = 0;
  const int tpr = blockDim.x, t = threadIdx.x, D = P.D;
  int64_t r0, r1;
  // kRowsShifted: eight CTAs share a range of rows, by row mod 8
  constexpr int STEP = MODE == kRowsShifted ? 8 : 1;
  chunk_range(P, blockIdx.x / STEP, r0, r1);
  if (STEP == 8) r0 += (int)((blockIdx.x - r0) & 7);
  const int rows = r1 > r0 ? (int)((r1 - r0 + STEP - 1) / STEP) : 0;
  const int e = MODE == kRowsShifted ? (int)((r0 & 7) * D & 7) : 0;
  const Cols cols = {t, tpr, D, e};
  // a stage: s, then ds, dh, y, gate where they are
  const uint32_t rx = (uint32_t)D * (uint32_t)sizeof(TX), ry_ = (uint32_t)D * (uint32_t)sizeof(TY);
  const Staged arr[5] = {
      {static_cast<const uint8_t *>(P.s), P.lds * (int64_t)sizeof(TX), sizeof(TX), rx},
      {static_cast<const uint8_t *>(P.ds), (int64_t)rx, sizeof(TX), rx},
      {static_cast<const uint8_t *>(P.dh), (int64_t)ry_, sizeof(TY), ry_},
      {BRANCH ? static_cast<const uint8_t *>(P.y) : nullptr, P.ldy * (int64_t)sizeof(TY),
       sizeof(TY), ry_},
      {ELEM ? static_cast<const uint8_t *>(P.gate) : nullptr, D * (int64_t)sizeof(TG), sizeof(TG),
       (uint32_t)D * (uint32_t)sizeof(TG)}};
  uint32_t place[5], bytes = 0;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    place[i] = bytes;
    if (arr[i].base) bytes += stage_bytes<MODE>(D, arr[i].size);
  }
  float *kept_w = reinterpret_cast<float *>(dyn + (size_t)P.stages * bytes);
  float *kept_pw = kept_w + (P.w ? NV * 8 * tpr : 0);
  if constexpr (MODE != kRowsAligned) {
    if (P.w) keep_param<MODE>(kept_w, P.w, P.w_dt, cols, NV * 8 * tpr);
    if (POST && P.pw) keep_param<MODE>(kept_pw, P.pw, P.pw_dt, cols, NV * 8 * tpr);
  }
  auto request = [&](int k, int stage) {  // thread 0: row k of the chunk
    uint8_t *at = dyn + (size_t)stage * bytes;
    const int64_t row = r0 + (int64_t)k * STEP;
    uint32_t total = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i)
      if (arr[i].base) total += span_of<MODE>(arr[i], row, P.T, e).n;
    mbar_expect_tx(&full[stage], total);
#pragma unroll
    for (int i = 0; i < 5; ++i)
      if (arr[i].base) copy_row<MODE>(at + place[i], arr[i], row, P.T, e, &full[stage]);
  };
  if (t == 0) {
    for (int i = 0; i < P.stages; ++i) mbar_init(&full[i], 1);
    lost_row = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < P.stages && i < rows; ++i) request(i, i);
  }
  float2 acc_w[NV][4], acc_p[POST ? NV : 1][4], acc_g[GATE == 2 ? NV : 1][4];
  float2 ga[GATE == 2 ? NV : 1][4];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc_w[v][i] = both(0.f);
      if (POST) acc_p[v][i] = both(0.f);
      if (GATE == 2) acc_g[v][i] = both(0.f);
    }
  __syncthreads();
  int stage = 0;
  uint32_t phase = 0;
  bool lost = false;  // a wait gave up: go on without waiting or copying (results invalid)
  float r_next = rows > 0 ? P.r_pre[r0] : 0.f;
  float ry_next = POST && rows > 0 ? P.r_post[r0] : 1.f;
  for (int k = 0; k < rows; ++k) {
    const int64_t row = r0 + (int64_t)k * STEP;
    const float r = r_next, ry = ry_next;
    if (k + 1 < rows) {
      r_next = P.r_pre[row + STEP];
      if (POST) ry_next = P.r_post[row + STEP];
    }
    const int64_t grow = GATE ? gate_row(row, P.gate_rows) : 0;
    float a1 = 1.f;  // the gate of the row, where it has one column
    if (GATE == 3) a1 = gate_act(load_one(P.gate, P.gate_dt, grow), P.act);
    if constexpr (GATE == 2) {
      // (kRowsShifted: all rows of the CTA are of one group)
      if (k == 0 || (STEP == 1 && (uint32_t)row % (uint32_t)P.gate_rows == 0)) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          get_param<MODE>(ga[v], P.gate, P.gate_dt, grow * D, v, cols);
#pragma unroll
          for (int i = 0; i < 4; ++i) ga[v][i] = gate_act(ga[v][i], P.act);
        }
      }
    }
    RowParam<MODE, NV, TW> param_w = {P.w, kept_w, P.w_dt};
    RowParam<MODE, NV, TPW> param_pw = {P.pw, kept_pw, P.pw_dt};
    param_w.fetch(cols);
    if (POST) param_pw.fetch(cols);
    if (!lost) {
      uint32_t n = 0;
      while (!mbar_try_wait(&full[stage], phase) && n < kMaxPolls) ++n;
      if (n == kMaxPolls) {
        lost = true;
        if (t == 0) lost_row = k;
        status_or(P.status, BS_STATUS_TIMEOUT);
      }
    }
    uint8_t *at = dyn + (size_t)stage * bytes;
    uint32_t in[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) in[i] = place[i];
    if constexpr (MODE != kRowsAligned) {
      if (near_end(row, P.T)) {
#pragma unroll
        for (int i = 0; i < 5; ++i)
          if (arr[i].base) copy_rest<MODE>(at + place[i], arr[i], row, P.T, e);
        __syncthreads();
      }
    }
    if constexpr (MODE == kRowsAny) {
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (arr[i].base) in[i] += span_of<MODE>(arr[i], row, P.T, e).off;
    }
    float2 xh[NV][4], A[NV][4], sum2[NS];
    Raw8<TY> yr[BRANCH ? NV : 1];
    Raw8<TG> gr[ELEM ? NV : 1];
#pragma unroll
    for (int i = 0; i < NS; ++i) sum2[i] = both(0.f);
    const float2 r2 = both(r), skip_r = both(BRANCH ? P.skip * r : r);
    // q leaves the factors of the row out: ry (POST), a1 (one gate)
    const float2 branch_r = both(P.branch * ry * a1 * r);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Raw8<TX> xr, sr = {};
      Raw8<TY> hr = {};
      float2 w[4], pw[4];
      take<MODE>(xr, at + in[0], v, cols);
      if (P.ds) take<MODE>(sr, at + in[1], v, cols);
      if (P.dh) take<MODE>(hr, at + in[2], v, cols);
      if constexpr (BRANCH) take<MODE>(yr[v], at + in[3], v, cols);
      if constexpr (ELEM) take<MODE>(gr[v], at + in[4], v, cols);
      if (P.w) param_w.take(w, v, cols);
      if (POST && P.pw) param_pw.take(pw, v, cols);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 x = mul(skip_r, pair(xr, i)), q = both(0.f);
        if constexpr (BRANCH) {
          q = pair(yr[v], i);
          if (POST && P.pw) q = mul(q, pw[i]);
          if constexpr (ELEM) q = mul(q, gate_act(pair(gr[v], i), ACT));
          if constexpr (GATE == 2) q = mul(q, ga[v][i]);
          x = fma2(branch_r, q, x);
        }
        const float2 h = pair(hr, i), dxh = P.w ? mul(h, w[i]) : h;
        const float2 a = fma2(r2, dxh, pair(sr, i));
        acc_w[v][i] = fma2(h, x, acc_w[v][i]);
        sum2[0] = fma2(dxh, x, sum2[0]);
        if constexpr (BRANCH) {
          sum2[1] = fma2(q, a, sum2[1]);
          sum2[2] = fma2(q, x, sum2[2]);
        }
        xh[v][i] = x;
        A[v][i] = a;
      }
    }
    float sums[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) sums[i] = sum2[i].x + sum2[i].y;
    row_sums<NS, true>(sums, buf, turn);
    if (t == 0 && !lost && k + P.stages < rows) {  // every thread has read this stage
      fence_proxy_async_smem();
      request(k + P.stages, stage);
    }
    if (++stage == P.stages) {
      stage = 0;
      phase ^= 1;
    }
    const float c1 = r * (sums[0] * P.rcp_d);
    float qd = 0.f;  // sum over the row of (ry q) d
    if constexpr (BRANCH) qd = ry * (sums[1] - c1 * sums[2]);
    if (GATE == 3 && t == 0) {  // the one gate of the row
      const float dg = P.branch * qd * gate_slope(a1, P.act);
      if (P.gate_rows > 1) P.row_gate[row] = dg;
      else if (P.dgate) store_one(P.dgate, P.gate_dt, row, dg);
    }
    // dy = ry (du w_post - n mean(du w_post n)):  the factors of the row, once
    const float2 minus_c1 = both(-c1), skip = both(P.skip);
    const float2 to_du = both(P.branch * (GATE == 3 ? a1 : 1.f)), ry2 = both(ry);
    const float2 to_y = both(-ry * (P.branch * a1 * qd * P.rcp_d));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float2 pw[4], o[4], dg[4];
      if (POST && P.pw) param_pw.take(pw, v, cols);
#pragma unroll
      for (int i = 0; i < 4; ++i) A[v][i] = fma2(minus_c1, xh[v][i], A[v][i]);
      if (P.dx) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mul(skip, A[v][i]);
        put8<MODE, true>(static_cast<TX *>(P.dx) + row * D, o, v, cols);
      }
      if constexpr (BRANCH) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 d = mul(to_du, A[v][i]);
          const float2 y = pair(yr[v], i), n = POST ? mul(y, ry2) : y;
          if constexpr (ELEM || GATE == 2) {
            float2 a;
            if constexpr (ELEM) a = gate_act(pair(gr[v], i), ACT);
            else a = ga[v][i];
            dg[i] = mul(d, mul(POST && P.pw ? mul(n, pw[i]) : n, gate_slope(a, ELEM ? ACT : P.act)));
            if constexpr (GATE == 2) acc_g[v][i] = add(acc_g[v][i], dg[i]);
            d = mul(d, a);
          }
          if constexpr (POST) {
            acc_p[v][i] = fma2(d, n, acc_p[v][i]);
            d = mul(d, ry2);
            if (P.pw) d = mul(d, pw[i]);
            d = fma2(to_y, n, d);
          }
          o[i] = d;
        }
        if (P.dy) put8<MODE, true>(static_cast<TY *>(P.dy) + row * D, o, v, cols);
        if constexpr (ELEM)
          if (P.dgate) put8<MODE, true>(static_cast<TG *>(P.dgate) + row * D, dg, v, cols);
      } else if (P.dy) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mul(to_du, A[v][i]);
        put8<MODE, true>(static_cast<TY *>(P.dy) + row * D, o, v, cols);
      }
    }
    if constexpr (GATE == 2) {
      if (P.groups_per_chunk && (uint32_t)(row + 1) % (uint32_t)P.gate_rows == 0) {
        // the last row of a group that this CTA has whole
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (P.dgate) put_param<MODE>(P.dgate, acc_g[v], P.gate_dt, grow * D, v, cols);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc_g[v][i] = both(0.f);
        }
      }
    }
  }
  if (t == 0 && lost_row >= 0) drain(full, lost_row, rows, P.stages);
  const int64_t mine = (int64_t)blockIdx.x * D, plane = P.chunks * (int64_t)D;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    put8<MODE, false>(P.part + mine, acc_w[v], v, cols);
    if constexpr (POST) put8<MODE, false>(P.part + plane + mine, acc_p[v], v, cols);
    if constexpr (GATE == 2)
      if (!P.groups_per_chunk)
        put8<MODE, false>(P.part + 2 * plane + mine, acc_g[v], v, cols);
  }
}

// Rows wider than the registers hold: the sums in one pass over the row, the
// outputs in a second, the column sums kept in this CTA's rows of `part`.
template <class TX, class TY>
__global__ void __launch_bounds__(512) norm_bwd_wide_kernel(const NormParams P) {
  __shared__ float buf[2][3][32];
  int turn = 0;
  const int D = P.D;
  const bool post = P.post != 0, gate = P.gate != nullptr;
  const bool sum_gate = gate && P.gate_wide && P.gate_rows > 1;
  int64_t r0, r1;
  chunk_range(P, blockIdx.x, r0, r1);
  const int64_t plane = P.chunks * (int64_t)D;
  float *pw_ = P.part + (int64_t)blockIdx.x * D, *pp_ = pw_ + plane, *pg_ = pp_ + plane;
  for (int c = threadIdx.x; c < D; c += blockDim.x) {
    pw_[c] = 0.f;
    if (post) pp_[c] = 0.f;
    if (sum_gate) pg_[c] = 0.f;
  }
  for (int64_t row = r0; row < r1; ++row) {
    const float r = P.r_pre[row], ry = post ? P.r_post[row] : 1.f;
    const int64_t grow = gate ? gate_row(row, P.gate_rows) : 0;
    const float a1 =
        gate && !P.gate_wide ? gate_act(load_one(P.gate, P.gate_dt, grow), P.act) : 1.f;
    const TX *s = static_cast<const TX *>(P.s) + row * P.lds;
    const TX *ds = P.ds ? static_cast<const TX *>(P.ds) + row * D : nullptr;
    const TY *dh = P.dh ? static_cast<const TY *>(P.dh) + row * D : nullptr;
    const TY *y = post || gate ? static_cast<const TY *>(P.y) + row * P.ldy : nullptr;
    auto branch = [&](int c) {  // act(gate) u, without a one-column gate
      float q = to_f32(y[c]) * (post && P.pw ? ry * load_one(P.pw, P.pw_dt, c) : ry);
      if (gate && P.gate_wide) q *= gate_act(load_one(P.gate, P.gate_dt, grow * D + c), P.act);
      return q;
    };
    auto unit = [&](int c, float q) {
      const float v = to_f32(s[c]);
      return (y ? fmaf(P.branch, a1 * q, P.skip * v) : v) * r;
    };
    float sums[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float q = y ? branch(c) : 0.f, xh = unit(c, q);
      const float dxh = dh ? to_f32(dh[c]) * (P.w ? load_one(P.w, P.w_dt, c) : 1.f) : 0.f;
      const float A = fmaf(r, dxh, ds ? to_f32(ds[c]) : 0.f);
      sums[0] = fmaf(dxh, xh, sums[0]);
      sums[1] = fmaf(q, A, sums[1]);
      sums[2] = fmaf(q, xh, sums[2]);
    }
    row_sums<3, true>(sums, buf, turn);
    const float c1 = r * (sums[0] * P.rcp_d), qd = sums[1] - c1 * sums[2];
    if (gate && !P.gate_wide && threadIdx.x == 0) {
      const float dg = P.branch * qd * gate_slope(a1, P.act);
      if (P.gate_rows > 1) P.row_gate[row] = dg;
      else if (P.dgate) store_one(P.dgate, P.gate_dt, row, dg);
    }
    const float c2 = P.branch * a1 * qd * P.rcp_d;
    const bool last = sum_gate && P.groups_per_chunk && (uint32_t)(row + 1) % (uint32_t)P.gate_rows == 0;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float xh = unit(c, y ? branch(c) : 0.f);
      const float dhv = dh ? to_f32(dh[c]) : 0.f;
      const float A = fmaf(r, dhv * (P.w ? load_one(P.w, P.w_dt, c) : 1.f),
                           ds ? to_f32(ds[c]) : 0.f);
      float d = fmaf(-c1, xh, A);
      pw_[c] = fmaf(dhv, xh, pw_[c]);
      if (P.dx) static_cast<TX *>(P.dx)[row * D + c] = from_f32<TX>(P.skip * d);
      d *= P.branch;
      const float yc = y ? to_f32(y[c]) : 0.f;
      const float n = yc * ry, p = post && P.pw ? load_one(P.pw, P.pw_dt, c) : 1.f;
      if (gate && P.gate_wide) {
        const float a = gate_act(load_one(P.gate, P.gate_dt, grow * D + c), P.act);
        const float dg = d * (post ? n * p : yc) * gate_slope(a, P.act);
        if (sum_gate) {
          const float v = pg_[c] + dg;
          pg_[c] = last ? 0.f : v;
          if (last && P.dgate) store_one(P.dgate, P.gate_dt, grow * D + c, v);
        } else if (P.dgate) {
          store_one(P.dgate, P.gate_dt, row * D + c, dg);
        }
        d *= a;
      } else if (gate) {
        d *= a1;
      }
      if (post) {
        pp_[c] = fmaf(d, n, pp_[c]);
        d = ry * fmaf(-n, c2, d * p);
      }
      if (P.dy) static_cast<TY *>(P.dy)[row * D + c] = from_f32<TY>(d);
    }
  }
}

// Sums of `n` rows of D columns, in a fixed order: out[group][c] =
// sum_k in[group * n + k][c].  W columns a thread (four where D allows 16-byte
// loads), 32 columns x 256 W / 32 row lanes a block, four loads in flight.
struct SumJob {
  const float *in;
  void *out;
  int dt;
  int64_t n, groups;
};
struct SumJobs {
  SumJob job[3];
};
template <int W>
__global__ void __launch_bounds__(256) norm_sum_kernel(const SumJobs J, int D) {
  constexpr int X = 32 / W, LANES = 256 / X;
  __shared__ float part[LANES][33];
  const SumJob j = J.job[blockIdx.z];
  const int x = threadIdx.x % X, k0 = threadIdx.x / X, c = blockIdx.x * 32 + x * W;
  if (!j.out) return;
  const int n = (int)j.n;
  for (int64_t g = blockIdx.y; g < j.groups; g += gridDim.y) {
    float s[W];
#pragma unroll
    for (int w = 0; w < W; ++w) s[w] = 0.f;
    if (c < D) {
      const float *in = j.in + g * j.n * D + c;
      for (int k = k0; k < n; k += 4 * LANES) {
        float v[4][W];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int w = 0; w < W; ++w) v[i][w] = 0.f;
          const int r = k + i * LANES;
          if (r >= n) continue;
          if constexpr (W == 4) {
            const float4 q = *reinterpret_cast<const float4 *>(in + (int64_t)r * D);
            v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
          } else {
            v[i][0] = in[(int64_t)r * D];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < W; ++w) s[w] += v[i][w];
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) part[k0][x * W + w] = s[w];
    __syncthreads();
    // eight threads a column add its lanes
    const int col = threadIdx.x >> 3, e = threadIdx.x & 7;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < LANES / 8 + (LANES < 8); ++k)
      if (k * 8 + e < LANES) v += part[k * 8 + e][col];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (e == 0 && blockIdx.x * 32 + col < D) store_one(j.out, j.dt, g * D + blockIdx.x * 32 + col, v);
    __syncthreads();
  }
}
// The gate sums of rows of a one-column gate: out[g] = sum of its rows.
__global__ void __launch_bounds__(256) norm_gate_sum_kernel(const float *rows, int64_t n,
                                                            void *out, int dt,
                                                            int64_t groups) {
  __shared__ float buf[2][1][32];
  int turn = 0;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    float s[1] = {0.f};
    for (int64_t k = threadIdx.x; k < n; k += 256) s[0] += rows[g * n + k];
    row_sums<1, true>(s, buf, turn);
    if (threadIdx.x == 0) store_one(out, dt, g, s[0]);
  }
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
constexpr int kMaxDev = 64;
inline int sm_count(int *sms) {
  static std::mutex mu;
  static int of[kMaxDev] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return BS_ERR_LAUNCH;
  std::lock_guard<std::mutex> lock(mu);
  if (!of[dev] && (cudaDeviceGetAttribute(&of[dev], cudaDevAttrMultiProcessorCount, dev) !=
                       cudaSuccess || of[dev] <= 0)) {
    of[dev] = 0;
    return BS_ERR_LAUNCH;
  }
  *sms = of[dev];
  return BS_OK;
}
inline int launched() { return launch_code(cudaGetLastError()); }

// Threads of a row and vectors a thread: forward, one warp up to 1024
// columns, then 16 columns a thread up to 8192 and 32 up to 16384.
constexpr int kFwdMaxD = 16384, kBwdMaxD = 8192;

template <class TX, class TY, int NV, bool VEC, bool BLOCK>
int launch_fwd(const NormParams &P, bool post, cudaStream_t st) {
  const int threads = BLOCK ? ((P.D + 8 * NV * 32 - 1) / (8 * NV * 32)) * 32 : 128;
  const int64_t grid = BLOCK ? P.T : (P.T + 3) / 4;
  const bool gate = P.gate != nullptr;
  if (post && gate)
    norm_fwd_kernel<TX, TY, NV, VEC, BLOCK, true, true><<<(unsigned)grid, threads, 0, st>>>(P);
  else if (post)
    norm_fwd_kernel<TX, TY, NV, VEC, BLOCK, true, false><<<(unsigned)grid, threads, 0, st>>>(P);
  else if (gate)
    norm_fwd_kernel<TX, TY, NV, VEC, BLOCK, false, true><<<(unsigned)grid, threads, 0, st>>>(P);
  else
    norm_fwd_kernel<TX, TY, NV, VEC, BLOCK, false, false><<<(unsigned)grid, threads, 0, st>>>(P);
  return launched();
}
template <class TX, class TY, bool VEC>
int fwd_by_width(const NormParams &P, bool post, cudaStream_t st) {
  if (P.D <= 256) return launch_fwd<TX, TY, 1, VEC, false>(P, post, st);
  if (P.D <= 512) return launch_fwd<TX, TY, 2, VEC, false>(P, post, st);
  if (P.D <= 1024) return launch_fwd<TX, TY, 4, VEC, false>(P, post, st);
  if (P.D <= 2048) return launch_fwd<TX, TY, 1, VEC, true>(P, post, st);
  if (P.D <= 8192) return launch_fwd<TX, TY, 2, VEC, true>(P, post, st);
  return launch_fwd<TX, TY, 4, VEC, true>(P, post, st);
}
// Columns that the threads of a row cover: a shifted row has up to 7 more at
// either end.
inline int64_t row_width(int64_t D, int mode) {
  return mode == kRowsShifted ? (D + 14) / 8 * 8 : D;
}
// The limit of dynamic shared memory is per device: set once for each kernel and
// device (`set` is the kernel's own).
struct SmemSet {
  std::mutex mu;
  bool done[kMaxDev] = {};
};
template <class K>
int raise_smem(K kernel, SmemSet &set) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return BS_ERR_LAUNCH;
  std::lock_guard<std::mutex> lock(set.mu);
  if (!set.done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kStagedSmem) != cudaSuccess)
      return BS_ERR_LAUNCH;
    set.done[dev] = true;
  }
  return BS_OK;
}
inline int elt(int dt) { return dt == BS_F32 ? 4 : 2; }

template <class TX, class TY, class TG, int W, bool POST, int GATE, int MODE, class TW>
int launch_fwd_typed(NormParams P, int sms, cudaStream_t st) {
  auto kernel = norm_fwd_staged_kernel<TX, TY, TG, W, POST, GATE, MODE, TW>;
  constexpr int NV = vectors(W);
  static SmemSet set;
  if (raise_smem(kernel, set) != BS_OK) return BS_ERR_LAUNCH;
  const int threads = (int)((row_width(P.D, MODE) + 256 * NV - 1) / (256 * NV) * 32);
  const size_t row = stage_bytes<MODE>(P.D, sizeof(TX)) + stage_bytes<MODE>(P.D, sizeof(TY)) +
                     (GATE == 1 ? stage_bytes<MODE>(P.D, sizeof(TG)) : 0);
  int64_t per_sm = W == 4 ? 1 : 768 / threads;
  if (per_sm > 16) per_sm = 16;
  const size_t kept = MODE != kRowsAligned ? (size_t)((P.w ? 1 : 0) + (P.pw ? 1 : 0)) * NV * 8 * threads * 4 : 0;
  while (per_sm > 1 && 2 * row + kept > kStagedSmem / per_sm) --per_sm;
  P.stages = (int)((kStagedSmem / per_sm - kept) / row);
  if (P.stages > kMaxStages) P.stages = kMaxStages;
  int64_t grid = sms * per_sm < P.T ? sms * per_sm : P.T;
  if (MODE == kRowsShifted) grid = grid / 8 * 8;  // (there are four rows an SM at least)
  kernel<<<(unsigned)grid, threads, P.stages * row + kept, st>>>(P);
  return launched();
}
template <class TX, class TY, class TG, int W, bool POST, int GATE, int MODE>
int launch_fwd_staged(const NormParams &P, int sms, cudaStream_t st) {
  if constexpr (MODE == kRowsAligned) {
    const bool wide = (P.w && P.w_dt == BS_F32) || (P.pw && P.pw_dt == BS_F32);
    if (!wide) return launch_fwd_typed<TX, TY, TG, W, POST, GATE, MODE, uint16_t>(P, sms, st);
    if ((!P.w || P.w_dt == BS_F32) && (!P.pw || P.pw_dt == BS_F32))
      return launch_fwd_typed<TX, TY, TG, W, POST, GATE, MODE, float>(P, sms, st);
  }
  return launch_fwd_typed<TX, TY, TG, W, POST, GATE, MODE, void>(P, sms, st);
}
template <class TX, class TY, int W, bool POST, int MODE>
int fwd_staged_by_gate(const NormParams &P, int sms, cudaStream_t st) {
  if (!P.gate) return launch_fwd_staged<TX, TY, TY, W, POST, 0, MODE>(P, sms, st);
  if (!P.gate_wide || P.gate_rows > 1)
    return launch_fwd_staged<TX, TY, TY, W, POST, 2, MODE>(P, sms, st);
  return P.gate_dt == BS_F32 ? launch_fwd_staged<TX, TY, float, W, POST, 1, MODE>(P, sms, st)
                             : launch_fwd_staged<TX, TY, uint16_t, W, POST, 1, MODE>(P, sms, st);
}
template <class TX, class TY, int MODE>
int fwd_staged(const NormParams &P, int sms, cudaStream_t st) {
  if (row_width(P.D, MODE) <= 4096)
    return P.post ? fwd_staged_by_gate<TX, TY, 2, true, MODE>(P, sms, st)
                  : fwd_staged_by_gate<TX, TY, 2, false, MODE>(P, sms, st);
  return P.post ? fwd_staged_by_gate<TX, TY, 4, true, MODE>(P, sms, st)
                : fwd_staged_by_gate<TX, TY, 4, false, MODE>(P, sms, st);
}

template <class TX, class TY>
int fwd_typed(const NormParams &P, bool post, int mode, cudaStream_t st) {
  // many rows of more than a warp's columns: staged (below four rows an SM the
  // start of the pipeline costs more than it hides)
  int sms = 0;
  if (P.y && P.D > 1024 && P.D <= kBwdMaxD && sm_count(&sms) == BS_OK && P.T >= 4 * (int64_t)sms)
    return mode == kRowsAligned   ? fwd_staged<TX, TY, kRowsAligned>(P, sms, st)
           : mode == kRowsShifted ? fwd_staged<TX, TY, kRowsShifted>(P, sms, st)
                                  : fwd_staged<TX, TY, kRowsAny>(P, sms, st);
  const bool vec = mode == kRowsAligned;
  if (P.D > kFwdMaxD) {
    norm_fwd_wide_kernel<TX, TY><<<(unsigned)P.T, 512, 0, st>>>(P);
    return launched();
  }
  return vec ? fwd_by_width<TX, TY, true>(P, post, st) : fwd_by_width<TX, TY, false>(P, post, st);
}

inline int gate_kind(const void *gate, int64_t gate_rows, int gate_wide) {
  return !gate ? 0 : !gate_wide ? 3 : gate_rows == 1 ? 1 : 2;
}
// Vectors of eight columns a thread: two, with at most 256 threads and two
// CTAs an SM (one CTA's reduction is hidden by the other) or, above 4096 columns,
// 512 threads; one where a warp has the row (up to 256).  The form with the most
// registers, a gate's columns and their sums, takes half of that up to 4096.
inline int staged_nv(int64_t width, int kind) {
  return width <= 256 || (kind == 2 && width <= 4096) ? 1 : 2;
}
// Resident CTAs an SM, of at most 128 registers a thread: 512 threads, and 16
// CTAs at most.
inline int64_t per_sm_for(int64_t threads) {
  const int64_t n = 512 / threads;
  return n < 1 ? 1 : n > 16 ? 16 : n;
}
inline BwdPlan plan_bwd(int64_t D, int x_dt, int y_dt, bool ds, bool dh, bool post, int kind,
                        int gate_dt, int params, int mode, int sms) {
  BwdPlan p = {};
  p.mode = mode;
  const bool branch = post || kind;
  const uint32_t d = (uint32_t)(D < kBwdMaxD ? D : kBwdMaxD);
  auto bytes = [&](int dt) {
    return (size_t)(mode == kRowsAligned   ? stage_bytes<kRowsAligned>(d, elt(dt))
                    : mode == kRowsShifted ? stage_bytes<kRowsShifted>(d, elt(dt))
                                           : stage_bytes<kRowsAny>(d, elt(dt)));
  };
  const size_t row = bytes(x_dt) * (ds ? 2 : 1) + bytes(y_dt) * ((dh ? 1 : 0) + (branch ? 1 : 0)) +
                     (kind == 1 ? bytes(gate_dt) : 0);
  const int64_t width = row_width(D, mode);
  const int nv = staged_nv(width, kind);
  p.threads = (int)((width + 256 * nv - 1) / (256 * nv)) * 32;
  const size_t kept = mode == kRowsAligned ? 0 : (size_t)params * nv * 8 * p.threads * 4;
  p.staged = width <= kBwdMaxD && row + kept <= kStagedSmem;
  if (!p.staged) {
    p.threads = 512;
    p.ctas = sms;
    return p;
  }
  int64_t per_sm = width > 4096 ? 1 : per_sm_for(p.threads);
  while (per_sm > 1 && 2 * row + kept > kStagedSmem / per_sm) --per_sm;
  p.stages = (int)((kStagedSmem / per_sm - kept) / row);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.smem = p.stages * row + kept;
  p.ctas = sms * per_sm;
  return p;
}
// The most CTAs that any form of the backward divides rows of D columns among.
inline int64_t most_ctas(int64_t D, int sms) {
  return sms * (D > 4096 ? 1 : per_sm_for((D + 511) / 512 * 32));
}
template <class TX, class TY, class TG, int W, bool POST, int GATE, int MODE, class TW = void>
int launch_staged(const NormParams &P, const BwdPlan &plan, cudaStream_t st) {
  if constexpr (MODE == kRowsAligned && std::is_void<TW>::value)
    if ((!P.w || P.w_dt != BS_F32) && (!P.pw || P.pw_dt != BS_F32))
      return launch_staged<TX, TY, TG, W, POST, GATE, MODE, uint16_t>(P, plan, st);
  auto kernel = norm_bwd_staged_kernel<TX, TY, TG, W, POST, GATE, MODE, TW>;
  static SmemSet set;
  if (raise_smem(kernel, set) != BS_OK) return BS_ERR_LAUNCH;
  kernel<<<(unsigned)P.chunks, plan.threads, plan.smem, st>>>(P);
  return launched();
}
template <class TX, class TY, int W, bool POST, int MODE>
int staged_by_gate(const NormParams &P, const BwdPlan &plan, cudaStream_t st) {
  switch (gate_kind(P.gate, P.gate_rows, P.gate_wide)) {
    case 0: return launch_staged<TX, TY, TY, W, POST, 0, MODE>(P, plan, st);
    case 1:
      if (P.act == kActSigmoid)
        return P.gate_dt == BS_F32
                   ? launch_staged<TX, TY, float, W, POST, 4, MODE>(P, plan, st)
                   : launch_staged<TX, TY, uint16_t, W, POST, 4, MODE>(P, plan, st);
      return P.gate_dt == BS_F32 ? launch_staged<TX, TY, float, W, POST, 1, MODE>(P, plan, st)
                                 : launch_staged<TX, TY, uint16_t, W, POST, 1, MODE>(P, plan, st);
    case 2: return launch_staged<TX, TY, TY, W == 4 ? 2 : 1, POST, 2, MODE>(P, plan, st);
    default: return launch_staged<TX, TY, TY, W, POST, 3, MODE>(P, plan, st);
  }
}
template <class TX, class TY, int MODE>
int bwd_staged(const NormParams &P, const BwdPlan &plan, cudaStream_t st) {
  const int64_t width = row_width(P.D, MODE);
  if (width <= 256)
    return P.post ? staged_by_gate<TX, TY, 1, true, MODE>(P, plan, st)
                  : staged_by_gate<TX, TY, 1, false, MODE>(P, plan, st);
  if (width <= 4096)
    return P.post ? staged_by_gate<TX, TY, 2, true, MODE>(P, plan, st)
                  : staged_by_gate<TX, TY, 2, false, MODE>(P, plan, st);
  return P.post ? staged_by_gate<TX, TY, 4, true, MODE>(P, plan, st)
                : staged_by_gate<TX, TY, 4, false, MODE>(P, plan, st);
}
template <class TX, class TY>
int bwd_typed(const NormParams &P, const BwdPlan &plan, cudaStream_t st) {
  if (!plan.staged) {
    norm_bwd_wide_kernel<TX, TY><<<(unsigned)P.chunks, 512, 0, st>>>(P);
    return launched();
  }
  return plan.mode == kRowsAligned   ? bwd_staged<TX, TY, kRowsAligned>(P, plan, st)
         : plan.mode == kRowsShifted ? bwd_staged<TX, TY, kRowsShifted>(P, plan, st)
                                     : bwd_staged<TX, TY, kRowsAny>(P, plan, st);
}

}  // namespace

// One file for each pair of types (stream, activations): norm_f32.cu, norm_mix.cu, norm_bf16.cu.
int norm_forward_f32(const NormParams &P, int mode, cudaStream_t st);
int norm_forward_mix(const NormParams &P, int mode, cudaStream_t st);
int norm_forward_bf16(const NormParams &P, int mode, cudaStream_t st);
int norm_backward_f32(const NormParams &P, const BwdPlan &plan, cudaStream_t st);
int norm_backward_mix(const NormParams &P, const BwdPlan &plan, cudaStream_t st);
int norm_backward_bf16(const NormParams &P, const BwdPlan &plan, cudaStream_t st);

}  // namespace bs
