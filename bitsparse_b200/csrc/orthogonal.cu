// Orthogonalisation of an optimiser's update by Newton-Schulz products.
//
//   X = G / (|G|_F + eps);  per step  S = X X^T,  P = a I + b S + c S^2,  X = P X
//
// (for a tall G the same on the other side: S = X^T X, X = X P), for a batch
// of equal matrices.  Every singular value s goes to s p(s^2), so the result
// has G's singular vectors and singular values near 1.
//
// All products run on the tensor cores with fp16 operands and fp32
// accumulation.  fp16 rather than bf16: three more bits of mantissa at the
// same rate, and the exponent range is no concern, because every matrix here
// has a known bound on its spectral norm (1 after the division, then the
// maximum of the step's polynomial over the previous range) which bounds its
// elements too: each is stored times a power of two that puts the bound at
// 2^14.  Rounding X, S and P to bf16 moves the result by 0.9 to 1.2 per cent
// (256 x 256 and 384 x 768 matrices of a few strong directions over noise), to
// scaled fp16 by 0.11 to 0.15.
//
// S and P are symmetric: only the tiles on and below the diagonal are
// computed, and each is stored twice, the second time transposed through
// shared memory.  a I is put into P, so that X = P X needs no second read of
// X and P's rounding is relative to p(s^2) near 1, not to its larger terms.
// No matrix is ever transposed in memory: TMA delivers either operand K-major
// or MN-major and the instruction descriptor says which.
//
// One launch does all products of all steps.  Its tiles are in one order --
// step, phase (S, P, X), matrix, tile -- and dealt to the resident CTAs (or CTA
// pairs, cta_group::2, on 256 x 256 tiles) in turn.  A tile waits only for the
// phase before it of its own matrix, by a counter that the epilogues of that
// phase raise once their stores are complete; matrices of a batch overlap, so
// neither a phase's last, partly filled round of tiles nor a launch's start
// and drain is paid 15 times.  Every wait is on tiles that come earlier in the
// order, all CTAs are resident (cooperative launch) and every wait is bounded
// (BS_STATUS_TIMEOUT).  Within a CTA: warp 10 waits for the counters ahead of
// the others (a look at one, and the proxy fence, take over 1000 clocks), warp
// 0 loads, warp 1 issues the MMAs, warps 2..9 are the epilogue of the previous
// tile out of the other half of TMEM (the scheme of gemm.cu).  Stores by TMA:
// with plain stores and the release that has to follow them 24 x 1024 x 1024 took
// 1.09 times as long.
#include "common.cuh"
#include "orthogonal.cuh"
#include "tcgen05.cuh"

#include <cmath>
#include <mutex>

namespace bs {
namespace {

constexpr int kEpiWarps = 8;
constexpr int kThreadsO = 96 + 32 * kEpiWarps;
constexpr int kOK = 64;                   // K elements a stage
constexpr int kOperand = 128 * kOK * 2;   // bytes of one operand a stage and CTA
constexpr int kStageO = 2 * kOperand;
constexpr int kBoxO = 32 * 32 * 2;        // an epilogue staging box: 32 x 32 elements

enum { kGram = 0, kPoly = 1, kApply = 2 };

// The tensor maps of one call: X of even and odd steps, S, P and the result.
// k, mn: operand boxes, K-major 64 x 128 and MN-major 64 x 64; st: 32 x 32
// store boxes; mi: those of the transposed copies (not swizzled).
struct OrthMaps {
  CUtensorMap xk[2], xmn[2], xst[2], sk, sst, smi, pk, pst, pmi, out;
};
struct OrthParams {
  int64_t R, C, m, batch;   // X is [R, C], S and P [m, m], m = min(R, C)
  int steps, tall;
  int sym_tiles;            // tiles of S on and below the diagonal
  int app_mt, app_nt;       // blocks of X
  int tiles;                // of the whole call
  uint16_t *out;            // written directly where TMA cannot (out_tma 0)
  int out_tma;
  const uint16_t *S;
  int64_t lds, ss;
  uint32_t *done;           // [3 steps][batch]: finished epilogue warps
  uint32_t polls;           // limit of every wait
  int32_t *status;
  OrthSteps s;
};

// CG CTAs share a tile of 128 CG rows and 128 CG columns.
template <int CG>
struct OrthCfg {
  static constexpr int T = 128 * CG;
  static constexpr uint32_t COLS = T;  // TMEM columns of an accumulator
  // 4 and 6 stages measure alike (back to back 24 x 1024 x 1024: 685 and 694 us;
  // 4096 x 4096: 1324 and 1306): the main loop takes about 780 clocks for the 512
  // of a stage's MMAs because 32 KB a stage come in at 42 bytes a clock, not
  // because they come late.
  static constexpr int NST = 6;
  static constexpr int EPI = kEpiWarps * 2 * kBoxO;  // a box and a transposed one a warp
  static constexpr size_t SMEM = 1024 + (size_t)NST * kStageO + EPI + 256;
};

// One operand of a stage: 128 rows (M or N) x 64 of K.  K-major: one box of
// 64 x 128; MN-major: two boxes of 64 (M or N) x 64 (K).
template <int CG, bool MN>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap *map, int k, int mn,
                                             int z, uint32_t bar) {
  if constexpr (MN) {
#pragma unroll
    for (int j = 0; j < 2; ++j) tma_load_3d_at<CG>(dst + j * 8192, map, mn + 64 * j, k, z, bar);
  } else {
    tma_load_3d_at<CG>(dst, map, k, mn, z, bar);
  }
}
// Low word's K slice step (>> 4) and the other bits of an operand's
// descriptor: K-major, 128-byte rows in 8-row atoms 1024 B apart, 32 B for 16
// of K; MN-major, 64-wide atoms 8 KB apart, 8-row K groups 1024 B apart, 2048 B
// for 16 of K.
template <bool MN>
constexpr uint32_t slice_step() { return (MN ? 2048 : 32) >> 4; }
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t base) {
  return MN ? smem_desc(base, 8192, 1024) : smem_desc(base, 16, 1024);
}

__device__ __forceinline__ bool bounded_wait(uint64_t *bar, uint32_t parity,
                                             const OrthParams &P) {
  for (uint32_t n = 0; n < P.polls; ++n)
    if (mbar_try_wait(bar, parity)) return true;
  status_or(P.status, BS_STATUS_TIMEOUT);
  return false;
}
__device__ __forceinline__ uint32_t ld_acquire_u32(const uint32_t *p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// A tile of the whole call's order.
struct Tile {
  int step, mode, z, mb, nb;
  bool amn, bmn;  // MN-major operands
};
__device__ __forceinline__ Tile find_tile(const OrthParams &P, int tile) {
  Tile w;
  const uint32_t sym = (uint32_t)P.batch * P.sym_tiles, one = (uint32_t)P.app_mt * P.app_nt;
  const uint32_t per = 2 * sym + (uint32_t)P.batch * one;
  uint32_t t = (uint32_t)tile;
  w.step = (int)(t / per);
  t -= (uint32_t)w.step * per;
  w.mode = t < sym ? kGram : t < 2 * sym ? kPoly : kApply;
  if (w.mode == kApply) {
    t -= 2 * sym;
    w.z = (int)(t / one);
    t -= (uint32_t)w.z * one;
    // groups of kGroupM row blocks sweep the column blocks together
    const uint32_t group = (uint32_t)kGroupM * P.app_nt, g = t / group;
    const uint32_t rows = min((uint32_t)kGroupM, (uint32_t)P.app_mt - g * kGroupM);
    t -= g * group;
    w.nb = (int)(t / rows);
    w.mb = (int)(g * kGroupM + t % rows);
  } else {
    if (w.mode == kPoly) t -= sym;
    w.z = (int)(t / (uint32_t)P.sym_tiles);
    const int i = (int)(t - (uint32_t)w.z * P.sym_tiles);
    int64_t r = (int64_t)((sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) / 2 > i) --r;
    while ((r + 1) * (r + 2) / 2 <= i) ++r;
    w.mb = (int)r;
    w.nb = (int)(i - r * (r + 1) / 2);
  }
  // S = X X^T (K-major both) or X^T X (MN-major both); S S; P X or X P
  w.amn = w.mode == kGram && P.tall;
  w.bmn = w.mode == kGram ? P.tall != 0 : w.mode == kApply && !P.tall;
  return w;
}
__device__ __forceinline__ int64_t k_of(const OrthParams &P, const Tile &w) {
  return w.mode == kGram ? (P.tall ? P.R : P.C) : P.m;
}
// Finished epilogue warps of matrix w.z in the phase before w, when complete.
template <int CG>
__device__ __forceinline__ uint32_t before(const OrthParams &P, const Tile &w,
                                           const uint32_t **at) {
  const int phase = 3 * w.step + w.mode;
  *at = P.done + (int64_t)(phase - 1) * P.batch + w.z;
  return phase == 0 ? 0u
                    : (uint32_t)(kEpiWarps * CG * (w.mode == kGram ? P.app_mt * P.app_nt : P.sym_tiles));
}

// Waits until phase w's predecessor is complete for its matrix.
template <int CG>
__device__ __forceinline__ bool phase_done(const OrthParams &P, const Tile &w) {
  const uint32_t *at;
  const uint32_t want = before<CG>(P, w, &at);
  if (want == 0) return true;
  for (uint32_t n = 0; n < P.polls; ++n) {
    if (ld_acquire_u32(at) >= want) {
      // the tiles were written, and are read, by the async proxy
      asm volatile("fence.proxy.async;" ::: "memory");
      return true;
    }
    __nanosleep(32);
  }
  status_or(P.status, BS_STATUS_TIMEOUT);
  return false;
}

// Waits until warp 10 has seen that this CTA's tile j may be loaded.
__device__ __forceinline__ bool tile_cleared(const OrthParams &P, const uint32_t *cleared,
                                             uint32_t j) {
  for (uint32_t n = 0; n < P.polls; ++n) {
    uint32_t v;
    asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(v) : "r"(saddr(cleared)) : "memory");
    if (v == ~0u) return false;
    if (v > j) return true;
    __nanosleep(20);
  }
  status_or(P.status, BS_STATUS_TIMEOUT);
  return false;
}

// Position in the ring of stages: stage, parity of its next use.
template <int N>
struct Ring {
  uint32_t s = 0, phase = 0, laps = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      phase ^= 1;
      laps = 1;
    }
  }
  __device__ __forceinline__ bool used() const { return laps != 0; }
};

// The loads of a tile (all lanes call).
template <int CG, bool AMN, bool BMN, class R>
__device__ __forceinline__ bool produce(const OrthParams &P, R &ring, uint8_t *smem,
                                        uint64_t *full, uint64_t *empty, const CUtensorMap *ma,
                                        const CUtensorMap *mb, int nk, int am, int bn, int z) {
  const bool one = (threadIdx.x & 31) == 0;
  const bool leader = CG == 1 || cluster_rank() == 0;
  const uint32_t base = saddr(smem), bars = saddr(full);
  const uint32_t lead_bars = CG == 2 ? map_rank(bars, 0) : bars;
  for (int kb = 0; kb < nk; ++kb, ring.next()) {
    if (ring.used() && !bounded_wait(&empty[ring.s], ring.phase ^ 1, P)) return false;
    const uint32_t a = base + ring.s * kStageO, bar = lead_bars + 8 * ring.s;
    if (one) {
      if (leader) mbar_expect_tx(&full[ring.s], CG * kStageO);
      load_operand<CG, AMN>(a, ma, kb * kOK, am, z, bar);
      load_operand<CG, BMN>(a + kOperand, mb, kb * kOK, bn, z, bar);
    }
    __syncwarp();
  }
  return true;
}
// The products of a tile into TMEM at d (all lanes of the leader's warp call).
template <int CG, bool AMN, bool BMN, class R>
__device__ __forceinline__ bool issue(const OrthParams &P, R &ring, uint8_t *smem, uint64_t *full,
                                      uint64_t *empty, uint32_t d, int nk) {
  constexpr int T = OrthCfg<CG>::T;
  // fp32 accumulator, fp16 A and B, their major-ness, N, M
  constexpr uint32_t IDESC = (1u << 4) | ((AMN ? 1u : 0u) << 15) | ((BMN ? 1u : 0u) << 16) |
                             ((uint32_t)(T >> 3) << 17) | ((uint32_t)(T >> 4) << 24);
  const bool one = (threadIdx.x & 31) == 0;
  const uint64_t ad0 = operand_desc<AMN>(saddr(smem));
  const uint64_t bd0 = operand_desc<BMN>(saddr(smem) + kOperand);
  const uint32_t free0 = saddr(empty), free1 = CG == 2 ? map_rank(free0, 1) : free0;
  for (int kb = 0; kb < nk; ++kb, ring.next()) {
    if (!bounded_wait(&full[ring.s], ring.phase, P)) return false;
    tc_fence_after();
    const uint64_t ad = ad0 + ring.s * (kStageO >> 4), bd = bd0 + ring.s * (kStageO >> 4);
    if (one) {
#pragma unroll
      for (int k = 0; k < kOK / 16; ++k)
        mma_bf16<CG>(d, ad + k * slice_step<AMN>(), bd + k * slice_step<BMN>(), IDESC,
                     (kb > 0 || k > 0) ? 1u : 0u);
      // the stage is free (in both CTAs) once these MMAs have read it
      mma_commit_to<CG>(free0 + 8 * ring.s);
      if constexpr (CG == 2) mma_commit_to<CG>(free1 + 8 * ring.s);
    }
    __syncwarp();
  }
  return true;
}

// kThreadsO threads; see the head of the file.
template <int CG>
__global__ void __launch_bounds__(kThreadsO, 1)
    orth_kernel(const __grid_constant__ OrthMaps maps, const __grid_constant__ OrthParams P) {
  using G = OrthCfg<CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *epi = smem + (size_t)G::NST * kStageO;
  uint64_t *full = reinterpret_cast<uint64_t *>(epi + G::EPI);
  uint64_t *empty = full + G::NST;
  uint64_t *acc_full = empty + G::NST;
  uint64_t *acc_empty = acc_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  uint32_t *cleared = tmem_slot + 1;  // tiles of this CTA that may be loaded; ~0: given up

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const bool leader = rank == 0;
  const int cid = (int)blockIdx.x / CG, ncl = (int)gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::NST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps * CG);
    }
    *cleared = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       saddr(tmem_slot)),
                   "r"(2 * G::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       saddr(tmem_slot)),
                   "r"(2 * G::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Producer and issuer: the whole warp walks the loop, so that stages, phases
  // and descriptors are warp-uniform, and one lane issues.
  if (warp == 0) {
    Ring<G::NST> ring;
    uint32_t j = 0;
    for (int t = cid; t < P.tiles; t += ncl, ++j) {
      const Tile w = find_tile(P, t);
      const CUtensorMap *ma, *mb;
      const int odd = w.step & 1;
      if (w.mode == kGram) ma = mb = P.tall ? &maps.xmn[odd] : &maps.xk[odd];
      else if (w.mode == kPoly) ma = mb = &maps.sk;
      else if (P.tall) ma = &maps.xk[odd], mb = &maps.pk;
      else ma = &maps.pk, mb = &maps.xmn[odd];
      if (!tile_cleared(P, cleared, j)) break;
      const int am = (int)(w.mb * G::T + rank * 128), bn = (int)(w.nb * G::T + rank * 128);
      const int nk = (int)((k_of(P, w) + kOK - 1) / kOK), z = w.z;
      bool ok;
      if (w.amn) ok = produce<CG, true, true>(P, ring, smem, full, empty, ma, mb, nk, am, bn, z);
      else if (w.bmn)
        ok = produce<CG, false, true>(P, ring, smem, full, empty, ma, mb, nk, am, bn, z);
      else ok = produce<CG, false, false>(P, ring, smem, full, empty, ma, mb, nk, am, bn, z);
      if (!ok) break;
    }
    // every copy landed before the CTA may exit (the leader's barriers count
    // the peer's copies too)
    if (leader)
      for (int i = 0; i < G::NST; ++i, ring.next())
        if (ring.used()) bounded_wait(&full[ring.s], ring.phase ^ 1, P);
  } else if (warp == 2 + kEpiWarps) {
    uint32_t j = 0;
    for (int t = cid; t < P.tiles; t += ncl) {
      const bool ok = phase_done<CG>(P, find_tile(P, t));
      j = ok ? j + 1 : ~0u;
      asm volatile("st.release.cta.shared.u32 [%0], %1;" ::"r"(saddr(cleared)), "r"(j) : "memory");
      if (!ok) break;
    }
  } else if (warp == 1) {
    if (leader) {
      Ring<G::NST> ring;
      int j = 0;
      for (int t = cid; t < P.tiles; t += ncl, ++j) {
        const Tile w = find_tile(P, t);
        const int nk = (int)((k_of(P, w) + kOK - 1) / kOK);
        const int buf = j & 1;
        if (j >= 2 && !bounded_wait(&acc_empty[buf], (uint32_t)(((j >> 1) - 1) & 1), P)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)buf * G::COLS;
        bool ok;
        if (w.amn) ok = issue<CG, true, true>(P, ring, smem, full, empty, d, nk);
        else if (w.bmn) ok = issue<CG, false, true>(P, ring, smem, full, empty, d, nk);
        else ok = issue<CG, false, false>(P, ring, smem, full, empty, d, nk);
        if (!ok) break;
        if (lane == 0) {
          mma_commit_to<CG>(saddr(&acc_full[buf]));
          if constexpr (CG == 2) mma_commit_to<CG>(map_rank(saddr(&acc_full[buf]), 1));
        }
        __syncwarp();
      }
    }
  } else {
    // epilogue: warp w has TMEM lanes 32 (w % 4) .. + 31, one row a lane, and
    // one half of the tile's columns
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t *box = epi + (size_t)(warp - 2) * 2 * kBoxO, *tbox = box + kBoxO;
    const uint32_t acc_empty_leader = map_rank(saddr(acc_empty), 0);
    int j = 0;
    for (int t = cid; t < P.tiles; t += ncl, ++j) {
      const Tile w = find_tile(P, t);
      const OrthStep st = P.s.step[w.step];
      const bool poly = w.mode == kPoly, last = w.mode == kApply && w.step + 1 == P.steps;
      const bool mirror = w.mode != kApply && w.mb != w.nb, tma = !last || P.out_tma;
      const int64_t M = w.mode == kApply ? P.R : P.m, N = w.mode == kApply ? P.C : P.m;
      const float alpha = w.mode == kGram ? st.gram : poly ? st.pc : st.apply;
      const CUtensorMap *mc = w.mode == kGram ? &maps.sst
                              : poly          ? &maps.pst
                              : last          ? &maps.out
                                              : &maps.xst[(w.step & 1) ^ 1];
      const CUtensorMap *mt = w.mode == kGram ? &maps.smi : &maps.pmi;
      const int64_t row0 = (int64_t)w.mb * G::T + rank * 128 + 32 * q, m = row0 + lane;
      const int64_t n0 = (int64_t)w.nb * G::T + half * (G::T / 2);
      const int buf = j & 1;
      // P reads its block of S, 32 columns ahead: lanes 4 i .. 4 i + 3 hold the
      // 64 bytes of rows i, i + 8, i + 16 and i + 24
      uint4 sv[4];
      auto fetch = [&](int64_t n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t r = row0 + 8 * i + (lane >> 2), c = n + 8 * (lane & 3);
          sv[i] = make_uint4(0, 0, 0, 0);
          if (r < M && c < N)  // rows are padded to whole vectors
            sv[i] = __ldcg(reinterpret_cast<const uint4 *>(P.S + w.z * P.ss + r * P.lds + c));
        }
      };
      if (poly) {  // complete when this tile's loads may start
        if (!phase_done<CG>(P, w)) break;
        fetch(n0);
      }
      if (!bounded_wait(&acc_full[buf], (uint32_t)((j >> 1) & 1), P)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)buf * G::COLS +
                             (uint32_t)(half * (G::T / 2));
      uint32_t r[2][32];
      tmem_ld32_nowait(tbase, r[0]);
#pragma unroll
      for (int c = 0; c < G::T / 64; ++c) {  // 32 columns at a time
        tmem_wait_ld();
        if (c + 1 < G::T / 64) {
          tmem_ld32_nowait(tbase + 32 * (c + 1), r[(c + 1) & 1]);
        } else {  // the accumulator is read: hand it back
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_peer(acc_empty_leader + (uint32_t)(8 * buf));
        }
        const int64_t n = n0 + 32 * c;
        if (lane == 0)  // the stores that last read the boxes are done reading
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        // A box has 64-byte rows, its 16-byte chunks swizzled as the store's
        // tensor map says: chunk i of row k at i ^ (k / 2 % 4).
        uint8_t *mine = box + lane * 64;
        const int swz = (lane >> 1) & 3;
        uint32_t s2[16];
        if (poly) {  // S through the box: from rows across lanes to a row a lane
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4 *>(box + (8 * i + (lane >> 2)) * 64 +
                                       (((lane & 3) ^ ((lane >> 3) & 3)) * 16)) = sv[i];
          __syncwarp();
          if (c + 1 < G::T / 64) fetch(n + 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4 *>(mine + ((i ^ swz) * 16));
            s2[4 * i] = v.x;
            s2[4 * i + 1] = v.y;
            s2[4 * i + 2] = v.z;
            s2[4 * i + 3] = v.w;
          }
        }
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v0 = alpha * __uint_as_float(r[c & 1][2 * i]);
          float v1 = alpha * __uint_as_float(r[c & 1][2 * i + 1]);
          if (poly) {
            v0 = fmaf(st.pb, f16_lo(s2[i]), v0);
            v1 = fmaf(st.pb, f16_hi(s2[i]), v1);
            if (m == n + 2 * i) v0 += st.pa;
            if (m == n + 2 * i + 1) v1 += st.pa;
          }
          o[i] = last ? bf16x2_from_f32(v0, v1) : f16x2_rn(v0, v1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4 *>(mine + ((i ^ swz) * 16)) =
              make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        if (tma) {
          if (mirror) {
            // rows n + i of the transposed box: 32 columns m, 64 bytes.  Two
            // lanes exchange halves: the even one has row 2 i of both, the
            // odd one row 2 i + 1; 16 + 16 words, all banks once.
            uint32_t *tb = reinterpret_cast<uint32_t *>(tbox) + (lane & 1) * 16 + (lane >> 1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, o[i], 1);
              tb[2 * i * 16] = lane & 1 ? __byte_perm(other, o[i], 0x7632)
                                        : __byte_perm(o[i], other, 0x5410);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && n < N && row0 < M) {
            asm volatile(
                "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                ::"l"(reinterpret_cast<uint64_t>(mc)), "r"((int)n), "r"((int)row0), "r"(w.z),
                "r"(saddr(box))
                : "memory");
            if (mirror)
              asm volatile(
                  "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], "
                  "[%4];" ::"l"(reinterpret_cast<uint64_t>(mt)),
                  "r"((int)row0), "r"((int)n), "r"(w.z), "r"(saddr(tbox))
                  : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {  // rows that do not start on 16 bytes: a row of the box at a time
          __syncwarp();
          uint16_t *out = P.out + (w.z * P.R + row0) * P.C + n + lane;
          const int rows = M - row0 < 32 ? (int)(M - row0) : 32;
          if (n + lane < N)
            for (int k = 0; k < rows; ++k)
              out[(int64_t)k * P.C] = *reinterpret_cast<const uint16_t *>(
                  box + k * 64 + (((lane >> 3) ^ ((k >> 1) & 3)) * 16) + (lane & 7) * 2);
          __syncwarp();
        }
      }
      if (lane == 0 && !last) {
        // the tile's stores are complete, and other CTAs may read it
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(
                         P.done + (int64_t)(3 * w.step + w.mode) * P.batch + w.z)
                     : "memory");
      }
    }
  }
  if (warp >= 2 && warp < 2 + kEpiWarps && lane == 0)
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(2 * G::COLS)
                   : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(2 * G::COLS)
                   : "memory");
  }
}

// ---------------------------------------------------------------------------
// The division by the norm: sums of squares (a fixed partition, no atomics),
// then X = fp16(G * scale / (norm + eps)).
// ---------------------------------------------------------------------------
// Eight values of a row from column c, as read (VEC: 16-byte loads; the second
// only of fp32) and as fp32, zeros past the row's end.
template <bool VEC>
struct Eight {
  uint4 a, b;
  float f[8];
  __device__ __forceinline__ void load(const OrthInput &I, int64_t row_at, int64_t c) {
    if constexpr (VEC) {
      if (I.dt == BS_F32) {
        a = ld_nc_v4(static_cast<const float *>(I.g) + row_at + c);
        b = ld_nc_v4(static_cast<const float *>(I.g) + row_at + c + 4);
      } else {
        a = ld_nc_v4(static_cast<const uint16_t *>(I.g) + row_at + c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i < I.C ? input_at(I, row_at + c + i) : 0.f;
    }
  }
  __device__ __forceinline__ void widen(const OrthInput &I) {
    if constexpr (VEC) {
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if (I.dt == BS_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  }
};
// f(values, row, column) for this thread's vectors of matrix z, four loads in
// flight; `reverse`: the last first (what was read last is still in L2).
template <bool VEC, class F>
__device__ __forceinline__ void each_vector(const OrthInput &I, int64_t z, bool reverse, F f) {
  constexpr int U = VEC ? 4 : 1;
  const uint32_t vecs = (uint32_t)((I.C + 7) / 8);
  const int64_t total = I.R * vecs, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i0 < total; i0 += U * step) {
    Eight<VEC> v[U];
    int64_t row[U];
    uint32_t col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = i0 + u * step;
      if (at >= total) continue;
      const int64_t i = reverse ? total - 1 - at : at;
      row[u] = total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / vecs) : i / vecs;
      col[u] = (uint32_t)(i - row[u] * vecs) * 8;
      v[u].load(I, z * I.sb + row[u] * I.ld, col[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * step >= total) continue;
      v[u].widen(I);
      f(v[u].f, row[u], (int64_t)col[u]);
    }
  }
}

constexpr int kThreadsN = 256;
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[kThreadsN / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kThreadsN / 32; ++i) s += part[i];
  return s;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreadsN)
    orth_norm_kernel(const OrthInput I, float *part, uint32_t *done, int phases) {
  if (blockIdx.x == 0)  // this matrix's counters of the products, which come after
    for (int i = threadIdx.x; i < phases; i += kThreadsN)
      done[(int64_t)i * gridDim.y + blockIdx.y] = 0;
  const int64_t z = blockIdx.y;
  float s = 0.f;
  each_vector<VEC>(I, z, false, [&](const float(&f)[8], int64_t, int64_t) {
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(f[k], f[k], s);
  });
  s = block_sum(s);
  if (threadIdx.x == 0) part[z * gridDim.x + blockIdx.x] = s;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreadsN)
    orth_cast_kernel(const OrthInput I, const float *part, int parts, float scale, float eps,
                     uint16_t *x, int64_t ldx, int64_t sx) {
  const int64_t z = gridDim.y - 1 - blockIdx.y;
  float sum = 0.f;
  for (int i = threadIdx.x; i < parts; i += kThreadsN) sum += part[z * parts + i];
  const float f0 = scale / (sqrtf(block_sum(sum)) + eps);
  each_vector<VEC>(I, z, true, [&](const float(&f)[8], int64_t r, int64_t c) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = f16x2_rn(f[2 * k] * f0, f[2 * k + 1] * f0);
    st_v4(x + z * sx + r * ldx + c, make_uint4(w[0], w[1], w[2], w[3]));
  });
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
// [batch, rows, cols] of 16-bit elements, cols contiguous.
bool map3(CUtensorMap *map, const void *base, bool bf16, int64_t batch, int64_t rows, int64_t cols,
          int64_t ld, int64_t sb, uint32_t box_cols, uint32_t box_rows, int swizzle) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)sb * 2};
  const cuuint32_t box[3] = {box_cols, box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                swizzle == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                : CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

template <int CG>
int launch_orth(const OrthMaps &maps, OrthParams &P, cudaStream_t st) {
  using G = OrthCfg<CG>;
  static_assert(G::SMEM <= 227 * 1024, "shared memory of one CTA");
  auto kernel = orth_kernel<CG>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsO);
  cfg.dynamicSmemBytes = G::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeCooperative;  // all CTAs resident: they wait for one another
  attr[1].val.cooperative = 1;
  cfg.attrs = attr;
  // The shared-memory attribute is per device, and so is the number of
  // clusters that are resident at once: set up once for each device.
  constexpr int kMaxDev = 64;
  static std::mutex mu;
  static int slots_of[kMaxDev] = {};
  int dev = 0;
  int64_t slots;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return BS_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!slots_of[dev]) {
      int n = 0, sms = 0;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)G::SMEM) != cudaSuccess ||
          cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return BS_ERR_LAUNCH;
      cfg.gridDim = dim3((unsigned)(sms / CG * CG));
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0)
        return BS_ERR_LAUNCH;
      slots_of[dev] = n < sms / CG ? n : sms / CG;
    }
    slots = slots_of[dev];
  }
  // CTAs beyond the largest phase's tiles would only wait
  const int64_t sym = P.batch * P.sym_tiles, app = P.batch * P.app_mt * P.app_nt;
  const int64_t most = sym > app ? sym : app;
  const int64_t tiles = P.steps * (2 * sym + app);
  if (tiles >= ((int64_t)1 << 30)) return BS_ERR_TOO_LARGE;
  P.tiles = (int)tiles;
  cfg.gridDim = dim3((unsigned)(CG * (most < slots ? most : slots)));
  cfg.numAttrs = 2;
  return launch_code(cudaLaunchKernelEx(&cfg, kernel, maps, P));
}

bool set_tiles(OrthParams &P, int64_t T) {
  const int64_t t = (P.m + T - 1) / T, mt = (P.R + T - 1) / T, nt = (P.C + T - 1) / T;
  if (t > 1 << 14 || mt * nt >= ((int64_t)1 << 30)) return false;
  P.sym_tiles = (int)(t * (t + 1) / 2);
  P.app_mt = (int)mt;
  P.app_nt = (int)nt;
  return true;
}
// CTA pairs on 256 x 256 tiles where those are enough to keep 64 pairs busy in
// every phase and their ragged edges cost less than the pairs gain; else 128 x
// 128 tiles.  Back to back, singles against pairs: on whole tiles 24 x 1024 x 1024
// 900 and 694 us, 4096 x 4096 1802 and 1306; where pairs compute 1.44 times as much,
// 24 x 600 x 1300, 585 and 518; at 1.53 times, 24 x 640 x 640 285 and 291, 48 x 520 x
// 520 555 and 525; above, 24 x 384 x 384 135 and 169, 24 x 300 x 300 132 and 162.  With
// fewer than 64 pair tiles a phase's latency decides (4 x 1024 x 1024: 191 and 218).
int run_orth(const OrthMaps &maps, OrthParams &P, cudaStream_t st) {
  if (!set_tiles(P, 128)) return BS_ERR_TOO_LARGE;
  auto products = [&](double tile) {  // of a step, by the tiles' areas
    const double n = (double)(P.tall ? P.R : P.C), m = (double)P.m;
    return tile * tile * (P.sym_tiles * (n + m) + (double)P.app_mt * P.app_nt * m);
  };
  const double single = products(128);
  if (!set_tiles(P, 256)) return BS_ERR_TOO_LARGE;
  if (P.batch * P.sym_tiles >= 64 && products(256) <= 1.57 * single)
    return launch_orth<2>(maps, P, st);
  set_tiles(P, 128);
  return launch_orth<1>(maps, P, st);
}

int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
// CTAs of the norm and the cast for a matrix.
int64_t norm_parts(int64_t batch, int64_t R, int64_t C) {
  const int64_t all = (R * ((C + 7) / 8) + 4 * kThreadsN - 1) / (4 * kThreadsN);
  const int64_t most = (148 * 8 + batch - 1) / batch;
  return all < most ? all : most;
}
struct OrthLayout {
  size_t x0, x1, s, p, part, done, bytes;
};
OrthLayout orth_layout(int64_t batch, int64_t R, int64_t C) {
  const int64_t m = R < C ? R : C;
  auto round = [](int64_t b) { return (size_t)((b + 255) / 256 * 256); };
  OrthLayout L = {};
  L.x0 = 0;
  L.x1 = L.x0 + round(batch * R * up8(C) * 2);
  L.s = L.x1 + round(batch * R * up8(C) * 2);
  L.p = L.s + round(batch * m * up8(m) * 2);
  L.part = L.p + round(batch * m * up8(m) * 2);
  L.done = L.part + round(batch * norm_parts(batch, R, C) * 4);
  L.bytes = L.done + round(batch * 3 * kMaxSteps * 4);
  return L;
}

// The largest |a s + b s^3 + c s^5| over 0 <= s <= top, and the largest
// |a + b t + c t^2| over t = s^2: at the ends or where the slope is zero.
double bound_step(double a, double b, double c, double top, double *poly) {
  const double T = top * top;
  auto p = [&](double t) { return std::fabs(a + t * (b + t * c)); };
  auto f = [&](double t) { return std::sqrt(t) * p(t); };
  *poly = std::fmax(p(0), p(T));
  if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < T) *poly = std::fmax(*poly, p(-b / (2 * c)));
  double most = f(T);
  auto at = [&](double t) {
    if (t > 0 && t < T) most = std::fmax(most, f(t));
  };
  if (c != 0) {  // a + 3 b t + 5 c t^2 = 0
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      at((-3 * b + std::sqrt(d)) / (10 * c));
      at((-3 * b - std::sqrt(d)) / (10 * c));
    }
  } else if (b != 0) {
    at(-a / (3 * b));
  }
  return most;
}
// The power of two that takes `bound` to 2^14 at most.
double scale_for(double bound) { return bound > 0 ? std::exp2(14 - std::ceil(std::log2(bound))) : 1; }

}  // namespace
}  // namespace bs

using namespace bs;

extern "C" size_t bs_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  return orth_layout(batch, rows, cols).bytes;
}

extern "C" int bs_orthogonalize(const void *g, int dtype, int64_t batch, int64_t rows,
                                int64_t cols, int64_t ld, int64_t batch_stride, int steps,
                                const float *coefficients, float eps, void *out, void *ws,
                                size_t ws_bytes, int32_t *status, void *stream) {
  if (batch < 0 || rows < 0 || cols < 0) return BS_ERR_SHAPE;
  if (dtype != BS_BF16 && dtype != BS_F32) return BS_ERR_DTYPE;
  if (steps < 1 || steps > kMaxSteps || !coefficients || !(eps > 0.f)) return BS_ERR_ARG;
  if (batch == 0 || rows == 0 || cols == 0) return BS_OK;
  if (rows >= ((int64_t)1 << 30) || cols >= ((int64_t)1 << 30) || batch >= ((int64_t)1 << 16))
    return BS_ERR_TOO_LARGE;
  if (ld < cols || batch_stride < 0) return BS_ERR_SHAPE;
  if (!g || !out || !ws) return BS_ERR_ARG;
  const int eb = dtype == BS_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(g) & (uintptr_t)(eb - 1)) ||
      (reinterpret_cast<uintptr_t>(out) & 1) || (reinterpret_cast<uintptr_t>(ws) & 255))
    return BS_ERR_ALIGN;
  const OrthLayout L = orth_layout(batch, rows, cols);
  if (ws_bytes < L.bytes) return BS_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t *base = static_cast<uint8_t *>(ws);
  const int64_t m = rows < cols ? rows : cols;
  const bool tall = rows > cols;
  const int64_t ldx = up8(cols), sx_ = rows * ldx, lds = up8(m), ss_ = m * lds;
  uint16_t *X[2] = {reinterpret_cast<uint16_t *>(base + L.x0),
                    reinterpret_cast<uint16_t *>(base + L.x1)};
  uint16_t *S = reinterpret_cast<uint16_t *>(base + L.s);
  uint16_t *Pm = reinterpret_cast<uint16_t *>(base + L.p);
  // singular values that could grow past 10^6 are refused: scaled for that
  // bound, smaller ones would lose their low bits
  OrthParams P = {};
  double top = 1, sx = scale_for(top);
  const double sx0 = sx;
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    double poly = 0;
    const double next = bound_step(a, b, c, top, &poly);
    if (!(next <= 1e6) || !(poly <= 1e6)) return BS_ERR_ARG;
    const double ss = scale_for(top * top), sp = scale_for(poly), sn = scale_for(next);
    P.s.step[i].gram = (float)(ss / (sx * sx));
    P.s.step[i].pa = (float)(sp * a);
    P.s.step[i].pb = (float)(sp * b / ss);
    P.s.step[i].pc = (float)(sp * c / (ss * ss));
    P.s.step[i].apply = (float)((i + 1 == steps ? 1 : sn) / (sp * sx));
    top = next;
    sx = sn;
  }
  const OrthInput I = {g, dtype, rows, cols, ld, batch_stride};
  if (m <= kSmallM && (tall ? rows : cols) <= kSmallN)
    return orth_small(I, batch, steps, P.s, (float)sx0, eps, static_cast<uint16_t *>(out), status,
                      st);
  OrthMaps T;
  bool ok = true;
  for (int i = 0; i < 2; ++i)
    ok = ok && map3(&T.xk[i], X[i], false, batch, rows, cols, ldx, sx_, kOK, 128, 128) &&
         map3(&T.xmn[i], X[i], false, batch, rows, cols, ldx, sx_, 64, kOK, 128) &&
         map3(&T.xst[i], X[i], false, batch, rows, cols, ldx, sx_, 32, 32, 64);
  ok = ok && map3(&T.sk, S, false, batch, m, m, lds, ss_, kOK, 128, 128) &&
       map3(&T.sst, S, false, batch, m, m, lds, ss_, 32, 32, 64) &&
       map3(&T.smi, S, false, batch, m, m, lds, ss_, 32, 32, 0) &&
       map3(&T.pk, Pm, false, batch, m, m, lds, ss_, kOK, 128, 128) &&
       map3(&T.pst, Pm, false, batch, m, m, lds, ss_, 32, 32, 64) &&
       map3(&T.pmi, Pm, false, batch, m, m, lds, ss_, 32, 32, 0);
  if (!ok) return BS_ERR_LAUNCH;
  P.out_tma = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && cols % 8 == 0 &&
              map3(&T.out, out, true, batch, rows, cols, cols, rows * cols, 32, 32, 64);
  if (!P.out_tma) T.out = T.xst[0];  // unused
  P.R = rows; P.C = cols; P.m = m; P.batch = batch; P.steps = steps; P.tall = tall;
  P.out = static_cast<uint16_t *>(out);
  P.S = S; P.lds = lds; P.ss = ss_;
  P.done = reinterpret_cast<uint32_t *>(base + L.done);
  P.status = status;
  // a wait lasts as long as the tiles before it: the limit is far above the
  // call's time at 100 TFLOP/s, at 20 ns a poll
  const double us = (double)steps * batch * m * m * (2.0 * m + 4.0 * (tall ? rows : cols)) / 1e8;
  P.polls = (uint32_t)std::fmin(4e9, 2097152.0 + 200.0 * us);

  float *part = reinterpret_cast<float *>(base + L.part);
  const int64_t parts = norm_parts(batch, rows, cols);
  const bool vec = (reinterpret_cast<uintptr_t>(g) & 15) == 0 && cols % 8 == 0 &&
                   ld * eb % 16 == 0 && batch_stride * eb % 16 == 0;
  const dim3 grid((unsigned)parts, (unsigned)batch);
  if (vec) {
    orth_norm_kernel<true><<<grid, kThreadsN, 0, st>>>(I, part, P.done, 3 * steps);
    orth_cast_kernel<true><<<grid, kThreadsN, 0, st>>>(I, part, (int)parts, (float)sx0, eps, X[0],
                                                       ldx, sx_);
  } else {
    orth_norm_kernel<false><<<grid, kThreadsN, 0, st>>>(I, part, P.done, 3 * steps);
    orth_cast_kernel<false><<<grid, kThreadsN, 0, st>>>(I, part, (int)parts, (float)sx0, eps,
                                                        X[0], ldx, sx_);
  }
  if (cudaGetLastError() != cudaSuccess) return BS_ERR_LAUNCH;
  return run_orth(T, P, st);
}
