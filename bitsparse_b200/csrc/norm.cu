// Entry points of the residual join and norm: checks, the division of the
// backward's rows, the sums of the parameter gradients.  Kernels: norm.cuh.
#include "norm.cuh"

namespace bs {
namespace {

bool aligned(const void *p, int64_t ld, int bytes) {
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && (ld * bytes) % 16 == 0);
}
bool norm_type(int dt) { return dt == BS_BF16 || dt == BS_F32; }
bool base_ok(const void *p, int dt) {  // natural alignment of the elements
  return !(reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elt(dt) - 1));
}

// The checks that both directions share; fills P.
int norm_setup(NormParams &P, int x_dt, int y_dt, int64_t T, int64_t D, const void *w, int w_dt,
               int post, const void *pw, int pw_dt, const void *gate, int gate_dt,
               int64_t gate_rows, int gate_wide, int act, float skip, float branch, float eps) {
  if (T < 0 || D <= 0) return BS_ERR_SHAPE;
  if (T >= ((int64_t)1 << 31) || D >= ((int64_t)1 << 31) - 8192) return BS_ERR_TOO_LARGE;
  if (!norm_type(x_dt) || !norm_type(y_dt) || (x_dt == BS_BF16 && y_dt == BS_F32))
    return BS_ERR_DTYPE;
  if ((w && !norm_type(w_dt)) || (pw && !norm_type(pw_dt)) || (gate && !norm_type(gate_dt)))
    return BS_ERR_DTYPE;
  if ((w && !base_ok(w, w_dt)) || (pw && !base_ok(pw, pw_dt)) || (gate && !base_ok(gate, gate_dt)))
    return BS_ERR_ALIGN;
  if (pw && !post) return BS_ERR_ARG;
  if (gate && T > 0 && (gate_rows <= 0 || gate_rows > T || T % gate_rows)) return BS_ERR_SHAPE;
  if (gate && ((act != kActNone && act != kActSigmoid))) return BS_ERR_ARG;
  if (!(eps > 0.f)) return BS_ERR_ARG;
  P.w = w; P.w_dt = w_dt; P.pw = pw; P.pw_dt = pw_dt; P.post = post != 0;
  P.gate = gate; P.gate_dt = gate_dt; P.gate_rows = gate ? gate_rows : 1;
  P.gate_wide = gate_wide; P.act = act;
  P.T = T; P.D = (int)D; P.skip = skip; P.branch = branch; P.eps = eps;
  P.rcp_d = (float)(1.0 / (double)D);
  return BS_OK;
}
bool params_vec(const NormParams &P) {
  return P.D % 8 == 0 && aligned(P.w, 8, 2) && aligned(P.pw, 8, 2) &&
         (!P.gate_wide || aligned(P.gate, 8, 2));
}
// Rows an SM from which shifted rows' backward pays for the eight CTAs that share
// a range.
constexpr int64_t kShiftedRows = 4;
// The rows' form (see norm.cuh), given that they are aligned, or that all of
// them are contiguous on 16-byte bases.  Just under 4096 columns the ends of
// shifted rows would need the form for wider ones, one CTA an SM (8000 x 4095
// with a gate: 249 + 292 us, by single elements 144 + 207).
int rows_mode(bool vec, bool contiguous, int64_t D) {
  const int64_t width = row_width(D, kRowsShifted);
  return vec                                                          ? kRowsAligned
         : contiguous && width <= kBwdMaxD && (D > 4096 || width <= 4096) ? kRowsShifted
                                                                          : kRowsAny;
}

// How the backward divides its rows: about `want` CTAs.  With fewer gate
// groups than that a group is divided among several CTAs, whose column sums
// are added up afterwards; with many, a CTA takes whole groups and writes
// their gate gradients itself.
struct Chunks {
  int64_t chunks, chunk_rows, per_group, groups_per_chunk;
};
Chunks divide(int64_t T, int64_t div_rows, int64_t want) {
  Chunks c = {};
  if (want > T) want = T;
  const int64_t groups = T / div_rows;
  if (groups >= 4 * want) {
    c.groups_per_chunk = (groups + want - 1) / want;
    c.chunks = (groups + c.groups_per_chunk - 1) / c.groups_per_chunk;
  } else {
    const int64_t per = want / groups < 1 ? 1 : want / groups;
    c.chunk_rows = (div_rows + per - 1) / per;
    c.per_group = (div_rows + c.chunk_rows - 1) / c.chunk_rows;
    c.chunks = groups * c.per_group;
  }
  return c;
}
// Only a wide gate that several rows share has its gradient summed by columns:
// its groups divide the rows; else all rows are one group.
int64_t division(bool gate, int64_t gate_rows, int gate_wide, int64_t T) {
  return gate && gate_wide && gate_rows > 1 ? gate_rows : T;
}
// Shifted rows: eight CTAs share a range, which has to be of one gate group, and
// each has a row of every sum.  For widths of eight, which take this form only
// where a parameter is off its alignment, no more than the other forms have: the
// workspace does not know how the tensors lie, and with eight a group it was 113 MB
// for 4600 x 512 bf16 (4.7 MB) in groups of two.
bool shares_groups(int64_t groups, int64_t D, int64_t ctas, int64_t most) {
  return groups < 4 * (ctas / 8) && (D % 8 != 0 || 8 * groups <= most);
}
}  // namespace
}  // namespace bs

using namespace bs;

extern "C" int bs_residual_norm(const void *x, int x_dtype, int64_t ldx, const void *y,
                                int y_dtype, int64_t ldy, int64_t T, int64_t D, const void *w,
                                int w_dtype, int post, const void *post_w, int post_w_dtype,
                                const void *gate, int gate_dtype, int64_t gate_rows,
                                int gate_wide, int gate_act, float skip, float branch, float eps,
                                void *s, void *h, float *r_post, float *r_pre, int32_t *status,
                                void *stream) {
  NormParams P = {};
  const int rc = norm_setup(P, x_dtype, y_dtype, T, D, w, w_dtype, post, post_w, post_w_dtype,
                            gate, gate_dtype, gate_rows, gate_wide, gate_act, skip, branch, eps);
  if (rc != BS_OK) return rc;
  if (T == 0) return BS_OK;
  if (!x || !h || (!y && (post || gate)) || (y && !s)) return BS_ERR_ARG;
  if (ldx < D || (y && ldy < D)) return BS_ERR_SHAPE;
  if (!base_ok(x, x_dtype) || (y && !base_ok(y, y_dtype)) || (s && !base_ok(s, x_dtype)) ||
      !base_ok(h, y_dtype))
    return BS_ERR_ALIGN;
  P.x = x; P.y = y; P.ldx = ldx; P.ldy = ldy; P.s = s; P.h = h;
  P.r_post = post ? r_post : nullptr;
  P.r_pre = r_pre;
  P.status = status;
  const bool vec = params_vec(P) && aligned(x, ldx, elt(x_dtype)) &&
                   aligned(y, ldy, elt(y_dtype)) && aligned(s, D, elt(x_dtype)) &&
                   aligned(h, D, elt(y_dtype));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool contiguous = ldx == D && ldy == D && aligned(x, 8, 2) && aligned(y, 8, 2) &&
                          aligned(s, 8, 2) && aligned(h, 8, 2) &&
                          (!gate_wide || gate_rows > 1 || aligned(gate, 8, 2));
  const int mode = rows_mode(vec, contiguous, D);
  if (x_dtype == BS_F32 && y_dtype == BS_F32) return norm_forward_f32(P, mode, st);
  if (x_dtype == BS_F32) return norm_forward_mix(P, mode, st);
  return norm_forward_bf16(P, mode, st);
}

extern "C" size_t bs_residual_norm_workspace_bytes(int64_t T, int64_t D, int post, int has_gate,
                                                   int64_t gate_rows, int gate_wide) {
  int sms = 0;
  if (T <= 0 || D <= 0 || (has_gate && (gate_rows <= 0 || gate_rows > T || T % gate_rows)) ||
      sm_count(&sms) != BS_OK) return 0;
  // divide() gives at most `want` chunks, or one for each of fewer than 4 want
  // groups; shifted rows have eight for each while shares_groups()
  const int64_t want = most_ctas(D, sms);
  const int64_t groups = T / division(has_gate, gate_rows, gate_wide, T);
  const bool shifted = T >= kShiftedRows * (int64_t)sms;
  int64_t chunks = shifted || want < T ? want : T;
  if (groups < 4 * want && groups > chunks) chunks = groups;
  if (shifted && shares_groups(groups, D, want, want) && 8 * groups > chunks) chunks = 8 * groups;
  const int64_t planes = 1 + (post || has_gate ? 1 : 0) + (has_gate ? 1 : 0);
  return (size_t)(planes * chunks * D + (has_gate && !gate_wide ? T : 0)) * sizeof(float);
}

extern "C" int bs_residual_norm_backward(
    const void *ds, const void *dh, const void *s, int x_dtype, int64_t lds, const void *y,
    int y_dtype, int64_t ldy, int64_t T, int64_t D, const void *w, int w_dtype, int post,
    const void *post_w, int post_w_dtype, const void *gate, int gate_dtype, int64_t gate_rows,
    int gate_wide, int gate_act, float skip, float branch, float eps, const float *r_post,
    const float *r_pre, void *dx, void *dy, void *dw, void *dpost_w, void *dgate, void *ws,
    size_t ws_bytes, int32_t *status, void *stream) {
  NormParams P = {};
  const int rc = norm_setup(P, x_dtype, y_dtype, T, D, w, w_dtype, post, post_w, post_w_dtype,
                            gate, gate_dtype, gate_rows, gate_wide, gate_act, skip, branch, eps);
  if (rc != BS_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // sums over no rows
    if (dw && cudaMemsetAsync(dw, 0, (size_t)D * elt(w_dtype), st) != cudaSuccess)
      return BS_ERR_LAUNCH;
    if (dpost_w && cudaMemsetAsync(dpost_w, 0, (size_t)D * elt(post_w_dtype), st) != cudaSuccess)
      return BS_ERR_LAUNCH;
    return BS_OK;
  }
  if (!s || !r_pre || (post && !r_post) || ((post || gate) && !y)) return BS_ERR_ARG;
  if ((dw && !w) || (dpost_w && !post_w) || (dgate && !gate)) return BS_ERR_ARG;
  if (lds < D || ((post || gate) && ldy < D)) return BS_ERR_SHAPE;
  const void *of_x[] = {ds, s, dx}, *of_y[] = {dh, y, dy};
  for (const void *p : of_x)
    if (!base_ok(p, x_dtype)) return BS_ERR_ALIGN;
  for (const void *p : of_y)
    if (!base_ok(p, y_dtype)) return BS_ERR_ALIGN;
  if ((dw && !base_ok(dw, w_dtype)) || (dpost_w && !base_ok(dpost_w, post_w_dtype)) ||
      (dgate && !base_ok(dgate, gate_dtype)))
    return BS_ERR_ALIGN;
  int sms = 0;
  if (sm_count(&sms) != BS_OK) return BS_ERR_LAUNCH;
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15)) return BS_ERR_ALIGN;
  const bool vec = params_vec(P) && aligned(ds, D, elt(x_dtype)) && aligned(s, lds, elt(x_dtype)) &&
                   aligned(dx, D, elt(x_dtype)) && aligned(dh, D, elt(y_dtype)) &&
                   aligned(y, ldy, elt(y_dtype)) && aligned(dy, D, elt(y_dtype)) &&
                   (!gate_wide || aligned(dgate, D, elt(gate_dtype)));
  const int kind = gate_kind(gate, gate_rows, gate_wide);
  const bool contiguous = lds == D && (!(post || gate) || ldy == D) && T >= kShiftedRows * (int64_t)sms &&
                          aligned(ds, 8, 2) && aligned(s, 8, 2) && aligned(dx, 8, 2) &&
                          aligned(dh, 8, 2) && aligned(y, 8, 2) && aligned(dy, 8, 2) &&
                          (kind != 1 || (aligned(gate, 8, 2) && aligned(dgate, 8, 2)));
  P.div_rows = division(gate, gate_rows, gate_wide, T);
  auto plan_of = [&](int mode) {
    return plan_bwd(D, x_dtype, y_dtype, ds != nullptr, dh != nullptr, post != 0, kind, gate_dtype,
                    (w ? 1 : 0) + (post_w ? 1 : 0), mode, sms);
  };
  BwdPlan plan = plan_of(rows_mode(vec, contiguous, D));
  if (plan.mode == kRowsShifted &&
      (!plan.staged || !shares_groups(T / P.div_rows, D, plan.ctas, most_ctas(D, sms))))
    plan = plan_of(kRowsAny);
  const int share = plan.mode == kRowsShifted ? 8 : 1;
  const Chunks c = divide(T, P.div_rows, plan.ctas / share);
  P.chunks = c.chunks * share; P.chunk_rows = c.chunk_rows; P.chunks_per_group = c.per_group;
  P.groups_per_chunk = c.groups_per_chunk;
  const int64_t planes = 1 + (post || gate ? 1 : 0) + (gate ? 1 : 0);
  if (ws_bytes < (size_t)(planes * P.chunks * D + (gate && !gate_wide ? T : 0)) * sizeof(float))
    return BS_ERR_WORKSPACE;
  P.ds = ds; P.dh = dh; P.s = const_cast<void *>(s); P.lds = lds; P.y = y; P.ldy = ldy;
  P.dx = dx; P.dy = dy; P.dgate = dgate;
  P.r_post = post ? const_cast<float *>(r_post) : nullptr;
  P.r_pre = const_cast<float *>(r_pre);
  P.part = static_cast<float *>(ws);
  P.row_gate = P.part + planes * P.chunks * D;
  P.stages = plan.stages;
  P.status = status;
  int e;
  if (x_dtype == BS_F32 && y_dtype == BS_F32) e = norm_backward_f32(P, plan, st);
  else if (x_dtype == BS_F32) e = norm_backward_mix(P, plan, st);
  else e = norm_backward_bf16(P, plan, st);
  if (e != BS_OK) return e;
  SumJobs J = {};
  const int64_t plane = P.chunks * D;
  const bool gate_sums = dgate && gate_wide && gate_rows > 1 && !c.groups_per_chunk;
  J.job[0] = {P.part, dw, w_dtype, P.chunks, 1};
  J.job[1] = {P.part + plane, dpost_w, post_w_dtype, P.chunks, 1};
  J.job[2] = {P.part + 2 * plane, gate_sums ? dgate : nullptr, gate_dtype, c.per_group * share,
              gate_sums ? T / gate_rows : 0};
  if (dw || dpost_w || gate_sums) {
    const int64_t groups = gate_sums ? T / gate_rows : 1;
    const dim3 grid((unsigned)((D + 31) / 32), (unsigned)(groups < 65535 ? groups : 65535), 3);
    if (D % 4 == 0) norm_sum_kernel<4><<<grid, 256, 0, st>>>(J, (int)D);
    else norm_sum_kernel<1><<<grid, 256, 0, st>>>(J, (int)D);
    if ((e = launched()) != BS_OK) return e;
  }
  if (dgate && !gate_wide && gate_rows > 1) {
    const int64_t groups = T / gate_rows;
    norm_gate_sum_kernel<<<(unsigned)(groups < 65535 ? groups : 65535), 256, 0, st>>>(
        P.row_gate, gate_rows, dgate, gate_dtype, groups);
    e = launched();
  }
  return e;
}
