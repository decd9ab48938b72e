"""GPU: residual_norm where a row's last threads have no columns, where gate
groups divide the rows in every way, and for wide rows with more rows than
SMs."""
import pytest
import torch

from bitsparse_b200 import _lib
from bitsparse_b200.norms import residual_norm

from tests.op_util import close
from tests.test_gpu_residual_norm import BF16, EPS, F32, check, formula, inputs

pytestmark = pytest.mark.gpu


def check_where_they_are(v, grads):
    """As check() with a norm on the branch, on the tensors themselves: copies
    would be aligned."""
    own = {k: t.detach().requires_grad_() for k, t in v.items()}
    out = residual_norm(own["x"], own["y"], own["weight"], post_norm=True,
                        post_weight=own["post_weight"], gate=own["gate"], eps=EPS)
    ref = {k: t.detach().double().requires_grad_() for k, t in v.items()}
    exact = formula(ref, True, "none", 1.0, 1.0)
    got = torch.autograd.grad(out, list(own.values()), grads)
    want = torch.autograd.grad(exact, list(ref.values()), [g.double() for g in grads])
    for k, a, b in zip(("stream", "normed", *own), (*out, *got), (*exact, *want)):
        close(a, b, k, scale=4.0 if k in own else 1.0)


@pytest.mark.parametrize("p_t", [BF16, F32])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("D", [72, 520, 1032, 1032 + 256, 2056, 2568, 4104, 5128, 7176])
def test_nan_rows_beside_idle_threads(D, gate, p_t):
    """Widths that leave threads without columns: every third row is NaN, and
    nothing of it, nor of anything that such a thread never read, reaches the
    other rows' outputs and gradients."""
    T = 1480
    v, grads = inputs((T,), D, BF16, BF16, p_t, True, gate, seed=D)
    bad = torch.arange(T, device="cuda") % 3 == 1
    v["y"][bad] = float("nan")
    own = {k: t.clone().requires_grad_() for k, t in v.items()}
    out = residual_norm(own["x"], own["y"], own["weight"], post_norm=True,
                        post_weight=own["post_weight"], gate=own.get("gate"))
    names = [k for k in ("x", "y") + (("gate",) if gate == "full" else ())]
    got = torch.autograd.grad(out, [own[k] for k in names], grads)
    for t in (*out, *got):
        assert torch.isnan(t[bad]).any(-1).all() and torch.isfinite(t[~bad]).all()
    fine = {k: t[~bad] if t.shape[:1] == (T,) and t.dim() == 2 else t for k, t in v.items()}
    check(fine, tuple(g[~bad] for g in grads), post=True)


def workspace(T, D, post, gate_rows, wide=1):
    return _lib.load().bs_residual_norm_workspace_bytes(T, D, post, 1, gate_rows, wide)


@pytest.mark.parametrize("groups, rows, D", [(2300, 2, 512), (140, 5, 8192), (300, 15, 512),
                                             (1183, 4, 512), (1184, 4, 512), (71, 9, 8192),
                                             (72, 9, 8192), (600, 2, 1024), (2000, 3, 24),
                                             (2300, 2, 511), (1183, 4, 511), (1184, 4, 511),
                                             (71, 9, 8191), (72, 9, 8191)])
def test_workspace_of_gate_groups(groups, rows, D):
    """The partial sums of the backward: three planes with a row for each CTA --
    sixteen an SM at most -- or for each group, or (only for widths off a multiple
    of eight, whose groups are shared by eight CTAs while they are fewer than half
    of those that fill the GPU) eight for each; and the backward has room in it."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    threads = (D + 511) // 512 * 32
    ctas = sms * (1 if D > 4096 else min(16, max(1, 512 // threads)))
    rows_of_sums = max(ctas, groups)
    if D % 8 and groups < 4 * (ctas // 8):
        rows_of_sums = max(rows_of_sums, 8 * groups)
    assert workspace(groups * rows, D, 1, rows) <= 3 * rows_of_sums * D * 4
    v, grads = inputs((groups, rows), D, BF16, BF16, BF16, True, "batch", seed=D)
    check(v, grads, post=True)
    # parameters off their alignment, everything off it: other forms, the same workspace
    off = {k: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for k, t in v.items()}
    check_where_they_are({**v, "weight": off["weight"]}, grads)
    check_where_they_are(off, grads)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gate, post", [("none", False), ("none", True), ("channel", True),
                                        ("batch", True), ("full", True), ("token", False)])
@pytest.mark.parametrize("D", [8200, 12288, 16385])
def test_wide_rows_in_number(D, gate, post, dtype):
    check(*inputs((5, 61), D, dtype, dtype, dtype, post, gate, seed=D), post=post, act="sigmoid",
          branch=0.5)
