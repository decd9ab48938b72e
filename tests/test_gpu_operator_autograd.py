"""GPU: residual_norm, rms_norm and token_logprobs inside autograd's other
tools: forward mode is refused, not answered without its tangents; what the
backward needs goes through saved-tensor hooks."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from bitsparse_b200.losses import token_logprobs
from bitsparse_b200.norms import residual_norm, rms_norm

pytestmark = pytest.mark.gpu


def each(out):
    return out if isinstance(out, tuple) else (out,)


def calls():
    x, y = torch.randn(2, 4, 64, device="cuda").unbind()
    w, t = torch.ones(64, device="cuda"), torch.arange(4, device="cuda")
    gate = torch.rand(64, device="cuda")
    return {"x": (lambda v: residual_norm(v, y, w), x), "y": (lambda v: residual_norm(x, v, w), y),
            "weight": (lambda v: residual_norm(x, y, v), w),
            "post": (lambda v: residual_norm(x, y, w, post_norm=True, post_weight=v), w),
            "gate": (lambda v: residual_norm(x, y, w, gate=v), gate),
            "rms": (lambda v: rms_norm(v, w), x), "rms_weight": (lambda v: rms_norm(x, v), w),
            "logits": (lambda v: token_logprobs(v, t, top=2), x)}


@pytest.mark.parametrize("name", ["x", "y", "weight", "post", "gate", "rms", "rms_weight",
                                  "logits"])
def test_forward_mode_is_refused(name):
    f, v = calls()[name]
    with fwd.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):  # NotImplementedError too
                f(fwd.make_dual(v, torch.ones_like(v)))
        plain = f(v)  # no tangent: answered as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda u: f(u)[0], (v,), (torch.ones_like(v),))
    again = f(v)
    for a, b in zip(each(plain), each(again)):
        assert torch.equal(a, b)


def test_saved_tensors_leave_the_gpu():
    """Under hooks that move what is saved to the host, nothing of the forward
    but its outputs stays on the device."""
    rows = 100_000
    x = torch.randn(rows, 8, device="cuda", requires_grad=True)
    y = torch.randn(rows, 8, device="cuda", requires_grad=True)
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    cases = (lambda: residual_norm(x, y, post_norm=True), lambda: rms_norm(x),
             lambda: token_logprobs(x, t)[:2])
    for f in cases:
        f()  # (what the library keeps by itself)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autograd.graph.save_on_cpu():
            out = f()
        out = each(out)
        own = sum(o.numel() * o.element_size() + 511 for o in out)
        held = torch.cuda.memory_allocated() - before
        assert held <= own  # (rows * 4 bytes of statistics would be 400 KB more)
        got = torch.autograd.grad([o.sum() for o in out], x)[0]
        want = torch.autograd.grad([o.sum() for o in each(f())], x)[0]
        assert torch.equal(got, want)
