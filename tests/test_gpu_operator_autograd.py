"""GPU: residual_norm, rms_norm and token_logprobs under forward mode, which is
refused, not answered without its tangents."""
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
