"""GPU: the training-step operators inside captured CUDA graphs, forward and
backward, and the status of a process whose first call is captured."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import bitsparse_b200 as B
from bitsparse_b200.losses import token_logprobs
from bitsparse_b200.norms import residual_norm, rms_norm
from bitsparse_b200.optim import orthogonalize

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def join(x, y, w, pw, gate):
    out = residual_norm(x, y, w, post_norm=True, post_weight=pw, gate=gate, gate_act="sigmoid")
    return [*out, *torch.autograd.grad(out, (x, y, w, pw, gate), (x.detach(), y.detach()))]


def norm(x, w):
    h = rms_norm(x, w)
    return [h, *torch.autograd.grad(h, (x, w), x.detach())]


def loss(logits, targets):
    r = token_logprobs(logits, targets, top=5, temperature=0.8)
    return [*r, *torch.autograd.grad((r.logprobs.sum(), r.entropy.sum()), logits)]


@pytest.mark.parametrize("which", ["join", "norm", "loss", "orthogonalize", "orthogonalize_small"])
def test_replays_follow_their_inputs(which):
    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rnd(*shape):
            return torch.randn(*shape, generator=g, device="cuda").to(BF16)
        return {"join": lambda: (rnd(40, 30, 1024), rnd(40, 30, 1024), rnd(1024), rnd(1024),
                                 rnd(40, 1, 1024)),
                "norm": lambda: (rnd(50, 768), rnd(768)),
                "loss": lambda: (rnd(30, 9001), torch.randint(0, 9001, (30,), generator=g,
                                                              device="cuda")),
                "orthogonalize": lambda: (rnd(3, 300, 520),),
                "orthogonalize_small": lambda: (rnd(2, 60, 1500),)}[which]()

    f = {"join": join, "norm": norm, "loss": loss, "orthogonalize": lambda g: [orthogonalize(g)],
         "orthogonalize_small": lambda g: [orthogonalize(g)]}[which]
    held = [t.requires_grad_() if t.is_floating_point() else t for t in inputs(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(*held)
    for seed in (1, 2):
        with torch.no_grad():
            for t, new in zip(held, inputs(seed)):
                t.copy_(new)
        graph.replay()
        want = f(*[t.detach().clone().requires_grad_(t.requires_grad) for t in held])
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    B.check_status()


FIRST = """
import torch
import bitsparse_b200 as B

x = torch.randn(4, 100, device="cuda")
t = torch.zeros(4, dtype=torch.int64, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # the library's first call in this process
    lp = B.token_logprobs(x, t).logprobs
graph.replay()
B.check_status()
t.fill_(100)  # outside the vocabulary
graph.replay()
t.zero_()
graph.replay()  # a later replay takes nothing back
try:
    B.check_status()
except RuntimeError as e:
    assert "vocabulary" in str(e)
else:
    raise SystemExit("not reported")
B.check_status()
del graph
assert torch.isfinite(B.token_logprobs(x, t).logprobs).all()
B.check_status()
print("as it should be")
"""


def test_first_call_inside_a_capture():
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "as it should be" in r.stdout, r.stdout + r.stderr
