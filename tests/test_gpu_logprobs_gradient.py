"""GPU: the gradient of token_logprobs where its terms nearly cancel (rows with
one token that has nearly all of the probability) and where they are largest
(the smallest temperatures, with masked tokens); the logits of a shifted
model."""
import pytest
import torch

from bitsparse_b200.losses import token_logprobs

from tests.op_util import close

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def confident(rows, V, dtype):
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(rows + V))
    sure = (torch.arange(rows) * 7919 + torch.arange(rows) // 3) % V
    sure[-1], sure[0] = V - 1, 0
    x[torch.arange(rows), sure] = 14.0 + torch.arange(rows) % 7
    return x.to(dtype).cuda(), sure.cuda()


def view(x, offset):
    """The same logits on another alignment."""
    n, v = x.shape
    wide = torch.zeros(n, v + 3 + offset, dtype=x.dtype, device="cuda")
    wide[:, offset:offset + v] = x
    return wide[:, offset:offset + v]


@pytest.mark.parametrize("temperature", [1.0, 0.75])
@pytest.mark.parametrize("offset", [None, 1])
@pytest.mark.parametrize("rows, V", [(1, 50304), (16, 20011), (200, 5003), (300, 130), (90, 3)])
def test_confident_rows(rows, V, offset, temperature):
    """d logprob / d logit of the sure token is (1 - p) / T, here 0.07 down to
    1e-9.  Terms that count have |z| below 30: five fp32 roundings of z make 30 *
    5 * 2^-24 = 9e-6, the exponentials and the sums less than 3e-6 more.  So the
    sure token's slope and the sum of the others' are right to 1.2e-5 each, and a
    row's sum is within 2.4e-5 of the slope of zero."""
    x, t = confident(rows, V, F32)
    x = x if offset is None else view(x, offset)
    x = x.detach().requires_grad_()
    gl = 0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()
    r = token_logprobs(x, t, temperature=temperature)
    d, = torch.autograd.grad(r.logprobs, x, gl)
    z = x.detach().double() / temperature
    z = z - z.amax(-1, keepdim=True)
    rest = z.exp().scatter(-1, t.unsqueeze(-1), 0).sum(-1)
    want = gl.double() / temperature * rest / (1 + rest)
    at = d.gather(-1, t.unsqueeze(-1)).squeeze(-1).double()
    assert ((at - want).abs() <= 1.2e-5 * want).all()
    assert (d.double().sum(-1).abs() <= 2.4e-5 * want).all()


@pytest.mark.parametrize("rows, V", [(4, 50304), (100, 5003), (60, 40)])
def test_confident_rows_with_entropy(rows, V):
    """The entropy's slope at the sure token, -p (lp + H), joins it: two terms
    with 1.2e-5 of the first and what H, 2e-5, and lp, 1e-5, bring to the second."""
    x, t = confident(rows, V, F32)
    x = x.requires_grad_()
    gl, gh = torch.ones(rows, device="cuda"), torch.full((rows,), 0.3, device="cuda")
    r = token_logprobs(x, t)
    d, = torch.autograd.grad((r.logprobs, r.entropy), x, (gl, gh))
    z = x.detach().double()
    z = z - z.amax(-1, keepdim=True)
    rest = z.exp().scatter(-1, t.unsqueeze(-1), 0).sum(-1)
    lse, p = torch.log1p(rest), 1 / (1 + rest)
    entropy = lse - (z.exp() * z).sum(-1) * p
    one, two = rest * p, -0.3 * p * (entropy - lse)
    at = d.gather(-1, t.unsqueeze(-1)).squeeze(-1).double()
    bound = 1.2e-5 * one + 0.3 * p * (2e-5 * entropy + 1e-5 * lse + 1e-6 * (entropy - lse))
    assert ((at - (one + two)).abs() <= bound).all()


def test_confident_bf16_logits():
    x, t = confident(50, 4099, BF16)
    x = x.requires_grad_()
    d, = torch.autograd.grad(token_logprobs(x, t).logprobs.sum(), x)
    z = x.detach().double()
    rest = (z - z.amax(-1, keepdim=True)).exp().scatter(-1, t.unsqueeze(-1), 0).sum(-1)
    at = d.gather(-1, t.unsqueeze(-1)).squeeze(-1).double()
    want = rest / (1 + rest)
    assert ((at - want).abs() <= (2.0 ** -8 + 2e-5) * want).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature, gh", [(1e-10, 1.0), (1e-10, 1000.0), (1e-8, 1e5)])
@pytest.mark.parametrize("V, offset", [(1000, None), (1003, None), (1003, 1), (20000, None)])
def test_masked_tokens_at_small_temperatures(V, offset, temperature, gh, dtype):
    """Logits as small as the temperature, so that the distribution is an
    ordinary one; masked tokens get exactly nothing, all others their slope."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(7, V, generator=g, device="cuda") * 3 * temperature).to(dtype)
    gone = torch.rand(V, generator=g, device="cuda") < 0.4
    for fill in (-float("inf"), torch.finfo(dtype).min):
        y = x.masked_fill(gone, fill)
        y[3] = fill
        y[3, 5] = 0.0
        y = y if offset is None else view(y, offset)
        t = torch.full((7,), int((~gone).nonzero()[0]), device="cuda")
        y = y.detach().requires_grad_()
        r = token_logprobs(y, t, temperature=temperature)
        w = torch.full((7,), gh, device="cuda")
        d, = torch.autograd.grad((r.logprobs, r.entropy), y, (w * 0.5, w))
        z = y.detach().double() / temperature
        lp = torch.log_softmax(z, -1)
        p = lp.exp()
        entropy = torch.special.entr(p)
        want = gh * (entropy - p * entropy.sum(-1, keepdim=True)) - 0.5 * gh * p
        want.scatter_add_(-1, t.unsqueeze(-1), 0.5 * w.double().unsqueeze(-1))
        close(d, want / temperature, "d_logits")
        keep = torch.arange(7, device="cuda") != 3
        assert (d[keep][:, gone] == 0).all()


def test_logits_of_a_shifted_model():
    logits = torch.randn(3, 9, 517, device="cuda", requires_grad=True)
    tokens = torch.randint(0, 517, (3, 9), device="cuda")
    lp = token_logprobs(logits[:, :-1], tokens[:, 1:]).logprobs
    got, = torch.autograd.grad(lp.sum(), logits)
    ref = logits.detach().double().requires_grad_()
    want = torch.log_softmax(ref[:, :-1], -1).gather(-1, tokens[:, 1:, None]).squeeze(-1)
    exact, = torch.autograd.grad(want.sum(), ref)
    assert (lp.double() - want).abs().max() <= 1e-5
    assert (got.double() - exact).abs().max() <= 1e-6
    assert got[:, -1].abs().sum() == 0
