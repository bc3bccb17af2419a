"""The fused up-projection in training: its gradients are those of the layers it stands for (it used to cut them off)."""
import pytest
import torch
import torch.nn.functional as F

from pragnosia_b200 import ops
from pragnosia_b200.model import MLP

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _grad_enabled():
    with torch.enable_grad():
        yield


@pytest.mark.parametrize("act", ["gelu", None])
@pytest.mark.parametrize("M,K,N", [(130, 64, 72), (512, 128, 256)])
def test_linear_act_gradients(M, K, N, act):
    g = torch.Generator(device="cuda").manual_seed(M)
    x, W, b, up = (torch.randn(*s, device="cuda", generator=g).mul(c).to(BF).requires_grad_() for s, c in (((M, K), 1), ((N, K), K ** -0.5), ((N,), 1), ((M, N), 1)))
    y = ops.linear_act(x, W, b, act=act)
    with torch.no_grad():
        assert torch.equal(y, ops.linear_act(x, W, b, act=act))
    got = torch.autograd.grad(y, [x, W, b], up.detach())
    x64, W64, b64 = (t.detach().double().requires_grad_() for t in (x, W, b))
    pre = F.linear(x64, W64, b64)
    ref = torch.autograd.grad(F.gelu(pre) if act else pre, [x64, W64, b64], up.detach().double())
    # the pre-activation is rounded to bf16 (its slope's own slope is below 1.2), the gradient behind the activation and the result once each: 2^-8
    e = 2.0 ** -8 * ((1.2 * pre.abs() if act else 0.0) + 1.2) * up.detach().double().abs()
    offs = (e @ W64.abs(), e.t() @ x64.abs(), e.sum(0))
    for a, r, o in zip(got, ref, offs):
        assert a.dtype == BF and ((a.double() - r).abs() <= o + 2.0 ** -8 * r.abs()).all()


def test_mlp_layer_trains():
    torch.manual_seed(0)
    m = MLP(128, 4).cuda().to(BF)
    x = torch.randn(2, 100, 128, device="cuda").to(BF).requires_grad_()
    m(x).square().mean().backward()
    assert x.grad is not None and all(p.grad is not None and bool(p.grad.any()) for p in m.parameters())
    fused = [p.grad.clone() for p in m.parameters()]
    m.zero_grad()
    m.fused_up = False
    m(x).square().mean().backward()
    # both round the same values to bf16, the fused one a hidden value on the other side of a tie now and then
    assert all(float((a - p.grad).float().norm()) <= 2.0 ** -6 * float(p.grad.float().norm()) for a, p in zip(fused, m.parameters()))
