"""Muon's step of 16-bit weights on the host: decay and update share one rounding."""
import pytest
import torch

from imfvideo_amd.muon import Muon, newton_schulz

HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("lr,decay", [(0.02, 0.5), (2e-3, 0.1), (0.1, 3.0), (0.02, 0.0)])
def test_a_step_rounds_once(dt, lr, decay):
    """(1 - lr wd) w - lr rms sqrt(max(R, C)) NS(u) in float64, within half a step of the type: u times the
    value, and what the formula's two products and its difference may be off in fp32, 2^-24 of |w| and of
    |d| each, and half as much again for the factors' own roundings."""
    torch.manual_seed(1)
    p = torch.nn.Parameter((0.2 * torch.randn(48, 96)).to(dt))
    w, g = p.detach().double(), torch.randn(48, 96).to(dt)
    p.grad = g
    Muon([p], lr=lr, weight_decay=decay, nesterov=False, rms=0.2).step()
    d = lr * 0.2 * 96 ** 0.5 * newton_schulz(g.float()).double()
    want = (1 - lr * decay) * w - d
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    tol = torch.finfo(dt).eps / 2 * want.abs() + 3 * 2.0 ** -24 * (w.abs() + d.abs()) + tiny
    assert ((p.detach().double() - want).abs() <= tol).all()


def test_decay_of_16_bit_weights_over_many_steps():
    """The share of the first weights that 150 steps leave, bf16 beside fp32 of the same gradients.  A factor
    of 0.999 alone rounds back to every bf16 weight, together with updates of 2e-3 (two of the weights'
    steps of 2^-10) it does not.  The roundings, each 2^-9 of a weight at most, are as good as independent:
    their sum's share of the first weights is 150^0.5 * 2^-9 / 128 = 2e-4, and 1 - 0.999^150 = 0.14 is what
    the decay takes away.  Allowed is 5e-3: 25 times the one, a 28th of the other."""
    torch.manual_seed(2)
    first = (0.2 * torch.randn(128, 128)).bfloat16()
    kept = []
    for dt in (torch.float32, torch.bfloat16):
        p = torch.nn.Parameter(first.clone().to(dt))
        opt = Muon([p], lr=0.01, weight_decay=0.1)
        rng = torch.Generator().manual_seed(3)
        for _ in range(150):
            p.grad = torch.randn(128, 128, generator=rng).bfloat16().to(dt)
            opt.step()
        f = first.double()
        kept.append(((p.detach().double() * f).sum() / f.square().sum()).item())
    assert abs(kept[0] - kept[1]) <= 5e-3, kept
