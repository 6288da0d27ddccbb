"""residual_norm on the host: the eager expression, what is refused, and the block around it."""
import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import TransformerBlock, residual_norm
from imfvideo_amd.mla_jvp_fast import pack_block
from tests import residual_norm_ref as R


def operands(dt=torch.float32):
    g = torch.Generator().manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g)
    return dict(x=rn(2, 5, 24), a=rn(2, 5, 24).to(dt), scale=rn(24), post_weight=1 + 0.1 * rn(24),
                gate=1 + 0.1 * rn(2, 24), pre_weight=1 + 0.1 * rn(24))


def test_the_eager_expression_and_its_gradients():
    o = operands()
    t = {k: v.clone().requires_grad_(True) for k, v in o.items()}
    y, n1, n2 = residual_norm(**t, consumers=2)
    dy, d1, d2 = (torch.randn_like(y) for _ in range(3))
    gr = torch.autograd.grad([y, n1, n2], list(t.values()), [dy, d1, d2])
    want = R.step(o["x"], o["a"], o["scale"], o["post_weight"], o["pre_weight"], o["gate"], 1e-6,
                  dy, [d1, d2])
    R.check(y.detach(), want["y"], "y")
    R.check(n1.detach(), want["n"], "n")
    for k, d in zip(("dx", "da", "dscale", "dpost", "dgate", "dpre"), gr):
        R.check(d, want[k], k)


def test_the_gradients_are_the_differences():
    o = {k: v.double() for k, v in operands().items()}
    for drop in ((), ("gate",), ("pre_weight",)):
        t = {k: v.clone().requires_grad_(True) for k, v in o.items() if k not in drop}
        assert torch.autograd.gradcheck(lambda *v: residual_norm(**dict(zip(t, v))),
                                        list(t.values()))


def test_without_a_following_norm_y_alone_comes_back():
    o = operands()
    o["pre_weight"] = None
    assert len(residual_norm(**o)) == 1
    assert len(residual_norm(**o, consumers=3)) == 1


def test_refusals():
    o = operands()
    for c in (0, 4):
        with pytest.raises(ValueError, match="consumers"):
            residual_norm(**o, consumers=c)
    for bad in (torch.ones(24), torch.ones(3, 24), torch.ones(2, 23)):
        with pytest.raises(ValueError, match="gate"):
            residual_norm(**{**o, "gate": bad})
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.residual_norm_fwd(o["x"], o["a"], o["scale"], o["post_weight"])
    m = TransformerBlock(64, 1, 32, 32, 32, 32, 64)
    with pytest.raises(ValueError, match="gates"):
        m(torch.randn(1, 2, 64), torch.ones(2, 16), torch.zeros(2, 16), gates=(None, None))
    with pytest.raises(ValueError, match="sandwich_norm"):
        pack_block(TransformerBlock(64, 1, 32, 32, 32, 32, 64, sandwich_norm=True))


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def test_operands_that_the_kernels_do_not_take_are_refused_by_name():
    gpu = lambda t: t.as_subclass(_Gpu)
    o = {k: gpu(v) for k, v in operands().items()}
    x, a, s, w, g = (o[k] for k in ("x", "a", "scale", "post_weight", "gate"))
    for args, what in (((gpu(x.half()), a, s, w), TypeError), ((x, gpu(a.double()), s, w), TypeError),
                       ((x, gpu(a[:, :4]), s, w), ValueError), ((x, a, gpu(s[:20]), w), ValueError),
                       ((x, a, s, gpu(w.half())), ValueError), ((x, a, s, w, None, w), ValueError),
                       ((gpu(x[:0]), gpu(a[:0]), s, w), ValueError)):
        with pytest.raises(what, match="residual_norm"):
            ops.residual_norm_fwd(*args)
    with pytest.raises(ValueError, match="three"):
        ops.residual_norm_bwd(x, [a] * 4, x, a, s, w, w)
    with pytest.raises(ValueError, match="without pre"):
        ops.residual_norm_bwd(x, [a], x, a, s, w)
    with pytest.raises(ValueError, match="gradient"):
        ops.residual_norm_bwd(None, [gpu(a.half())], x, a, s, w, w)


def test_sizes_past_the_kernels():
    lib = _lib.load()
    size = lib.sla2h_residual_norm_bwd_workspace_bytes
    assert size(1, 1, 8192) > 0 and size(2 ** 20, 1, 512) > 0
    for bad in ((1, 1, 8193), (0, 1, 8), (1, 0, 8), (1, 1, 0), (1, 2 ** 30, 8), (2 ** 30, 1, 8),
                (2 ** 15, 2 ** 15, 2048)):
        assert size(*bad) == 0, bad
        assert lib.sla2h_residual_norm_fwd(16, 16, 1, 16, 16, None, None, *bad, 1e-6, 16, None,
                                           None) == 1
    # an n without its weight, a weight without its n, no eps
    for pre, n, eps in ((None, 16, 1e-6), (16, None, 1e-6), (16, 16, 0.0)):
        assert lib.sla2h_residual_norm_fwd(16, 16, 1, 16, 16, pre, None, 1, 1, 8, eps, 16, n,
                                           None) == 1


def test_a_block_keeps_its_state_dict_without_sandwich_norm():
    names = set(TransformerBlock(64, 1, 32, 32, 32, 32, 64).state_dict())
    more = set(TransformerBlock(64, 1, 32, 32, 32, 32, 64, sandwich_norm=True).state_dict())
    assert more - names == {"attn_post_norm.weight", "mlp_post_norm.weight"}


def test_the_block_on_the_host():
    torch.manual_seed(2)
    m = TransformerBlock(64, 1, 32, 32, 32, 32, 64, sandwich_norm=True)
    torch.nn.init.normal_(m.attn_scale)
    torch.nn.init.normal_(m.mlp_scale)
    x, cos, sin = torch.randn(2, 6, 64), torch.ones(6, 16), torch.zeros(6, 16)
    g = torch.randn(2, 64), torch.randn(2, 64)
    y = x + m.attn_scale * g[0][:, None] * m.attn_post_norm(m.attn(m.norm1(x), cos, sin))
    y = y + m.mlp_scale * g[1][:, None] * m.mlp_post_norm(m.mlp(m.norm2(y)))
    assert torch.allclose(m(x, cos, sin, g), y, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("eps", [0.0, -1e-6, float("nan")])
def test_an_eps_that_is_not_above_zero(eps):
    with pytest.raises(ValueError, match="eps"):
        residual_norm(**operands(), eps=eps)
