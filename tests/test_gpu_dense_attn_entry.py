"""dense_attention's entry on the GPU: what it hands to autograd, tracing and forward mode, and
the sizes and lengths that it takes."""
import pytest
import torch

from tests import dense_attn_ref as R

pytestmark = pytest.mark.gpu


def operands(seed, B, L, H, Hkv, Lk, dt=torch.float16):
    """q, k, v and an output gradient, (B, L, H, 64) on the GPU."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    return rn(B, L, H, 64), rn(B, Lk, Hkv, 64), rn(B, Lk, Hkv, 64), rn(B, L, H, 64)


@pytest.mark.parametrize("leaf", [False, True])
def test_a_tangent_is_refused_and_never_dropped(leaf):
    import torch.autograd.forward_ad as fw
    from imfvideo_amd.imf_dit_video import dense_attention
    q, k, v, t = operands(1, 1, 8, 2, 2, 8)
    want = dense_attention(q, k, v)
    with fw.dual_level():
        for i in range(3):
            x = [q, k, v]
            x[i] = fw.make_dual(x[i].clone().requires_grad_(leaf), t)
            with pytest.raises(NotImplementedError, match="forward mode"):
                dense_attention(*x)
        # plain operands inside a dual level are answered
        assert torch.equal(dense_attention(q, k, v), want)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("leaf", [False, True])
def test_a_trace_records_the_call(leaf):
    from imfvideo_amd.imf_dit_video import dense_attention
    x = [t.requires_grad_(leaf) for t in operands(2, 1, 8, 2, 2, 8)[:3]]
    m = torch.jit.trace(lambda a, b, c: dense_attention(a, b, c, causal=True), x,
                        check_trace=False)
    y = operands(3, 1, 8, 2, 2, 8)[:3]
    want = dense_attention(*y, causal=True)
    for _ in range(3):
        assert torch.equal(m(*y), want)


def test_many_clips_train():
    """65,600 heads of three rows: forward and backward."""
    from imfvideo_amd.imf_dit_video import dense_attention
    q, k, v, do = operands(4, 8200, 3, 8, 8, 4, torch.bfloat16)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = dense_attention(*x, causal=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, x, do)), o=o.detach())
    heads = lambda t: t.detach().transpose(1, 2)
    want = R.attention(*map(heads, (q, k, v)), causal=True, do=heads(do), dev="cuda", lo=True)
    for n in ("o", "dq", "dk", "dv"):
        R.check(heads(got[n]), want[n], n)
