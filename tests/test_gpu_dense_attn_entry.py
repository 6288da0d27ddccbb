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


def fine_bounds(q, k, v, do, got, case):
    """Gradients of operands (1, H, L, 64) whose P and dS enter their products with the half
    that rounding them lost: an element is off by its own rounding u |x| and second-order terms,
    each at most u^2 P mag with mag = |dout| . |v_j| + |dout| . P |v| (dS's u^2 |dS|; through
    delta P's u^2 P |v| and the u^2 |o| of the output's second half), and T32 of the same sums for
    S, dP and delta in fp32."""
    dt, (_, H, Lq, _), (Hkv, Lk) = q.dtype, q.shape, k.shape[1:3]
    rep = H // Hkv
    want = R.attention(q, k, v, do=do, dev="cuda")
    u, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    K, V = (t.double().repeat_interleave(rep, 1) for t in (k, v))
    P = torch.softmax(q.double() @ K.transpose(-1, -2).contiguous() / 8, -1)
    g = do.double().abs()
    mag = g @ V.abs().transpose(-1, -2).contiguous() + (g * (P @ V.abs())).sum(-1, keepdim=True)
    E = (4 * u * u + 3 * R.T32) * P * mag + 2.0 ** -36 * mag.amax((-1, -2), keepdim=True)
    heads = lambda t: t.reshape(1, Hkv, rep, Lk, 64).sum(2)
    turn = lambda t: t.transpose(-1, -2).contiguous()
    more = dict(o=(2 * u * u + R.T32) * (P @ V.abs()), dq=E @ K.abs() / 8,
                dk=heads(turn(E) @ q.double().abs()) / 8,
                dv=heads(turn((2 * u * u + R.T32) * P + 2.0 ** -36) @ g))
    for n, m in more.items():
        val = want[n][0]
        print("[ratio]", n, round(R.check(got[n], (val, u * val.abs() + m + tiny), (case, n)), 3),
              flush=True)


# B, H, Hkv, Lq, Lk of the padded batch; rows and keys of its first clip, which alone takes each
# kernel's form for few of them: 128- and 256-row blocks of the forward, the backward's dq and dk/dv
PADDED = [(2, 128, 128, 130, 700, 130, 200), (8, 64, 32, 300, 700, 200, 97),
          (2, 4, 2, 700, 4200, 90, 150)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", PADDED)
def test_a_short_clip_keeps_its_accuracy_in_a_padded_batch(case, dt):
    """The halves that rounding P and dS loses are kept by a sequence's own length, however
    far its batch is padded."""
    from imfvideo_amd import ops
    B, H, Hkv, Lq, Lk, nq, nk = case
    print("[case]", case, dt, flush=True)
    q, k, v, do = (t.transpose(1, 2) for t in operands(5, B, Lq, H, Hkv, Lk, dt))
    ql = torch.tensor([nq] + [Lq] * (B - 1), device="cuda")
    kl = torch.tensor([nk] + [Lk] * (B - 1), device="cuda")
    o, lse, lo = ops.dense_attn_fwd(q, k, v, q_lens=ql, k_lens=kl, with_lo=True)
    grads = ops.dense_attn_bwd(do, q, k, v, o, lse, q_lens=ql, k_lens=kl, o_lo=lo)
    cut = lambda t, n: t[:1, :, :n]
    got = dict(o=cut(o, nq), dq=cut(grads[0], nq), dk=cut(grads[1], nk), dv=cut(grads[2], nk))
    fine_bounds(cut(q, nq), cut(k, nk), cut(v, nk), cut(do, nq), got, (case, dt))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 2, 2, 1, 29952), (2, 8, 2, 3, 5000), (1, 4, 4, 32, 1100),
                                   (1, 8, 8, 1000, 1000)])
def test_few_queries_keep_what_rounding_loses(shape, dt):
    """The output of calls of at most 256 blocks of 32 rows, over any number of keys: its own
    rounding, second-order terms and fp32 arithmetic."""
    from imfvideo_amd import ops
    B, H, Hkv, Lq, Lk = shape
    q, k, v, _ = (t.transpose(1, 2) for t in operands(6, B, Lq, H, Hkv, Lk, dt))
    o, _ = ops.dense_attn_fwd(q, k, v)
    val, _ = R.attention(q, k, v, dev="cuda")["o"]
    u, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    for b in range(B):
        x = [t[b:b + 1] for t in (q, k, v.abs())]
        pv, _ = R.attention(*x, dev="cuda")["o"]  # P |v|
        val_b = val[b:b + 1]
        print("[ratio]", round(R.check(o[b:b + 1], (val_b, u * val_b.abs() + (2 * u * u + R.T32) * pv
                                                    + tiny), (shape, dt)), 3), flush=True)
