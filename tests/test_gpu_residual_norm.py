"""The residual step with a norm on both of its sides (residual_norm, TransformerBlock with
sandwich_norm) on the GPU against float64."""
import pytest
import torch

from tests import residual_norm_ref as R

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def operands(seed, B, L, D, dt, gate=True, pre=True, consumers=2):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = dict(x=2 * rn(B, L, D), a=(0.7 * rn(B, L, D)).to(dt), scale=0.3 * rn(D),
             post=1 + 0.1 * rn(D), gate=1 + 0.2 * rn(B, D) if gate else None,
             pre=1 + 0.1 * rn(D) if pre else None, dy=0.1 * rn(B, L, D))
    dns = [(0.1 * rn(B, L, D)).to(dt).cuda() for _ in range(consumers if pre else 0)]
    return {k: None if v is None else v.cuda() for k, v in x.items()}, dns


def call(o, dns, eps=1e-6, order=("x", "a", "scale", "post", "gate", "pre")):
    """(outputs, gradients by name) of residual_norm."""
    from imfvideo_amd.imf_dit_video import residual_norm
    t = {k: o[k].detach().requires_grad_(True) for k in order if o[k] is not None}
    y, *n = residual_norm(t["x"], t["a"], t["scale"], t["post"], t.get("gate"), t.get("pre"), eps,
                          max(1, len(dns)))
    got = dict(y=y.detach())
    if n:
        got["n"] = n[0].detach()
        assert all(torch.equal(n[0], m) for m in n)
    outs, grads = [y, *n], [o["dy"], *dns]
    gr = torch.autograd.grad(outs, list(t.values()), grads)
    got.update({"d" + k: d for k, d in zip(t, gr)})
    return got


def compare(got, o, dns, eps=1e-6, what=None):
    want = R.step(o["x"], o["a"], o["scale"], o["post"], o["pre"], o["gate"], eps, o["dy"], dns)
    assert set(got) == set(want)
    for k in want:
        like = {"y": "x", "n": "a"}.get(k, k[1:])
        assert got[k].dtype == o[like].dtype, k
        print("[ratio]", what, k, round(R.check(got[k], want[k], (what, k)), 3), flush=True)


# widths of every form: 16, 32 and 64 lanes, a workgroup; each full, one short of it, odd
@pytest.mark.parametrize("D", [1, 7, 8, 64, 127, 128, 136, 255, 512, 513, 520, 1000, 1024, 1025,
                               1365, 2048, 2056, 4095, 8192, 8191])
@pytest.mark.parametrize("dt", HALF + [torch.float32])
def test_widths(D, dt):
    o, dns = operands(D, 2, 5, D, dt)
    compare(call(o, dns), o, dns, what=(D, dt))


@pytest.mark.parametrize("B,L,D", [(1, 1, 512), (3, 1, 512), (1, 7, 96), (2, 1042, 512),
                                   (5, 333, 160), (1, 9001, 256), (2, 4500, 512)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("consumers", [0, 1, 3])
def test_rows_and_clips(B, L, D, gate, consumers):
    o, dns = operands(L, B, L, D, torch.bfloat16, gate, consumers > 0, consumers)
    compare(call(o, dns), o, dns, what=(B, L, D, gate, consumers))


def test_large_rows_and_offsets():
    """Values far from one, a row of zeros, and the largest eps that keeps it finite."""
    o, dns = operands(3, 2, 40, 512, torch.float16)
    o["x"] *= 1e4
    o["a"][0, 3] = 0
    o["a"][1, 5] *= 100
    o["x"][1, 7] = 0
    compare(call(o, dns, 1e-3), o, dns, 1e-3)


def test_some_gradients_only():
    """Only n, only y, only one of three consumers has a gradient."""
    from imfvideo_amd.imf_dit_video import residual_norm
    o, dns = operands(5, 2, 33, 512, torch.bfloat16, True, True, 3)
    names = ("x", "a", "scale", "post", "gate", "pre")
    for use_y, used in ((False, [0, 1, 2]), (True, []), (False, [1]), (True, [2])):
        t = {k: o[k].detach().requires_grad_(True) for k in names}
        y, *n = residual_norm(t["x"], t["a"], t["scale"], t["post"], t["gate"], t["pre"],
                              consumers=3)
        outs = [y] * use_y + [n[i] for i in used]
        gr = torch.autograd.grad(outs, list(t.values()), [o["dy"]] * use_y + [dns[i] for i in used])
        want = R.step(o["x"], o["a"], o["scale"], o["post"], o["pre"], o["gate"], 1e-6,
                      o["dy"] if use_y else None, [dns[i] for i in used])
        for k, d in zip(names, gr):
            if "d" + k in want:
                R.check(d, want["d" + k], (use_y, used, k))
            else:
                assert torch.equal(d, torch.zeros_like(d))


def test_strided_and_unaligned_operands():
    """Views: rows of a wider tensor, data off 16 bytes, expanded vectors."""
    from imfvideo_amd.imf_dit_video import residual_norm
    o, dns = operands(6, 2, 50, 96, torch.bfloat16, True, True, 1)
    want = R.step(o["x"], o["a"], o["scale"], o["post"], o["pre"], o["gate"])
    wide = lambda t: torch.cat([torch.zeros_like(t[..., :3]), t, t], -1)[..., 3:3 + t.shape[-1]]
    y, n = residual_norm(wide(o["x"]), wide(o["a"]), wide(o["scale"]), wide(o["post"]),
                         wide(o["gate"]), wide(o["pre"]))
    R.check(y, want["y"], "y")
    R.check(n, want["n"], "n")
    flat = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].reshape(t.shape)
    y, n = residual_norm(flat(o["x"]), flat(o["a"]), flat(o["scale"]), o["post"], o["gate"],
                         o["pre"])
    R.check(y, want["y"], "y")
    R.check(n, want["n"], "n")
    # gradients that are expanded (a sum's)
    t = {k: o[k].detach().requires_grad_(True) for k in ("x", "a", "post", "pre")}
    y, n = residual_norm(t["x"], t["a"], o["scale"], t["post"], o["gate"], t["pre"])
    gr = torch.autograd.grad(y.sum() + n.sum(), list(t.values()))
    want = R.step(o["x"], o["a"], o["scale"], o["post"], o["pre"], o["gate"], 1e-6,
                  torch.ones_like(o["x"]), [torch.ones_like(o["a"])])
    for k, d in zip(t, gr):
        R.check(d, want["d" + k], k)


def test_calls_agree_bit_for_bit_on_streams_and_in_a_graph():
    o, dns = operands(7, 2, 700, 512, torch.bfloat16)
    want = call(o, dns)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(o, dns)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            captured = call(o, dns)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    for _ in range(3):
        for v in captured.values():
            v.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(captured[k], want[k]) for k in want)
        again = call(o, dns)
        assert all(torch.equal(again[k], want[k]) for k in want)


def test_rows_that_are_not_finite_stay_their_own():
    """A NaN row's outputs and gradients are NaN, every other row keeps its values."""
    from imfvideo_amd.imf_dit_video import residual_norm
    o, _ = operands(8, 1, 20, 512, torch.bfloat16, False, True, 1)
    want = residual_norm(o["x"], o["a"], o["scale"], o["post"], None, o["pre"])
    o["a"][0, 4, 9] = float("nan")
    o["x"][0, 11, 3] = float("inf")
    got = residual_norm(o["x"], o["a"], o["scale"], o["post"], None, o["pre"])
    keep = [i for i in range(20) if i not in (4, 11)]
    for a, b in zip(got, want):
        assert torch.equal(a[0, keep], b[0, keep])
        assert a[0, 4].isnan().all()


@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("gates", [False, True])
def test_block_with_sandwich_norm(act8, gates):
    """The block's step is the modules' one by one: a float32 block of plain expressions."""
    from imfvideo_amd.imf_dit_video import TransformerBlock, dense_attention, precompute_axial_rope_3d
    torch.manual_seed(1)
    H, D, L = 4, 256, 4 * 4 * 8 + 3
    m = TransformerBlock(D, H, 128, 64, 32, 32, 64, attn_impl=dense_attention, sandwich_norm=True,
                         act8=act8).cuda()
    with torch.no_grad():
        for p in (m.attn_scale, m.mlp_scale):
            p.copy_(0.5 * torch.randn_like(p))
        for p in (m.attn_post_norm.weight, m.mlp_post_norm.weight, m.norm2.weight):
            p.add_(0.1 * torch.randn_like(p))
    cos, sin = (t.cuda() for t in precompute_axial_rope_3d(32, (4, 4, 8), 3))
    x = torch.randn(2, L, D, device="cuda")
    gs = tuple(1 + 0.2 * torch.randn(2, D, device="cuda") for _ in range(2)) if gates else None
    do = torch.randn_like(x)

    def plain(x):
        rms = lambda t, w: (t.float() * torch.rsqrt(t.float().square().mean(-1, keepdim=True) + 1e-6)
                            * w)
        one = (1.0, 1.0) if gs is None else tuple(g[:, None] for g in gs)
        a = m.attn(rms(x, m.norm1.weight).bfloat16(), cos, sin)
        x = x + m.attn_scale * one[0] * rms(a, m.attn_post_norm.weight)
        h = m.mlp(rms(x, m.norm2.weight).bfloat16())
        return x + m.mlp_scale * one[1] * rms(h, m.mlp_post_norm.weight)

    leaves = [x.requires_grad_(True)] + list(m.parameters())
    outs = []
    for f in (lambda t: m(t, cos, sin, gs), plain):
        with torch.autocast("cuda", torch.bfloat16):
            y = f(x)
        assert y.dtype == torch.float32
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, do)])
    # bf16 tensors between the layers: a chain of about ten of them, each rounded on both sides
    # within 2^-8, so that two evaluations are apart by at most that many steps in 2-norm
    for i, (a, b) in enumerate(zip(*outs)):
        rel = (a - b).norm() / b.norm().clamp_min(1e-12)
        assert rel < 10 * 2.0 ** -8, (i, rel.item())
