"""diff_attention's entry on the GPU: what it hands to autograd, tracing and forward mode, offsets
past 32 bits, many clips, calls on two streams and in graphs, its kernels' other forms."""
import pytest
import torch

from tests import diff_attn_ref as R
from tests.test_gpu_diff_attn import call, compare, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("leaf", [False, True])
def test_a_tangent_is_refused_and_never_dropped(leaf):
    import torch.autograd.forward_ad as fw
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, _ = operands(1, 1, 8, 2)
    want = diff_attention(*x, lam)
    with fw.dual_level():
        for i in range(4):
            t = [*x, lam]
            t[i] = fw.make_dual(t[i].clone().requires_grad_(leaf), torch.ones_like(t[i]))
            with pytest.raises(NotImplementedError, match="forward mode"):
                diff_attention(*t)
        assert torch.equal(diff_attention(*x, lam), want)


def test_one_reverse_mode_derivative():
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, do = operands(2, 1, 40, 2)
    q = x[0].requires_grad_(True)
    o = diff_attention(q, x[1], x[2], lam)
    with pytest.raises(RuntimeError, match="one gradient at a time"):
        torch.autograd.grad(o, q, torch.stack([do, do]), is_grads_batched=True, retain_graph=True)
    d, = torch.autograd.grad(o, q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.float().sum(), q)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: diff_attention(a, x[1], x[2], lam))(torch.stack([q] * 2))
    with pytest.raises(RuntimeError), torch.no_grad():
        torch.func.vmap(lambda a: diff_attention(a, x[1], x[2], lam))(torch.stack([q] * 2))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("leaf", [False, True])
def test_a_trace_records_the_call(leaf):
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, _ = operands(3, 1, 8, 2)
    m = torch.jit.trace(lambda a, b, c, w: diff_attention(a, b, c, w, causal=True),
                        [t.requires_grad_(leaf) for t in (*x, lam)], check_trace=False)
    y, lam2, _ = operands(4, 1, 8, 2)
    want = diff_attention(*y, lam2, causal=True)
    for _ in range(3):
        assert torch.equal(m(*y, lam2), want)


def test_many_clips_train():
    """65,600 heads of three rows: forward and backward, each clip as it is alone."""
    x, lam, do = operands(5, 8200, 3, 8, Lk=4)
    got = call(x, lam, do, causal=True)
    want = R.attention(*x, lam, causal=True, do=do, dev="cuda")
    for n in ("o", "dq", "dk", "dv", "dlam"):
        R.check(got[n], want[n], n)


@pytest.mark.parametrize("which", ["batch", "heads", "rows"])
def test_offsets_past_32_bits(which):
    """Operands as views of buffers of more than 2^32 bytes, strides past 2^31 elements between clips
    or heads, and 300 rows of 2^23 - 8 elements."""
    x, lam, do = operands(6, 2, 300, 2, dt=torch.float16)
    want = call(x, lam, do)
    far = 2 ** 31 + 128
    strides = {"batch": (far, 300, 64), "heads": (300 * 64, 64, far),
               "rows": (64, 2 ** 23 - 8, 128)}[which]
    if which == "batch":
        strides = (far, 128, 64)
    views = []
    for t in x:
        size = sum((n - 1) * s for n, s in zip((2, 300, 2), strides)) + 64
        buf = torch.empty(size, device="cuda", dtype=t.dtype)
        view = buf.as_strided(t.shape, (*strides, 1))
        view.copy_(t)
        views.append(view)
    if which == "rows":  # (clip 1 begins 64 elements behind clip 0, its rows between those)
        assert torch.equal(views[0], x[0])
    got = call(views, lam, do)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("L", [274, 700, 1500, 2500])
def test_a_gradient_does_not_depend_on_the_others(L):
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, do = operands(19, 1, L, 8)
    want = call(x, lam, do)
    for i, n in enumerate(("dq", "dk", "dv", "dlam")):
        t = [*x, lam]
        t[i] = t[i].clone().requires_grad_(True)
        got, = torch.autograd.grad(diff_attention(*t), t[i], do)
        assert torch.equal(got, want[n]), n


def test_saved_tensors_that_went_to_the_host_and_back():
    """Views come back contiguous: their strides are not the forward's."""
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, do = operands(20, 2, 130, 4)
    want = call(x, lam, do, k_lens=[130, 77])
    wide = torch.stack([t.flatten(2) for t in x], 2).reshape(2, 130, 3, 4, 64).requires_grad_(True)
    w = lam.clone().requires_grad_(True)
    with torch.autograd.graph.save_on_cpu():
        o = diff_attention(*wide.unbind(2), w, k_lens=[130, 77])
    dx, dlam = torch.autograd.grad(o, (wide, w), do)
    assert torch.equal(o, want["o"]) and torch.equal(dlam, want["dlam"])
    for i, n in enumerate(("dq", "dk", "dv")):
        assert torch.equal(dx[:, :, i], want[n]), n


def test_two_streams_at_once():
    """Calls of both forms interleaved on two streams, with workspaces of their own."""
    sets = [operands(7, 1, 1, 4, Lk=9000), operands(8, 2, 700, 4), operands(9, 1, 64, 4, Lk=5000)]
    want = [call(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for r in range(4):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[(r + i) % 2]):
                got.append((i, call(*s)))
    torch.cuda.synchronize()
    for i, g in got:
        for n in want[i]:
            assert torch.equal(g[n], want[i][n]), (i, n)


def test_two_graphs_and_eager_calls_between_their_replays():
    """Captured forward and backward, a graph each for few and for many queries, replayed in turn on
    refilled operands, an eager graph of other leaves alive."""
    from imfvideo_amd.imf_dit_video import diff_attention
    sets = [operands(10, 1, 2, 4, Lk=6000), operands(11, 2, 300, 4)]
    for s in sets:
        call(*s)
    other = sets[0][0][0].clone().requires_grad_(True)
    alive = diff_attention(other, *sets[0][0][1:], sets[0][1])
    graphs, kept = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(call(*s, causal=True))
        graphs.append(g)
    for r in range(4):
        for s in sets:
            for t in (*s[0], s[2]):
                t.copy_(torch.randn(t.shape, device="cuda"))
        for i in (0, 1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            want = call(*sets[i], causal=True)
            torch.cuda.synchronize()
            for n in want:
                assert torch.equal(kept[i][n], want[n]), (r, i, n)
    del alive


def test_the_least_and_most_gradients_of_an_expanded_output():
    """An output gradient that is one number for all, and operands that share memory."""
    from imfvideo_amd.imf_dit_video import diff_attention
    x, lam, _ = operands(12, 2, 70, 4)
    q = x[0]
    leaves = [t.clone().requires_grad_(True) for t in (q, lam)]
    o = diff_attention(leaves[0], leaves[0], leaves[0], leaves[1])
    dq, dlam = torch.autograd.grad(o.sum(), leaves)
    want = call([q, q, q], lam, torch.ones_like(q))
    assert torch.equal(dlam, want["dlam"])
    # the three gradients of the one leaf, added by autograd in the operands' type: two roundings
    total = sum(want[n].double() for n in ("dq", "dk", "dv"))
    size = sum(want[n].double().abs() for n in ("dq", "dk", "dv"))
    assert ((dq.double() - total).abs() <= 2 * 2.0 ** -8 * size).all()


@pytest.mark.parametrize("Hkv", [2, 8])
@pytest.mark.parametrize("Lq,Lk,causal", [(600, 40, False), (520, 520, True), (40, 9000, False),
                                          (130, 4100, True), (1500, 1500, False)])
def test_other_forms(Lq, Lk, causal, Hkv):
    """Sizes on both sides of the rules for tiles, splits and lost halves."""
    compare(*operands(13, 1, Lq, 8, Hkv, Lk), "forms", causal=causal)


@pytest.mark.parametrize("B,H,Lq,Lk,ql,kl", [
    (3, 2, 1, 405, [1, 0, 1], [405, 263, 121]), (2, 6, 37, 928, [37, 0], [928, 928]),
    (2, 6, 37, 928, [0, 37], [928, 0]), (3, 2, 5, 3000, [5, 0, 2], [64, 3000, 2999]),
    (3, 2, 1893, 1893, [1893, 0, 700], [1893, 0, 700])])
@pytest.mark.parametrize("causal", [False, True])
def test_ranges_of_keys_in_a_padded_batch(B, H, Lq, Lk, ql, kl, causal):
    """Rows of two clips in one wave of the join, ranges without a key, clips without any."""
    x, lam, do = operands(16, B, Lq, H, Lk=Lk)
    n = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got = compare(x, lam, do, "ranges", ql=n(ql), kl=n(kl), causal=causal)
    for b in range(B):
        dead = ql[b] if kl[b] else 0
        assert (got["o"][b, dead:] == 0).all() and (got["dq"][b, dead:] == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Lk,causal", [(1267, 2, True), (2500, 2, False), (64, 3, False),
                                          (2, 2, True), (3000, 100, True), (1500, 1, False)])
def test_few_keys_keep_the_gradients_accuracy(Lq, Lk, causal, dt):
    """Rows that see few keys: dA - delta nearly cancels, and what the rounding of the maps lost would
    show in it.  As far off as roundings of the exact result and of its last operand are, in norm:
    sqrt(2) of one rounding's u / sqrt(3), and half as much again for the others."""
    x, lam, do = operands(17, 2, Lq, 4, Lk=Lk, dt=dt)
    got = call(x, lam, do, causal=causal)
    want = R.attention(*x, lam, causal=causal, do=do, dev="cuda")
    u = torch.finfo(dt).eps / 2
    for n in ("o", "dq", "dk", "dv"):
        err = (got[n].double() - want[n][0]).norm().item()
        print("[ratio]", n, err / max(want[n][0].norm().item() * u, 1e-300), flush=True)
        assert err <= 1.5 * 2 ** 0.5 * u / 3 ** 0.5 * want[n][0].norm().item(), n


@pytest.mark.parametrize("B,H,L", [(2, 4, 900), (3, 8, 5000)])
def test_a_short_clip_keeps_its_accuracy_in_a_padded_batch(B, H, L):
    """The clip's gradients are as far off as roundings in norm are (as above), among long ones."""
    x, lam, do = operands(18, B, L, H, dt=torch.float16)
    lens = [L, 3, 100][:B]
    got = call(x, lam, do, q_lens=lens, k_lens=lens)
    want = R.attention(*x, lam, ql=lens, kl=lens, do=do, dev="cuda")
    for b in range(1, B):
        for n in ("o", "dq", "dk", "dv"):
            w = want[n][0][b]
            err = (got[n][b].double() - w).norm().item()
            print("[ratio]", b, n, err / w.norm().item() * 2 ** 11, flush=True)
            assert err <= 1.5 * 2 ** 0.5 * 2 ** -11 / 3 ** 0.5 * w.norm().item(), (b, n)


@pytest.mark.parametrize("ql,kl", [([-3, 400], [400, 2 ** 31 - 1]), ([401, 0], [0, 17])])
def test_lengths_are_clamped(ql, kl):
    x, lam, do = operands(14, 2, 400, 2)
    n = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    clamp = lambda v: n([min(max(i, 0), 400) for i in v])
    got = call(x, lam, do, q_lens=n(ql), k_lens=n(kl))
    want = call(x, lam, do, q_lens=clamp(ql), k_lens=clamp(kl))
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_what_stands_behind_a_sequence_is_not_read():
    """NaN in the rows behind q_len and k_len, of the output gradient too, reaches no result."""
    x, lam, do = operands(15, 2, 400, 4)
    kw = dict(q_lens=[130, 400], k_lens=[77, 331])
    want = call(x, lam, do, **kw)
    for t, lens in ((x[0], kw["q_lens"]), (x[1], kw["k_lens"]), (x[2], kw["k_lens"]),
                    (do, kw["q_lens"])):
        for b in range(2):
            t[b, lens[b]:] = float("nan")
    got = call(x, lam, do, **kw)
    for n in want:
        assert torch.equal(got[n], want[n]), n
        assert torch.isfinite(got[n]).all(), n
