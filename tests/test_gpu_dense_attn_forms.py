"""The forms of the dense attention kernels that only large calls take, against float64
(tests/dense_attn_ref.py derives the per-element bounds): blocks of 256 and 128 query rows over
many key tiles, with and without causal order and lengths, and the backward of sequences past
the lengths whose P and dS are corrected."""
import pytest
import torch

from tests import dense_attn_ref as R
from tests.test_gpu_dense_attn import check_all, inputs, run

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def lens(B, Lq, Lk, seed):
    """A full sequence, then shorter ones (the last one's keys a quarter)."""
    g = torch.Generator().manual_seed(seed)
    ql = torch.randint(1, Lq + 1, (B,), generator=g)
    kl = torch.randint(1, Lk + 1, (B,), generator=g)
    ql[0], kl[0] = Lq, Lk
    kl[B - 1] = Lk // 4
    return ql.cuda(), kl.cuda()


# 256 rows a workgroup from 256 of them on (768 with a mask), 128 rows below
FORMS = [((1, 64, 64, 1000, 700), "none"), ((1, 64, 32, 1000, 300), "none"),
         ((1, 64, 64, 500, 700), "none")] + [
    ((3, 64, 16, 1000, Lk), m) for Lk in (700, 300) for m in ("causal", "ragged", "both")] + [
    ((1, 64, 64, 500, 700), "both"), ((2, 32, 32, 600, 1400), "causal")]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape, mask", FORMS)
def test_large_blocks_of_rows(shape, mask, dt):
    print("[case]", shape, mask, dt, flush=True)
    x = [t.cuda() for t in inputs(sum(shape), *shape, dt)]
    kw = dict(causal=mask in ("causal", "both"))
    ql = kl = None
    if mask in ("ragged", "both"):
        ql, kl = lens(shape[0], shape[3], shape[4], 1)
    got = run(*x, q_lens=ql, k_lens=kl, **kw)
    B = shape[0]
    for b in range(B):  # the reference of one sequence at a time: its matrices are large
        one = lambda t: None if t is None else t[b:b + 1]
        want = R.attention(*map(one, x[:3]), kw["causal"], one(ql), one(kl), do=one(x[3]),
                           dev="cuda", lo=True)
        check_all({n: one(t) for n, t in got.items()}, want, (shape, mask, dt, b))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("mask", ["none", "causal", "ragged", "both"])
@pytest.mark.parametrize("shape", [(1, 2, 2, 700, 4200), (2, 4, 1, 1500, 4300)])
def test_backward_of_long_sequences(shape, mask, dt):
    """More than 4,096 keys and 512 queries: P and dS without what their rounding lost."""
    print("[case]", shape, mask, dt, flush=True)
    x = [t.cuda() for t in inputs(sum(shape), *shape, dt)]
    causal = mask in ("causal", "both")
    ql = kl = None
    if mask in ("ragged", "both"):
        ql, kl = lens(shape[0], shape[3], shape[4], 2)
    got = run(*x, causal=causal, q_lens=ql, k_lens=kl)
    want = R.attention(*x[:3], causal, ql, kl, do=x[3], dev="cuda", lo=True)
    check_all(got, want, (shape, mask, dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(1, 64, 64, 1000, 900), (1, 64, 64, 500, 900), (2, 64, 64, 300, 500)])
@pytest.mark.parametrize("causal", [False, True])
def test_a_rising_row_maximum_in_large_blocks(shape, causal, dt):
    """Keys in rising order of their score move the running bound at every tile."""
    print("[case]", shape, causal, dt, flush=True)
    q, k, v, do = inputs(9, *shape, dt)
    k = (k.float().abs() * torch.linspace(0.0, 4.0, shape[4])[:, None]).to(dt)
    x = [t.cuda() for t in (q.abs(), k, v, do)]
    check_all(run(*x, causal=causal), R.attention(*x[:3], causal, do=x[3], dev="cuda", lo=True),
              (shape, causal, dt))


@pytest.mark.parametrize("L", [500, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_infinite_scores_in_large_blocks(L, causal):
    """Rows with a score of +inf and rows whose scores are all -inf are NaN, no other row changes."""
    from imfvideo_amd import ops
    q, k, v, _ = (t.cuda() for t in inputs(18, 1, 64, 64, L, L, torch.bfloat16))
    k = k.abs() + 0.1
    want, _ = ops.dense_attn_fwd(q, k, v, causal)
    rows = [3, 5, 130, 257, L - 1]
    for i, r in enumerate(rows):
        q[:, :, r] = float("inf") if i % 2 else float("-inf")
    o, lse = ops.dense_attn_fwd(q, k, v, causal)
    keep = [i for i in range(L) if i not in rows]
    assert torch.isnan(o[:, :, rows]).all() and torch.isfinite(want).all()
    assert torch.equal(o[:, :, keep], want[:, :, keep])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("scale", [0.03, 0.5, 1.0])
@pytest.mark.parametrize("shape", [(1, 2, 2, 5, 900), (2, 4, 2, 150, 170), (1, 64, 64, 500, 200)])
def test_scales(shape, scale, dt):
    """The scale argument, forward and backward; q's gain keeps the exponents of the bounds."""
    print("[case]", shape, scale, dt, flush=True)
    q, *x = inputs(sum(shape), *shape, dt)
    q = (q.float() * min(1.0, 0.125 / scale)).to(dt)
    x = [t.cuda() for t in (q, *x)]
    check_all(run(*x, causal=True, scale=scale),
              R.attention(*x[:3], True, scale=scale, do=x[3], dev="cuda", lo=True),
              (shape, scale, dt))


@pytest.mark.parametrize("dt", DTYPES)
def test_one_program_of_forms_in_a_graph(dt):
    """A call of 256-row blocks, forward and backward, replayed on refilled inputs."""
    from imfvideo_amd import ops
    x = [t.cuda() for t in inputs(21, 3, 64, 16, 1000, 300, dt)]
    ql, kl = lens(3, 1000, 300, 3)

    def step():
        q, k, v, do = x
        o, lse, lo = ops.dense_attn_fwd(q, k, v, True, ql, kl, with_lo=True)
        return [o, lse, *ops.dense_attn_bwd(do, q, k, v, o, lse, True, ql, kl, o_lo=lo)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    for r in range(3):
        for t in x:
            t.copy_(torch.randn(t.shape, device="cuda"))
        kl.fill_(300 - 70 * r)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
