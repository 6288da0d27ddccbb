"""Differential attention's refusals, on the host: shapes, types, weights, lengths, scale, the C
entries' argument checks and the modules around it."""
import ctypes
from functools import partial

import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import DiffAttentionImpl, TransformerBlock, diff_attention
from imfvideo_amd.mla_jvp_fast import pack_block


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Gpu)


def lam(n, dtype=torch.float32):
    return fake(n, dtype=dtype)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        diff_attention(x, x, x, torch.zeros(1))
    q = fake(1, 4, 2, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        diff_attention(q, q, q, torch.zeros(1))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.diff_attn_bwd(x, x, x, x, torch.zeros(1), torch.zeros(1, 2, 4),
                          torch.zeros(1, 4, 1, 2, 128))


@pytest.mark.parametrize("shapes, match", [
    (((1, 4, 2, 32), (1, 4, 2, 32), (1, 4, 2, 32)), "64"),
    (((4, 2, 64), (4, 2, 64), (4, 2, 64)), "expected"),
    (((1, 4, 2, 64), (1, 4, 2, 64), (1, 5, 2, 64)), "share"),
    (((1, 4, 2, 64), (1, 4, 2, 64), (1, 4, 4, 64)), "share"),
    (((1, 4, 6, 64), (1, 4, 4, 64), (1, 4, 4, 64)), "divides"),
    (((1, 4, 3, 64), (1, 4, 3, 64), (1, 4, 3, 64)), "even"),
    (((1, 4, 2, 64), (1, 4, 1, 64), (1, 4, 1, 64)), "even"),
    (((1, 4, 2, 64), (1, 4, 0, 64), (1, 4, 0, 64)), "even"),
    (((2, 4, 2, 64), (1, 4, 2, 64), (1, 4, 2, 64)), "batch"),
])
def test_shapes(shapes, match):
    with pytest.raises(ValueError, match=match):
        ops.diff_attn_fwd(*(fake(*s) for s in shapes), lam(shapes[0][-2] // 2))


def test_types_weights_scale_and_lengths():
    q, w = fake(2, 3, 4, 64), lam(2)
    with pytest.raises(ValueError, match="share their dtype"):
        ops.diff_attn_fwd(q, q, fake(2, 3, 4, 64, dtype=torch.float16), w)
    x = fake(2, 3, 4, 64, dtype=torch.float32)
    with pytest.raises(TypeError, match="16-bit"):
        ops.diff_attn_fwd(x, x, x, w)
    for bad in (lam(4), lam(1), fake(2, 1, dtype=torch.float32), lam(2, torch.int32),
                fake(dtype=torch.float32)):
        with pytest.raises(ValueError, match="lam"):
            ops.diff_attn_fwd(q, q, q, bad)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            ops.diff_attn_fwd(q, q, q, w, scale=bad)
    for bad in ([1], torch.ones(2), torch.ones(2, 1, dtype=torch.int32), [0.5, 1]):
        with pytest.raises(ValueError, match="k_lens"):
            diff_attention(q, q, q, w, k_lens=bad)
        with pytest.raises(ValueError, match="q_lens"):
            diff_attention(q, q, q, w, q_lens=bad)
    lse, maps = torch.zeros(2, 4, 3), torch.zeros(2, 3, 2, 2, 128)
    with pytest.raises(ValueError, match="do"):
        ops.diff_attn_bwd(fake(2, 5, 4, 64), q, q, q, w, lse, maps)
    with pytest.raises(ValueError, match="lse"):
        ops.diff_attn_bwd(q, q, q, q, w, torch.zeros(2, 3, 4), maps)
    with pytest.raises(ValueError, match="maps"):
        ops.diff_attn_bwd(q, q, q, q, w, lse, maps.double())


def test_c_entries_check_their_arguments():
    lib = _lib.load()
    bad = 1  # hipErrorInvalidValue
    st = lambda **kw: (ctypes.c_int64 * 9)(*[kw.get(f"s{i}", 64) for i in range(9)])

    def fwd(q=16, k=16, v=16, lam=16, lt=2, ls=1, s=st(), ql=None, dtype=1, B=1, H=2, Hkv=2, Lq=4,
            Lk=4, scale=0.125, ws=None, o=16, lse=4, maps=16):
        return lib.sla2h_diff_attn_fwd(q, k, v, lam, lt, ls, s, ql, None, dtype, B, H, Hkv, Lq, Lk,
                                       0, scale, ws, o, lse, maps, None)

    def bwd(q=16, k=16, v=16, lam=16, lt=2, ls=1, s=st(), ql=None, dtype=1, B=1, H=2, Hkv=2, Lq=4,
            Lk=4, scale=0.125, ws=16, o=16, lse=4, maps=16, grads=(16, 16, 16), dlam=16):
        return lib.sla2h_diff_attn_bwd(q, k, v, lam, lt, ls, o, lse, maps, s, ql, None, dtype, B,
                                       H, Hkv, Lq, Lk, 0, scale, ws, *grads, dlam, None)

    for f in (fwd, bwd):
        for name in ("q", "k", "v", "o"):
            assert f(**{name: None}) == bad and f(**{name: 8}) == bad, name  # missing, unaligned
        assert f(lam=None) == bad and f(lam=2) == bad and f(lt=3) == bad and f(ls=-1) == bad
        assert f(dtype=2) == bad and f(H=3, Hkv=3) == bad and f(H=6, Hkv=4) == bad
        assert f(B=0) == bad and f(Lq=0) == bad and f(Lk=0) == bad
        assert f(scale=0.0) == bad and f(scale=float("nan")) == bad
        assert f(s=None) == bad and f(s=st(s1=4)) == bad and f(s=st(s4=-64)) == bad
        assert f(s=st(s5=1 << 23)) == bad and f(s=st(s8=1 << 23)) == bad
        assert f(s=st(s2=0)) == bad                              # rows on top of each other
        assert f(lse=2) == bad and f(maps=8) == bad and f(ql=2) == bad
        assert f(maps=None) == bad
    assert fwd(lse=None) == bad                                  # both or neither
    assert bwd(lse=None) == bad and bwd(ws=None) == bad and bwd(dlam=None) == bad
    assert bwd(grads=(16, 16, None)) == bad and bwd(grads=(16, None, 16)) == bad
    # few queries over many keys: the split form needs its workspace
    assert lib.sla2h_diff_attn_fwd_workspace_bytes(1, 2, 2, 1, 100_000) > 0
    assert fwd(Lq=1, Lk=100_000) == bad
    assert lib.sla2h_diff_attn_fwd_workspace_bytes(1, 8, 8, 29952, 29952) == 0


def test_forward_and_backward_take_the_same_sizes():
    lib = _lib.load()
    st = (ctypes.c_int64 * 9)(*[64] * 9)
    bad, ok = 1, lambda *s: lib.sla2h_diff_attn_bwd_workspace_bytes(1, *s) > 0
    for sizes, good in (((8200, 8, 8, 3, 3), True), ((1, 65536, 2, 1, 1), True),
                        ((2 ** 20, 2, 2, 1, 1), False), ((1, 2, 2, 2 ** 30, 1), False),
                        ((1, 2, 2, 1, 2 ** 30), False), ((1, 16, 2, 2 ** 28, 1), False),
                        ((1, 6, 4, 4, 4), False), ((1, 3, 3, 4, 4), False)):
        assert ok(*sizes) == good, sizes
        if not good:
            assert lib.sla2h_diff_attn_fwd(16, 16, 16, 16, 2, 1, st, None, None, 1, *sizes, 0, 0.125,
                                           16, 16, 4, 16, None) == bad
            assert lib.sla2h_diff_attn_bwd(16, 16, 16, 16, 2, 1, 16, 4, 16, st, None, None, 1,
                                           *sizes, 0, 0.125, 16, 16, 16, 16, 16, None) == bad


@pytest.mark.parametrize("shape", [(2 ** 20, 1, 2, 64), (1, 2 ** 30, 2, 64), (1, 1, 2 ** 30, 64)])
def test_sizes_past_the_kernels_are_refused_by_name(shape):
    shape = torch.Size(shape)
    strides = (shape[1] * shape[2] * 64, shape[2] * 64, 64, 1)
    with pytest.raises(ValueError, match="too large"):
        ops._diff_plan(shape, strides, shape, strides, shape, strides, torch.bfloat16)


def test_rows_too_far_apart_are_refused_by_name():
    """2^17 heads of 64 channels side by side: rows past the 32-bit offsets of a tile, in a copy too."""
    x = torch.zeros(1, 2, 2 ** 17, 64, dtype=torch.bfloat16).as_subclass(_Gpu)
    with pytest.raises(ValueError, match="too large"):
        ops.diff_attn_fwd(x, x, x, lam(2 ** 16))


def test_the_module():
    for head_dim, heads in ((32, 4), (64, 3), (64, 0), (64, 1)):
        with pytest.raises(ValueError, match="pairs"):
            DiffAttentionImpl(head_dim, heads)
    m = DiffAttentionImpl(64, 4, lambda_init=0.3)
    with torch.no_grad():
        m.lambda_q1.fill_(0.1), m.lambda_k1.fill_(0.2), m.lambda_q2.fill_(0.0)
    want = torch.tensor(64 * 0.02).exp() - 1 + 0.3
    assert abs(m.weight().item() - want.item()) < 1e-5
    grads = torch.autograd.grad(m.weight(), [m.lambda_q1, m.lambda_k2])
    # d exp(a . b) / da = exp(a . b) b;  the second dot product is 0
    assert torch.allclose(grads[0], torch.tensor(64 * 0.02).exp() * m.lambda_k1)
    assert torch.equal(grads[1], -m.lambda_q2)


def test_a_packed_block_refuses_it():
    """The JVP chain computes plain attention only."""
    for impl in (diff_attention, partial(DiffAttentionImpl, num_heads=2)):
        b = TransformerBlock(128, 2, 64, 64, 32, 32, 64, attn_impl=impl)
        with pytest.raises(ValueError):
            pack_block(b)
