"""Dense attention's refusals, on the host: shapes, types, lengths, scale, and the C entries'
argument checks."""
import ctypes

import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import dense_attention


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        dense_attention(x, x, x)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.dense_attn_bwd(x, x, x, x, x, torch.zeros(1, 4, 2))


@pytest.mark.parametrize("shapes, match", [
    (((1, 2, 4, 32), (1, 2, 4, 32), (1, 2, 4, 32)), "64"),
    (((2, 4, 64), (2, 4, 64), (2, 4, 64)), "expected"),
    (((1, 2, 4, 64), (1, 2, 4, 64), (1, 2, 5, 64)), "share"),
    (((1, 3, 4, 64), (1, 2, 4, 64), (1, 2, 4, 64)), "divides"),
    (((2, 2, 4, 64), (1, 2, 4, 64), (1, 2, 4, 64)), "batch"),
])
def test_shapes(shapes, match):
    with pytest.raises(ValueError, match=match):
        ops.dense_attn_fwd(*(fake(*s) for s in shapes))


def test_types_scale_and_lengths():
    q = fake(2, 2, 4, 64)
    with pytest.raises(ValueError, match="share dtype"):
        ops.dense_attn_fwd(q, q, fake(2, 2, 4, 64, dtype=torch.float16))
    x = fake(2, 2, 4, 64, dtype=torch.float32)
    with pytest.raises(TypeError, match="16-bit"):
        ops.dense_attn_fwd(x, x, x)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            ops.dense_attn_fwd(q, q, q, scale=bad)
    for bad in ([1], torch.ones(2), torch.ones(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="k_lens"):
            ops.dense_attn_fwd(q, q, q, k_lens=bad)
    with pytest.raises(ValueError, match="lse"):
        ops.dense_attn_bwd(q, q, q, q, q, torch.zeros(2, 2, 5))
    with pytest.raises(ValueError, match="o_lo"):
        ops.dense_attn_bwd(q, q, q, q, q, torch.zeros(2, 2, 4), o_lo=fake(2, 2, 4, 64))
    with pytest.raises(ValueError, match="do"):
        ops.dense_attn_bwd(fake(2, 2, 5, 64), q, q, q, q, torch.zeros(2, 2, 4))


def test_c_entries_check_their_arguments():
    lib = _lib.load()
    bad = 1  # hipErrorInvalidValue
    st = lambda **kw: (ctypes.c_int64 * 24)(*[kw.get(f"s{i}", 64) for i in range(24)])

    def fwd(q=16, k=16, v=16, s=st(), dtype=1, B=1, H=2, Hkv=2, Lq=4, Lk=4, scale=0.125, o=16,
            lse=4, ws=None, lo=None):
        return lib.sla2h_dense_attn_fwd(q, k, v, s, None, None, dtype, B, H, Hkv, Lq, Lk, 0,
                                        scale, ws, o, lse, lo, None)

    def bwd(q=16, lse=4, s=st(), dtype=1, B=1, H=2, Hkv=2, Lq=4, Lk=4, scale=0.125, ws=16,
            lo=None, grads=(16, 16, 16)):
        return lib.sla2h_dense_attn_bwd(q, 16, 16, 16, lo, 16, lse, s, None, None, dtype, B, H, Hkv,
                                        Lq, Lk, 0, scale, ws, *grads, None)

    for f in (fwd, bwd):
        assert f(q=None) == bad and f(q=8) == bad          # missing, unaligned
        assert f(dtype=2) == bad and f(H=3) == bad         # fp32, heads that do not divide
        assert f(B=0) == bad and f(Lq=0) == bad and f(Lk=0) == bad
        assert f(scale=0.0) == bad and f(scale=float("nan")) == bad
        assert f(s=st(s1=4)) == bad and f(s=st(s4=-64)) == bad   # rows off 16 bytes, negative
        assert f(s=st(s5=1 << 23)) == bad                        # a row stride past 32-bit offsets
        assert f(s=st(s2=0)) == bad                              # rows on top of each other
        assert f(lse=2) == bad and f(lo=8) == bad
    assert bwd(lse=None) == bad and bwd(ws=None) == bad
    assert bwd(grads=(None, None, None)) == bad and bwd(grads=(16, 16, None)) == bad
    # few queries over many keys: the split form needs its workspace
    assert lib.sla2h_dense_attn_fwd_workspace_bytes(1, 1, 1, 1, 100_000) > 0
    assert fwd(H=1, Hkv=1, Lq=1, Lk=100_000) == bad
    assert lib.sla2h_dense_attn_fwd_workspace_bytes(1, 8, 8, 29952, 29952) == 0
    assert lib.sla2h_dense_attn_bwd_workspace_bytes(1, 1, 3, 2, 4, 4) == 0
