"""8-bit activations on the host: refusals of the ops and the C entries, and the modules'
CPU form."""
import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import SituAndMul, SwiGLUMlp, TransformerBlock


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


def act(rows, cols, **kw):
    rb, cb = -(-rows // 64), -(-cols // 64)
    return ops.Act8(fake(rb, cb, 64, 64, dtype=torch.int8), fake(rb, cb, dtype=torch.float32),
                    kw.get("r", rows), kw.get("c", cols))


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for f in (lambda: ops.act8_pack(x), lambda: ops.situ8_fwd(x, x, 4.0),
              lambda: ops.situ8_bwd(x, act(4, 8), act(4, 8), 4.0),
              lambda: ops.linear_wgrad8(x, act(4, 8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            f()


def test_refusals():
    with pytest.raises(TypeError, match="16-bit"):
        ops.act8_pack(fake(4, 8, dtype=torch.float32))
    with pytest.raises(ValueError, match="nothing"):
        ops.act8_pack(fake(0, 8))
    with pytest.raises(ValueError, match="share"):
        ops.situ8_fwd(fake(4, 8), fake(4, 9), 4.0)
    for beta, lb in ((0.0, None), (float("nan"), None), (4.0, -1.0), (4.0, float("inf"))):
        with pytest.raises(ValueError, match="beta"):
            ops.situ8_fwd(fake(4, 8), fake(4, 8), beta, lb)
    with pytest.raises(ValueError, match="does not fit"):
        ops.situ8_bwd(fake(4, 9), act(4, 8), act(4, 8), 4.0)
    with pytest.raises(ValueError, match="does not fit"):
        ops.situ8_bwd(fake(4, 8), act(4, 8), act(4, 16), 4.0)
    with pytest.raises(ValueError, match="not the 8-bit tiles"):
        ops.situ8_bwd(fake(4, 8), act(4, 8, c=65), act(4, 8), 4.0)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_wgrad8(fake(5, 8), act(4, 8))
    with pytest.raises(ValueError, match="not the 8-bit tiles"):
        ops.linear_wgrad8(fake(65, 8), act(4, 8, r=65))


def test_c_entries_check_their_arguments():
    lib, bad = _lib.load(), 1
    assert lib.sla2h_act8_pack(None, 8, 1, 4, 8, 16, 4, None) == bad
    assert lib.sla2h_act8_pack(16, 7, 1, 4, 8, 16, 4, None) == bad       # rows overlap
    assert lib.sla2h_act8_pack(16, 8, 2, 4, 8, 16, 4, None) == bad       # fp32
    assert lib.sla2h_act8_pack(16, 8, 1, 0, 8, 16, 4, None) == bad
    assert lib.sla2h_act8_pack(16, 8, 1, 4, 8, 8, 4, None) == bad        # codes off 16 bytes
    assert lib.sla2h_act8_unpack(16, 4, 1, 4, 0, 16, None) == bad
    assert lib.sla2h_situ8_fwd(16, 16, 1, 4, 8, 8, 8, 0.0, 0.0, 16, 16, 4, 16, 4, None) == bad
    assert lib.sla2h_situ8_fwd(16, 16, 1, 4, 8, 7, 8, 4.0, 0.0, 16, 16, 4, 16, 4, None) == bad
    assert lib.sla2h_situ8_bwd(16, 8, 16, 4, 16, 4, 1, 4, 8, 4.0, 0.0, 7, 16, 16, None,
                               None) == bad
    assert lib.sla2h_linear_wgrad8(16, 7, 16, 4, 1, 4, 8, 8, None, 16, None) == bad
    assert lib.sla2h_linear_wgrad8(16, 1 << 23, 16, 4, 1, 4, 8, 8, None, 16, None) == bad
    need = lib.sla2h_linear_wgrad8_workspace_bytes(59904, 160, 512)
    assert need > 0 and need % (160 * 512 * 4) == 0
    assert lib.sla2h_linear_wgrad8(16, 160, 16, 4, 1, 59904, 160, 512, None, 16, None) == bad


def test_modules_on_the_cpu_are_the_plain_ones():
    torch.manual_seed(0)
    x = torch.randn(5, 16, requires_grad=True)
    assert torch.equal(SituAndMul(4.0, 25.0, act8=True)(x), SituAndMul(4.0, 25.0)(x))
    a, b = SwiGLUMlp(16, 24, act8=True), SwiGLUMlp(16, 24)
    b.load_state_dict(a.state_dict())
    assert torch.equal(a(x), b(x))
    blk = TransformerBlock(64, 1, 32, 32, 32, 32, 64, act8=True)
    assert blk.mlp.act8 and blk.mlp.act.act8
    assert set(blk.state_dict()) == set(TransformerBlock(64, 1, 32, 32, 32, 32, 64).state_dict())
