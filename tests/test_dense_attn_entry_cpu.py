"""What dense_attention and the modules around it may be asked for, on the host: calls that the
kernels cannot answer are refused, and nothing else is."""
import ctypes
import pickle
from functools import partial

import pytest
import torch

from imfvideo_amd import _lib, ops
from imfvideo_amd.imf_dit_video import (SwiGLUMlp, TransformerBlock, dense_attention,
                                        sdpa_math_attention)
from imfvideo_amd.mla_jvp_fast import pack_block


def block(impl):
    return TransformerBlock(64, 1, 32, 32, 32, 32, 64, attn_impl=impl)


@pytest.mark.parametrize("impl", [
    partial(dense_attention, causal=True),
    partial(dense_attention, scale=0.25),
    partial(dense_attention, k_lens=torch.tensor([3])),
    partial(dense_attention, q_lens=[3]),
    partial(partial(dense_attention, scale=0.25), causal=False),
    partial(partial(dense_attention, causal=True), scale=None),
])
def test_the_jvp_refuses_attention_that_it_does_not_compute(impl):
    """The fast JVP's dense branch is bidirectional over all tokens at scale 64^-1/2."""
    with pytest.raises(ValueError, match="dense_attention"):
        pack_block(block(impl))


@pytest.mark.parametrize("impl", [
    dense_attention, sdpa_math_attention, partial(dense_attention),
    partial(dense_attention, causal=False, q_lens=None, k_lens=None, scale=None),
    partial(dense_attention, scale=64 ** -0.5),
    partial(partial(dense_attention, causal=True), causal=0),
    lambda q, k, v: q,
])
def test_the_jvp_takes_plain_attention(impl):
    p, w16 = pack_block(block(impl))
    assert "cube" not in p and "sla2" not in p and w16["w_out"].dtype == torch.float16


@pytest.mark.parametrize("act8", [False, True])
def test_an_mlp_with_replaced_layers_runs(act8):
    """Layers that are no plain linears (an adapter around one, two in a row) run one by one."""
    torch.manual_seed(1)
    m = SwiGLUMlp(16, 24, act8=act8)
    x = torch.randn(5, 16, requires_grad=True)
    want = m(x)
    for n in ("w1", "w3", "w2"):
        setattr(m, n, torch.nn.Sequential(getattr(m, n)))
    assert torch.equal(m(x), want)


def test_modules_saved_whole_without_act8_run():
    """A module pickled before act8 existed has no such entry in its __dict__."""
    m = SwiGLUMlp(16, 24)
    del m.__dict__["act8"], m.act.__dict__["act8"]
    x = torch.randn(5, 16, requires_grad=True)
    m = pickle.loads(pickle.dumps(m))
    assert not m.act8 and not m.act.act8
    assert torch.equal(m(x), m.w2(m.act(m.w1(x), m.w3(x))))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64,
                                   torch.uint16, torch.uint32])
def test_lengths_of_every_whole_number_type(dtype):
    info = torch.iinfo(dtype)
    q = torch.zeros(5, 1, 1, 64)
    vals = [0, 1, 5, info.max, info.min]
    got = ops.attn_lens(torch.tensor(vals, dtype=dtype), q, "k_lens")
    assert got.dtype == torch.int32 and got.is_contiguous()
    # below zero nothing, above 32 bits more than any length has
    clamped = [min(max(v, -2 ** 31), 2 ** 31 - 1) for v in vals]
    assert [max(v, 0) for v in got.tolist()] == [max(v, 0) for v in clamped]


def test_lengths_that_are_no_whole_numbers_of_int64():
    q = torch.zeros(1, 1, 1, 64)
    for bad in ([0.5], [True], torch.tensor([1], dtype=torch.uint64)):
        with pytest.raises(ValueError, match="k_lens"):
            ops.attn_lens(bad, q, "k_lens")


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the checks run, no launch is reached."""
    is_cuda = property(lambda self: True)


def test_forward_and_backward_take_the_same_sizes():
    """What the forward answers has a backward: as many heads, lengths and groups."""
    lib = _lib.load()
    st = (ctypes.c_int64 * 24)(*[64] * 24)
    bad, ok = 1, lambda *s: lib.sla2h_dense_attn_bwd_workspace_bytes(1, *s) > 0
    for sizes, good in (((8200, 8, 8, 3, 3), True), ((1, 65536, 1, 1, 1), True),
                        ((2 ** 20 - 1, 1, 1, 1, 1), True), ((2 ** 20, 1, 1, 1, 1), False),
                        ((1, 2, 2, 2 ** 30, 1), False), ((1, 2, 2, 1, 2 ** 30), False),
                        ((1, 8, 1, 2 ** 28, 1), False), ((1, 3, 2, 4, 4), False)):
        assert ok(*sizes) == good, sizes
        if not good:
            assert lib.sla2h_dense_attn_fwd(16, 16, 16, st, None, None, 1, *sizes, 0, 0.125, 16, 16,
                                            4, None, None) == bad
            assert lib.sla2h_dense_attn_bwd(16, 16, 16, 16, None, 16, 4, st, None, None, 1, *sizes,
                                            0, 0.125, 16, 16, 16, 16, None) == bad


@pytest.mark.parametrize("shape", [(2 ** 20, 1, 2, 64), (1, 2 ** 20, 2, 64), (1, 1, 2 ** 30, 64)])
def test_sizes_past_the_kernels_are_refused_by_name(shape):
    """The forward refuses what it or its backward could not launch."""
    shape = torch.Size(shape)
    strides = (shape[1] * shape[2] * 64, shape[2] * 64, 64, 1)
    with pytest.raises(ValueError, match="too large"):
        ops._attn_plan(shape, strides, shape, strides, shape, strides, torch.bfloat16, False)


def test_rows_too_far_apart_are_refused_by_name():
    """2^17 heads of 64 channels side by side: rows past the 32-bit offsets of a tile, in a copy too."""
    x = torch.zeros(1, 2, 2 ** 17, 64, dtype=torch.bfloat16).as_subclass(_Gpu)
    with pytest.raises(ValueError, match="too large"):
        ops.dense_attn_fwd(x, x, x, tok=True)
