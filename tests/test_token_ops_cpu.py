"""Refusals of the transformer-block operators and their C entry points, and the host-side helpers.  No kernel is launched."""
import ctypes

import pytest
import torch

import gan_amd
from gan_amd import _lib, token_ops

F = gan_amd.functional


def test_norm_refusals():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        F.block_input_norm(x)
    with pytest.raises(RuntimeError, match="kind"):
        F.block_input_norm(x, kind="batch")
    with pytest.raises(RuntimeError, match=r"\[B, ..., C\]"):
        F.block_input_norm(torch.zeros(8))
    with pytest.raises(RuntimeError, match="shape and dtype"):
        F.block_output_norm(x, torch.zeros(2, 3, 4))
    with pytest.raises(RuntimeError, match="shape and dtype"):
        F.block_boundary_norm(x, x.bfloat16())
    with pytest.raises(RuntimeError, match="f must be"):
        F.block_output_norm(x, None)
    with pytest.raises(RuntimeError, match="8192"):
        F.block_input_norm(torch.zeros(1, 1, 8193))
    with pytest.raises(RuntimeError, match="eps"):
        F.block_input_norm(x, eps=0.0)
    with pytest.raises(RuntimeError, match="dtype"):
        F.block_input_norm(x.half())


def test_rotary_refusals_and_table():
    t = F.rotary_table((4, 6), base=(100.0, 10.0))
    assert t.pairs == 5 and t.axes == 2 and t.axis.tolist() == [0, 0, 1, 1, 1] and t.interleaved
    want = torch.tensor([1.0, 0.1, 1.0, 10.0 ** (-1 / 3), 10.0 ** (-2 / 3)], dtype=torch.float64) / (2 * torch.pi)
    assert torch.allclose(t.turns, want, rtol=1e-14, atol=0)
    for bad in ((3,), (), (0, 2), (512, 2)):
        with pytest.raises(RuntimeError, match="dims|rotated"):
            F.rotary_table(bad)
    with pytest.raises(RuntimeError, match="base"):
        F.rotary_table((4, 4), base=(10.0,))
    q, pos = torch.zeros(2, 5, 3, 16), torch.zeros(5, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        F.axial_rotary(q, None, pos, t)
    with pytest.raises(RuntimeError, match="heads have"):
        F.axial_rotary(q[..., :8], None, pos, t)
    with pytest.raises(RuntimeError, match="positions must be"):
        F.axial_rotary(q, None, pos[:, :1], t)
    with pytest.raises(RuntimeError, match="positions must be"):
        F.axial_rotary(q, None, pos.bool(), t)
    with pytest.raises(RuntimeError, match="k must be"):
        F.axial_rotary(q, q[:, :4], pos, t)
    with pytest.raises(RuntimeError, match="rotary_table"):
        F.axial_rotary(q, None, pos, None)


def test_attention_refusals():
    bf = torch.bfloat16
    q, k, v, lam = torch.zeros(2, 5, 4, 2, 16, dtype=bf), torch.zeros(2, 7, 2, 2, 16, dtype=bf), torch.zeros(2, 7, 2, 32, dtype=bf), torch.zeros(4)
    call = F.differential_attention
    with pytest.raises(RuntimeError, match="GPU"):
        call(q, k, v, lam)
    with pytest.raises(RuntimeError, match="bf16"):
        call(q.float(), k, v, lam)
    with pytest.raises(RuntimeError, match="lam"):
        call(q, k, v, lam[:3])
    with pytest.raises(RuntimeError, match="go together"):
        call(q[:, :, :3], k, v, lam[:3])
    with pytest.raises(RuntimeError, match="go together"):
        call(q, k[:, :6], v, lam)
    with pytest.raises(RuntimeError, match="takes q"):
        call(q[:, :, :, 0], k, v, lam)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(q[..., :12], k[..., :12], v, lam)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(torch.zeros(2, 5, 4, 2, 136, dtype=bf), torch.zeros(2, 7, 2, 2, 136, dtype=bf), v, lam)
    with pytest.raises(RuntimeError, match="scale"):
        call(q, k, v, lam, scale=0.0)
    with pytest.raises(RuntimeError, match="scale"):
        call(q, k, v, lam, scale=1e-38)
    with pytest.raises(RuntimeError, match="key_lengths"):
        call(q, k, v, lam, key_lengths=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="key_lengths"):
        call(q, k, v, lam, key_lengths=torch.zeros(2))


def _attention_desc(**kw):
    d = _lib.DiffAttention()
    base = dict(B=2, NQ=100, NK=100, H=4, HK=2, d=64, dv=128, causal=0, scale=0.125)
    base.update(kw)
    for n, val in base.items():
        setattr(d, n, val)
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = (51200, 512, 128, 64), (25600, 256, 128, 64), (25600, 256, 128)
    for n in ("q", "k", "v", "lam", "out", "out2", "lse", "dout", "dq", "dk", "dv_out", "dlam"):
        if n not in kw:
            setattr(d, n, 256)
    return d


def test_attention_entry_points_validate_before_any_launch():
    L = _lib.lib()
    fwd = lambda d, ws=None, n=0: L.gc_diff_attention_fwd(ctypes.byref(d), ws, n, None)
    bwd = lambda d, ws=None, n=0: L.gc_diff_attention_bwd(ctypes.byref(d), ws, n, None)
    assert L.gc_diff_attention_fwd(None, None, 0, None) == -5
    for bad in (dict(d=12), dict(d=136), dict(dv=264), dict(dv=0), dict(H=3), dict(HK=0), dict(NQ=-1), dict(NK=1 << 30)):
        assert fwd(_attention_desc(**bad)) == -2, bad
    for bad in (dict(q=None), dict(k=264), dict(out=8), dict(lam=None), dict(scale=0.0), dict(scale=float("nan"))):
        assert fwd(_attention_desc(**bad)) == -5, bad
    d = _attention_desc()
    d.k_stride[1] = 20
    assert fwd(d) == -5
    d = _attention_desc()
    d.v_stride[1] = 64                                   # rows that overlap
    assert fwd(d) == -2
    d = _attention_desc()
    d.q_stride[1] = 1 << 23
    assert fwd(d) == -2
    assert fwd(_attention_desc(B=0)) == 0 and fwd(_attention_desc(NQ=0)) == 0
    long = _attention_desc(NQ=1, NK=65536)
    assert L.gc_diff_attention_workspace_bytes(ctypes.byref(long), 0) > 0
    assert fwd(long) == -3 and b"workspace" in L.gc_last_error()
    need = L.gc_diff_attention_workspace_bytes(ctypes.byref(_attention_desc()), 1)
    assert need >= 2 * 4 * 100 * 2 * 4 and bwd(_attention_desc(), 256, need - 1) == -3 and bwd(_attention_desc(), 264, need) == -3
    assert bwd(_attention_desc(dq=None), 256, need) == -5 and bwd(_attention_desc(NK=0), 256, need) == -5


def test_norm_and_rotary_entry_points_validate_before_any_launch():
    L = _lib.lib()
    d = _lib.BlockNorm()
    d.batch, d.rows, d.cols, d.eps, d.with_input_norm = 2, 3, 64, 1e-6, 1
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == -5                        # no x
    d.x = 256
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == -5                        # no h
    d.h = 256
    d.dtype = 7
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == -5
    d.dtype, d.cols = 0, 8193
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == -2
    d.cols, d.with_input_norm = 64, 0
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == -5                        # neither part
    d.with_input_norm, d.batch = 1, 0
    assert L.gc_block_norm_fwd(ctypes.byref(d), None) == 0
    d.batch = 2
    assert L.gc_block_norm_bwd(ctypes.byref(d), 256, 1 << 20, None) == -5          # no statistics, no gradients
    d.stats, d.dh, d.dx = 256, 256, 256
    need = L.gc_block_norm_workspace_bytes(2, 3, 64)
    assert need >= 2 * 5 * 64 * 4 and L.gc_block_norm_bwd(ctypes.byref(d), 256, need - 1, None) == -3
    r = _lib.Rotary()
    r.batch, r.tokens, r.q_heads, r.dim, r.pairs, r.axes = 2, 3, 4, 16, 8, 2
    assert L.gc_axial_rotary(ctypes.byref(r), None) == -5
    r.q = r.q_out = r.positions = r.pair_turns = r.pair_axis = 256
    r.pairs = 9
    assert L.gc_axial_rotary(ctypes.byref(r), None) == -2
    r.pairs, r.k_heads = 8, 1
    assert L.gc_axial_rotary(ctypes.byref(r), None) == -5                          # k is missing
    r.k_heads, r.tokens = 0, 0
    assert L.gc_axial_rotary(ctypes.byref(r), None) == 0


def test_layout_helpers():
    t = torch.zeros(3, 10, 200)
    v, b, r = token_ops._rows(t[:, 2:9, 64:128])
    assert v.data_ptr() == t[:, 2:9, 64:128].data_ptr() and (b, r) == (2000, 200)
    v, b, r = token_ops._rows(t[:, ::2, :64])
    assert (b, r) == (2000, 400)
    v, b, r = token_ops._rows(t[:1].expand(3, 10, 200))
    assert (b, r) == (0, 200)
    v, b, r = token_ops._rows(t[:, :1].expand(3, 10, 200))                          # rows on top of each other: copied
    assert v.is_contiguous() and (b, r) == (2000, 200)
    v, b, r = token_ops._rows(t.transpose(1, 2))
    assert v.is_contiguous() and (b, r) == (2000, 10)
    v, b, r = token_ops._rows(torch.zeros(2, 4, 5, 32)[:, :, 1:4])                  # rows of two strides: copied
    assert v.is_contiguous()
    assert token_ops._strides(torch.zeros(4, 1, 8).expand(4, 1, 8).as_strided((4, 1, 8), (8, 3, 1))) == [8, 8, 1]
    q = torch.zeros(2, 1, 3, 2, 32, dtype=torch.bfloat16)
    assert token_ops._aligned(q, 32)[0] is q and token_ops._aligned(q, 32)[1] == [192, 192, 64, 32]
    assert token_ops._aligned(q.expand(2, 5, 3, 2, 32), 32)[0].is_contiguous()
    wide = torch.zeros(2, 4, 3, 2, 40, dtype=torch.bfloat16)[..., :32]
    v, st = token_ops._aligned(wide, 32)
    assert v.data_ptr() == wide.data_ptr() and st == [960, 240, 80, 40]
    assert token_ops._aligned(wide[..., 1:], 31)[0].is_contiguous()


def test_packed_descriptors_match_the_structures():
    """The one-line packings against the field-by-field structures of the C ABI."""
    for packer, cls in ((token_ops._NORM, _lib.BlockNorm), (token_ops._ROTARY, _lib.Rotary), (token_ops._ATTENTION, _lib.DiffAttention)):
        assert packer.size == ctypes.sizeof(cls)
        flat = []
        for name, kind in cls._fields_:
            n = getattr(kind, "_length_", 1)
            flat += [(name, i if n > 1 else None) for i in range(n)]
        values = [float(i + 1) if getattr(cls, name).size == 4 and dict(cls._fields_)[name] is ctypes.c_float else i + 1 for i, (name, _) in enumerate(flat)]
        d = cls.from_buffer_copy(packer.pack(*values))
        for (name, i), value in zip(flat, values):
            got = getattr(d, name) if i is None else getattr(d, name)[i]
            assert got == value, (cls.__name__, name, i)


def test_modules_and_the_biggan_option():
    import copy

    from gan_amd.harness import biggan as H
    m = gan_amd.nn.DifferentialAttention2d(128, depth=2)
    assert m.blocks[0].heads == 2 and m.blocks[0].head_dim == 32 and m.blocks[0].rotary.dims == (16, 16)
    names = set(dict(m.named_parameters()))
    assert {"blocks.0.qkv.weight", "blocks.1.out.weight", "blocks.0.lambda_q1", "blocks.0.head_norm", "in_norm.1", "out_norm.0", "gate.1"} <= names
    assert not list(m.buffers()) and torch.equal(m.blocks[0].lam().detach().shape and m.blocks[0].lam() * 0, torch.zeros(2))
    c = copy.deepcopy(m)
    c.load_state_dict(m.state_dict())
    with pytest.raises(RuntimeError, match="GPU"):
        m(torch.zeros(1, 128, 4, 4))
    with pytest.raises(RuntimeError, match="expected"):
        m(torch.zeros(1, 64, 4, 4))
    with pytest.raises(ValueError, match="heads"):
        gan_amd.nn.DifferentialAttention2d(40)
    gan_amd.set_precision("fp32x3")
    try:
        with pytest.raises(RuntimeError, match="bf16"):
            m(torch.zeros(1, 128, 4, 4))
    finally:
        gan_amd.set_precision("bf16")
    torch.manual_seed(0)
    plain = H.Generator(10, 16).state_dict()
    torch.manual_seed(0)
    again = H.Generator(10, 16, attention="self").state_dict()
    assert list(plain) == list(again) and all(torch.equal(plain[n], again[n]) for n in plain)
    g, d = H.Generator(10, 16, attention="differential"), H.Discriminator(10, 16, attention="differential")
    assert isinstance(g.main_sequence[4], H.DifferentialAttentionBlock) and isinstance(d.main_sequence[1], H.DifferentialAttentionBlock)
    assert "main_sequence.4.blocks.0.qkv.U_vector" in g.state_dict()
    with pytest.raises(KeyError):
        H.Generator(10, 16, attention="none")


def test_positions_made_in_inference_mode_serve_training():
    from gan_amd import nn as gnn

    block = gnn.DifferentialAttention2d(32, heads=1)
    with torch.inference_mode():
        first = block.positions(3, 5, torch.device("cpu"))
    assert not first.is_inference() and block.positions(3, 5, torch.device("cpu")) is first
    assert first.tolist() == [[i, j] for i in range(3) for j in range(5)]
