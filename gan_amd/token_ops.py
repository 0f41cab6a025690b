"""Operators of image / video transformer blocks over libganconv.so: the norms before and after a block, rotary positions with
several axes, differential attention.  Extensions beside the reference's one attention block (BigGAN/model.py:80-105); tokens lie
in rows, an image [B, C, H, W] in channels-last memory being [B, H * W, C].

Unlike the convolutions these are plain autograd functions, not torch.library operators: a call and its backward pass cost
30 us of host time less that way, which is what a single token costs altogether.  First-order gradients only.  There is no
fallback: on a CPU tensor or an unsupported geometry they raise RuntimeError.
"""
import contextlib
import ctypes

import torch

from . import _lib

_NO_CONTEXT = contextlib.nullcontext()


def _on(t):
    """Context that makes t's device the current one (launches, streams and allocations follow it)."""
    return _NO_CONTEXT if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _require(cond, msg):
    if not cond:
        raise RuntimeError("ganconv: " + msg)


def _same_gpu(who, first, *rest):
    _require(first.is_cuda, f"{who}: tensors must live on the GPU (this library has no CPU path)")
    for t in rest:
        _require(t is None or t.device == first.device, f"{who}: all tensors must be on one device (got {first.device} and {None if t is None else t.device})")


def _code(who, t):
    if t.dtype == torch.bfloat16:
        return _lib.GC_BF16
    _require(t.dtype == torch.float32, f"{who}: unsupported dtype {t.dtype} (float32 or bfloat16)")
    return _lib.GC_F32


def _p(t):
    return None if t is None else t.data_ptr()


def _graph_follows(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _strides(t):
    """t's strides, with those of dimensions of one element (where torch allows anything) as in a contiguous tensor."""
    out, step = [], 1
    for n, st in zip(reversed(t.shape), reversed(t.stride())):
        out.append(st if n != 1 else step)
        step *= n
    return out[::-1]


class _OnceOnly(torch.autograd.Function):
    """Base of the functions here: a backward pass that would itself be differentiated is refused."""

    @staticmethod
    def refuse_second_order(who, *grads):
        if torch.is_grad_enabled() and any(g is not None and g.requires_grad for g in grads):
            raise RuntimeError(f"ganconv: {who} has no second-order backward")


# ---- norms before and after a block ----------------------------------------------------------------------------------------
def _rows(t, shared=False):
    """(tensor, batch stride, row stride) of [B, ..., C] read as [B, rows, C] with contiguous channels; copied if its rows do not
    lie at one stride (or overlap).  A [B, C] tensor is B samples of one row, or with `shared` one sample of B rows."""
    if t.dim() == 2:
        t = t.unsqueeze(0 if shared else 1)
    if t.is_contiguous():
        C = t.shape[-1]
        return t, (t.numel() // t.shape[0] if t.shape[0] else 0), C
    st = _strides(t)
    ok = st[-1] == 1 and st[-2] >= t.shape[-1]
    for i in range(1, t.dim() - 2):
        ok = ok and st[i] == st[i + 1] * t.shape[i + 1]
    return (t, st[0], st[-2]) if ok else _rows(t.contiguous())


def _param(who, name, t, C, B=None):
    """fp32 contiguous copy-or-self of a [C] (or, with B, [B, C]) parameter and whether it is per sample."""
    if t is None:
        return None, 0
    per_sample = B is not None and t.dim() == 2
    _require(tuple(t.shape) == ((B, C) if per_sample else (C,)),
             f"{who}: {name} must be [{C}]" + (f" or [{B}, {C}]" if B is not None else "") + f", got {tuple(t.shape)}")
    _require(t.dtype in (torch.float32, torch.bfloat16), f"{who}: {name} must be float32 or bfloat16, got {t.dtype}")
    t = t.detach()
    return (t if t.dtype == torch.float32 else t.float()).contiguous(), int(per_sample)


_KINDS = {"rms": 0, "layer": 1}


class _BlockNorm(_OnceOnly):
    """forward(cfg, x, f, out_weight, out_bias, gate, residual_scale, in_weight, in_bias, scale, shift) -> y, h or one of them.
    cfg: (who, kind code, eps, with_input_norm, residual constant, a backward pass may follow)."""

    @staticmethod
    def forward(ctx, cfg, x, f, out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift):
        who, layer, eps, with_in, constant, grads = cfg
        B, C = x.shape[0], x.shape[-1]
        given = (out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift)
        d = _lib.BlockNorm()
        ow, _ = _param(who, "out_weight", out_weight, C)
        ob, _ = _param(who, "out_bias", out_bias, C)
        gt, d.gate_per_sample = _param(who, "gate", gate, C, B)
        iw, _ = _param(who, "in_weight", in_weight, C)
        ib, _ = _param(who, "in_bias", in_bias, C)
        sc, ps = _param(who, "scale", scale, C, B)
        sh, qs = _param(who, "shift", shift, C, B)
        _require(sc is None or sh is None or ps == qs, f"{who}: scale and shift must both be [C] or both [B, C]")
        d.mod_per_sample = ps or qs
        rt = None
        if rho is not None:
            _require(rho.numel() in (1, C) and rho.dim() <= 1, f"{who}: residual_scale must be a number, one element or [{C}], got {tuple(rho.shape)}")
            d.residual_per_channel = int(rho.numel() == C and C > 1)
            rt = rho.detach().float().contiguous()
        d.residual_constant = constant
        shared = not (d.gate_per_sample or d.mod_per_sample)   # nothing tells the samples apart: one run of rows where they lie so
        xr, d.x_batch_stride, d.x_row_stride = _rows(x, shared)
        fr = None
        if f is not None:
            fr, d.f_batch_stride, d.f_row_stride = _rows(f, shared)
        rows = x.numel() // (B * C) if B else 0
        d.batch, d.rows, d.cols = B, rows, C
        if shared and (x.dim() == 2 or (d.x_batch_stride == rows * d.x_row_stride and (fr is None or d.f_batch_stride == rows * d.f_row_stride))):
            d.batch, d.rows = 1, B * rows
        d.dtype, d.layer, d.with_input_norm, d.eps = _code(who, x), layer, with_in, eps
        d.x, d.f = _p(xr), _p(fr)
        d.out_weight, d.out_bias, d.gate, d.residual_scale = _p(ow), _p(ob), _p(gt), _p(rt)
        d.in_weight, d.in_bias, d.scale, d.shift = _p(iw), _p(ib), _p(sc), _p(sh)
        with _on(x):
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if f is not None else None
            h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if with_in else None
            stats = torch.empty(4, max(B * rows, 1), dtype=torch.float32, device=x.device) if grads else None
            d.y, d.h, d.stats = _p(y), _p(h), _p(stats)
            if x.numel():
                _lib.check(_lib.lib().gc_block_norm_fwd(ctypes.byref(d), _stream()), "gc_block_norm_fwd")
        if grads:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x, f, *given)
            ctx.stats, ctx.desc, ctx.kept, ctx.who = stats, d, (xr, fr, ow, ob, gt, rt, iw, ib, sc, sh), who
        return (y, h) if (f is not None and with_in) else (y if f is not None else h)

    @staticmethod
    def backward(ctx, *gs):
        _OnceOnly.refuse_second_order(ctx.who, *gs)
        x, f, *given = ctx.saved_tensors               # (raises if one of them was written since)
        d = _lib.BlockNorm.from_buffer_copy(ctx.desc)
        dy, dh = (gs if len(gs) == 2 else ((gs[0], None) if f is not None else (None, gs[0])))
        if dy is None and dh is None:
            return (None,) * 11
        need = ctx.needs_input_grad
        with _on(x):
            seeds = [None if g is None else g.to(x.dtype).contiguous() for g in (dy, dh)]
            d.dy, d.dh = _p(seeds[0]), _p(seeds[1])
            empty = x.numel() == 0
            make = torch.zeros if empty else torch.empty
            dx = make(x.shape, dtype=x.dtype, device=x.device)
            df = make(x.shape, dtype=x.dtype, device=x.device) if f is not None else None
            d.dx, d.df = _p(dx), _p(df)
            outs = [make(t.shape, dtype=torch.float32, device=x.device) if (t is not None and n) else None for t, n in zip(given, need[3:])]
            d.d_out_weight, d.d_out_bias, d.d_gate, d.d_residual_scale, d.d_in_weight, d.d_in_bias, d.d_scale, d.d_shift = (_p(t) for t in outs)
            d.stats = _p(ctx.stats)
            if not empty:
                L = _lib.lib()
                n = L.gc_block_norm_workspace_bytes(d.batch, d.rows, d.cols)
                ws = torch.empty(n, dtype=torch.uint8, device=x.device)
                _lib.check(L.gc_block_norm_bwd(ctypes.byref(d), ws.data_ptr(), n, _stream()), "gc_block_norm_bwd")
            outs = [t if t is None or t.dtype == g.dtype else t.to(g.dtype) for t, g in zip(outs, given)]
        return (None, dx, df, *outs)


def block_norm(who, x, f, out_weight, out_bias, gate, residual_scale, in_weight, in_bias, scale, shift, kind, eps, with_input_norm):
    _require(kind in _KINDS, f"{who}: kind must be one of {list(_KINDS)}, got {kind!r}")
    _require(x.dim() >= 2 and x.shape[-1] > 0, f"{who}: x must be [B, ..., C], got {tuple(x.shape)}")
    _code(who, x)
    _require(f is None or (f.shape == x.shape and f.dtype == x.dtype),
             f"{who}: f must have x's shape and dtype (got {None if f is None else (tuple(f.shape), f.dtype)} and {tuple(x.shape)}, {x.dtype})")
    _require(x.shape[-1] <= 8192, f"{who}: at most 8192 channels are supported, got {x.shape[-1]}")
    eps = float(eps)
    _require(eps > 0.0, f"{who}: eps must be positive")
    rho, constant = (residual_scale, 1.0) if torch.is_tensor(residual_scale) else (None, float(residual_scale))
    _same_gpu(who, x, f, out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift)
    tensors = (x, f, out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift)
    return _BlockNorm.apply((who, _KINDS[kind], eps, int(with_input_norm), constant, _graph_follows(*tensors)), *tensors)


# ---- rotary positions with several axes ------------------------------------------------------------------------------------
class RotaryTable:
    """Frequencies of a rotary layer: per pair of elements the turns (2 pi radians) per unit of position and the axis it belongs
    to, on the device.  Made once by functional.rotary_table."""

    def __init__(self, turns, axis, axes, interleaved):
        self.turns, self.axis, self.axes, self.interleaved = turns, axis, axes, interleaved

    @property
    def pairs(self):
        return self.turns.numel()

    def to(self, device):
        return RotaryTable(self.turns.to(device), self.axis.to(device), self.axes, self.interleaved)


_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


def _heads(t):
    """t with contiguous heads (its other three strides are free)."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) else t.contiguous()


def _rotate(q, k, positions, table, inverse):
    q = _heads(q)
    k = _heads(k) if k is not None else None
    d = _lib.Rotary()
    B, N, d.q_heads, d.dim = q.shape
    d.batch, d.tokens, d.k_heads = B, N, (k.shape[2] if k is not None else 0)
    d.pairs, d.axes, d.halves, d.inverse = table.pairs, table.axes, int(not table.interleaved), inverse
    d.dtype, d.position_dtype, d.positions_per_sample = _code("axial_rotary", q), _POSITIONS[positions.dtype], int(positions.dim() == 3)
    d.q_stride[:] = _strides(q)[:3]
    if k is not None:
        d.k_stride[:] = _strides(k)[:3]
    with _on(q):
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
        if B and N:
            d.q, d.k, d.q_out, d.k_out = _p(q), _p(k), _p(qo), _p(ko)
            d.positions, d.pair_turns, d.pair_axis = _p(positions), _p(table.turns), _p(table.axis)
            _lib.check(_lib.lib().gc_axial_rotary(ctypes.byref(d), _stream()), "gc_axial_rotary")
    return qo, ko


class _AxialRotary(_OnceOnly):
    @staticmethod
    def forward(ctx, q, k, positions, table):
        ctx.save_for_backward(positions)
        ctx.table, ctx.set = table, ctx.set_materialize_grads(False)
        ctx.shapes = (q.shape, None if k is None else k.shape, q.dtype, q.device)
        qo, ko = _rotate(q, k, positions, table, 0)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, *gs):
        _OnceOnly.refuse_second_order("axial_rotary", *gs)
        (positions,) = ctx.saved_tensors
        gq, gk = gs[0], (gs[1] if len(gs) == 2 else None)
        dtype = ctx.shapes[2]
        gq, gk = (None if g is None else g.to(dtype) for g in (gq, gk))
        if gq is None and gk is None:
            return None, None, None, None
        if gq is None:                                  # a rotation's adjoint does not ask which of the two it turns
            return None, _rotate(gk, None, positions, ctx.table, 1)[0], None, None
        dq, dk = _rotate(gq, gk, positions, ctx.table, 1)
        return dq, dk, None, None


def axial_rotary(q, k, positions, table):
    who = "axial_rotary"
    _require(isinstance(table, RotaryTable), f"{who}: table must come from functional.rotary_table")
    _require(q.dim() == 4, f"{who}: q must be [B, N, heads, dim], got {tuple(q.shape)}")
    _code(who, q)
    B, N, _, D = q.shape
    _require(q.shape[2] > 0, f"{who}: q has no heads")
    _require(2 * table.pairs <= D, f"{who}: the table turns {2 * table.pairs} elements, heads have {D}")
    if k is not None:
        _require(k.dim() == 4 and k.shape[:2] == q.shape[:2] and k.shape[3] == D and k.shape[2] > 0 and k.dtype == q.dtype,
                 f"{who}: k must be [{B}, {N}, heads, {D}] in q's dtype, got {tuple(k.shape)}, {k.dtype}")
    _require(positions.dtype in _POSITIONS, f"{who}: positions must be int32, int64, float32 or float64, got {positions.dtype}")
    _require(tuple(positions.shape) in ((N, table.axes), (B, N, table.axes)),
             f"{who}: positions must be [{N}, {table.axes}] or [{B}, {N}, {table.axes}], got {tuple(positions.shape)}")
    _same_gpu(who, q, k, positions, table.turns)
    positions = positions.detach().contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _AxialRotary.apply(q, k, positions, table)
    qo, ko = _rotate(q, k, positions, table, 0)
    return qo if k is None else (qo, ko)


def rotary_table(dims, base=10000.0, interleaved=True, device=None):
    dims = (dims,) if isinstance(dims, int) else tuple(int(n) for n in dims)
    bases = (float(base),) * len(dims) if isinstance(base, (int, float)) else tuple(float(b) for b in base)
    _require(len(dims) > 0 and all(n > 0 and n % 2 == 0 for n in dims), f"rotary_table: dims must be positive even numbers, got {dims}")
    _require(len(bases) == len(dims) and all(b > 0 for b in bases), "rotary_table: base must be a positive number or one per axis")
    _require(sum(dims) <= 512, f"rotary_table: at most 512 rotated elements are supported, got {sum(dims)}")
    turns = torch.cat([torch.tensor(b, dtype=torch.float64) ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n, b in zip(dims, bases)])
    axis = torch.cat([torch.full((n // 2,), i, dtype=torch.int32) for i, n in enumerate(dims)])
    return RotaryTable((turns / (2.0 * torch.pi)).to(device), axis.to(device), len(dims), bool(interleaved))


# ---- differential attention ------------------------------------------------------------------------------------------------
def _aligned(t, width):
    """t as the kernels take it: contiguous heads, strides that are multiples of 8 elements, 16-byte aligned, rows apart."""
    st = _strides(t)
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and width <= st[1] < (1 << 23) and all(s % 8 == 0 and s >= 0 for s in st[:-1]):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _attention_desc(q, k, v, lam, lengths, causal, scale):
    d = _lib.DiffAttention()
    d.B, d.NQ, d.H, _, d.d = q.shape
    d.NK, d.HK, d.dv = v.shape[1:]
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = _strides(q)[:4], _strides(k)[:4], _strides(v)[:3]
    d.causal, d.scale = causal, scale
    d.q, d.k, d.v, d.lam, d.key_lengths = _p(q), _p(k), _p(v), _p(lam), _p(lengths)
    return d


class _DiffAttention(_OnceOnly):
    @staticmethod
    def forward(ctx, q, k, v, lam, lengths, causal, scale, grads):
        B, NQ, H, _, dk = q.shape
        NK, dv = v.shape[1], v.shape[3]
        qa, ka, va = _aligned(q, dk), _aligned(k, dk), _aligned(v, dv)
        la = lam.detach().float().contiguous()
        with _on(q):
            make = torch.zeros if NK == 0 else torch.empty
            out = make(B, NQ, H, dv, dtype=q.dtype, device=q.device)
            out2 = torch.empty_like(out) if grads else None
            lse = torch.empty(B, H, 2, NQ, dtype=torch.float32, device=q.device) if grads else None
            if out.numel() and NK:
                d = _attention_desc(qa, ka, va, la, lengths, causal, scale)
                d.out, d.out2, d.lse = _p(out), _p(out2), _p(lse)
                L = _lib.lib()
                n = L.gc_diff_attention_workspace_bytes(ctypes.byref(d), 0)
                ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
                _lib.check(L.gc_diff_attention_fwd(ctypes.byref(d), _p(ws), n, _stream()), "gc_diff_attention_fwd")
        if grads:
            ctx.save_for_backward(q, k, v, lam, lengths, out)
            ctx.kept, ctx.cfg = (qa, ka, va, la, out2, lse), (causal, scale)
        return out

    @staticmethod
    def backward(ctx, g):
        _OnceOnly.refuse_second_order("differential_attention", g)
        q, k, v, lam, lengths, out = ctx.saved_tensors
        qa, ka, va, la, out2, lse = ctx.kept
        with _on(q):
            if not (out.numel() and k.shape[1]):
                return tuple(torch.zeros_like(t) for t in (q, k, v, lam)) + (None,) * 4
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
            dlam = torch.empty(lam.shape, dtype=torch.float32, device=q.device)
            g = g.to(q.dtype).contiguous()
            if g.data_ptr() % 16:
                g = g.clone()
            d = _attention_desc(qa, ka, va, la, lengths, *ctx.cfg)
            d.out, d.out2, d.lse, d.dout = _p(out), _p(out2), _p(lse), _p(g)
            d.dq, d.dk, d.dv_out, d.dlam = _p(dq), _p(dk), _p(dv), _p(dlam)
            L = _lib.lib()
            n = L.gc_diff_attention_workspace_bytes(ctypes.byref(d), 1)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            _lib.check(L.gc_diff_attention_bwd(ctypes.byref(d), ws.data_ptr(), n, _stream()), "gc_diff_attention_bwd")
            return dq, dk, dv, dlam.to(lam.dtype), None, None, None, None


def differential_attention(q, k, v, lam, scale=None, causal=False, key_lengths=None):
    who = "differential_attention"
    _require(q.dim() == 5 and k.dim() == 5 and v.dim() == 4 and q.shape[3] == 2 and k.shape[3] == 2,
             f"{who} takes q [B, NQ, H, 2, d], k [B, NK, HK, 2, d] and v [B, NK, HK, dv] (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    B, NQ, H, _, d = q.shape
    NK, HK, dv = v.shape[1:]
    _require(tuple(k.shape) == (B, NK, HK, 2, d) and v.shape[0] == B and HK > 0 and H > 0 and H % HK == 0,
             f"{who}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together (heads of q: a multiple of those of k and v)")
    _require(0 < d <= 128 and d % 8 == 0 and 0 < dv <= 256 and dv % 8 == 0,
             f"{who}: d must be a multiple of 8 up to 128 and dv one up to 256 (got d={d}, dv={dv})")
    _require(torch.is_tensor(lam) and tuple(lam.shape) == (H,) and lam.dtype in (torch.float32, torch.bfloat16),
             f"{who}: lam must be a float32 or bfloat16 tensor [{H}]")
    for t in (q, k, v):
        _require(t.dtype == torch.bfloat16, f"{who}: operands are bf16, got {t.dtype}")
    scale = float(d ** -0.5 if scale is None else scale)
    _require(0.0 < scale < 1e30, f"{who}: scale must be positive and finite, got {scale}")
    if key_lengths is not None:
        _require(tuple(key_lengths.shape) == (B,) and key_lengths.dtype in (torch.int32, torch.int64), f"{who}: key_lengths must be int32 or int64 [{B}]")
    _same_gpu(who, q, k, v, lam, key_lengths)
    if key_lengths is not None:
        key_lengths = key_lengths.to(torch.int32).contiguous()
    return _DiffAttention.apply(q, k, v, lam, key_lengths, int(bool(causal)), scale, _graph_follows(q, k, v, lam))
