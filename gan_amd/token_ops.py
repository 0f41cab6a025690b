"""Operators of image / video transformer blocks over libganconv.so: the norms before and after a block, rotary positions with
several axes, differential attention.  Extensions beside the reference's one attention block (BigGAN/model.py:80-105); tokens lie
in rows, an image [B, C, H, W] in channels-last memory being [B, H * W, C].

Unlike the convolutions these are plain autograd functions, not torch.library operators, and their descriptors are packed in one go:
a call on a single token is host time and little else (a norm 35 -> 18 us, one query of attention 34 -> 19 us).  First-order
gradients only.  There is no fallback: on a CPU tensor or an unsupported geometry they raise RuntimeError.
"""
import contextlib
import struct

import torch

from . import _lib

_NO_CONTEXT = contextlib.nullcontext()

# the descriptors of include/ganconv.h, field by field (no padding: every group starts aligned)
_NORM = struct.Struct("2q4i2f4i4q25Q")          # gc_block_norm
_ROTARY = struct.Struct("2q10i6q7Q")            # gc_rotary
_ATTENTION = struct.Struct("11q8ifi13Q")        # gc_diff_attention


def _on(t):
    """Context that makes t's device the current one (launches, streams and allocations follow it)."""
    return _NO_CONTEXT if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _refuse(msg):
    raise RuntimeError("ganconv: " + msg)


def _same_gpu(who, first, *rest):
    d = first.get_device()
    if d < 0:
        _refuse(f"{who}: tensors must live on the GPU (this library has no CPU path)")
    for t in rest:
        if t is not None and t.get_device() != d:
            _refuse(f"{who}: all tensors must be on one device (got {first.device} and {t.device})")


def _code(who, t):
    if t.dtype == torch.bfloat16:
        return _lib.GC_BF16
    if t.dtype != torch.float32:
        _refuse(f"{who}: unsupported dtype {t.dtype} (float32 or bfloat16)")
    return _lib.GC_F32


def _p(t):
    return 0 if t is None else t.data_ptr()


def _graph_follows(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_second_order(who, *grads):
    if torch.is_grad_enabled() and any(g is not None and g.requires_grad for g in grads):
        _refuse(f"{who} has no second-order backward")


def _strides(t):
    """t's strides, with those of dimensions of one element (where torch allows anything) as in a contiguous tensor."""
    out, step = [], 1
    for n, st in zip(reversed(t.shape), reversed(t.stride())):
        out.append(st if n != 1 else step)
        step *= n
    return out[::-1]


def _grad_buffers(tensors, wanted, device, zero=False):
    """fp32 gradients of the wanted small parameters, as parts of one allocation."""
    sizes = [t.numel() if (t is not None and w) else 0 for t, w in zip(tensors, wanted)]
    buf = (torch.zeros if zero else torch.empty)(sum(sizes), dtype=torch.float32, device=device)
    return [(part if t.dim() == 1 else part.view(t.shape)) if n else None for t, n, part in zip(tensors, sizes, buf.split(sizes))]


# ---- norms before and after a block ----------------------------------------------------------------------------------------
def _rows(t, shared=False):
    """(tensor, batch stride, row stride) of [B, ..., C] read as [B, rows, C] with contiguous channels; copied if its rows do not
    lie at one stride (or overlap).  A [B, C] tensor is B samples of one row, or with `shared` one sample of B rows."""
    if t.dim() == 2:
        t = t.unsqueeze(0 if shared else 1)
    if t.is_contiguous():
        B, C = t.size(0), t.size(-1)
        return t, (t.numel() // B if B else 0), C
    st = _strides(t)
    ok = st[-1] == 1 and st[-2] >= t.shape[-1]
    for i in range(1, t.dim() - 2):
        ok = ok and st[i] == st[i + 1] * t.shape[i + 1]
    return (t, st[0], st[-2]) if ok else _rows(t.contiguous())


def _fp32(t):
    return t if (t.dtype == torch.float32 and t.is_contiguous()) else t.detach().to(torch.float32).contiguous()


def _param(who, name, t, C, B=None):
    """fp32 contiguous copy-or-self of a [C] (or, with B, [B, C]) parameter and whether it is per sample."""
    if t is None:
        return None, 0
    per_sample = B is not None and t.dim() == 2
    if t.numel() != (B * C if per_sample else C) or t.dim() != (2 if per_sample else 1) or t.size(-1) != C:
        _refuse(f"{who}: {name} must be [{C}]" + (f" or [{B}, {C}]" if B is not None else "") + f", got {tuple(t.shape)}")
    if t.dtype != torch.float32 and t.dtype != torch.bfloat16:
        _refuse(f"{who}: {name} must be float32 or bfloat16, got {t.dtype}")
    return _fp32(t), int(per_sample)


_KINDS = {"rms": 0, "layer": 1}


def _copies(given, used):
    """What a backward pass keeps of the tensors that a descriptor points to: the copies that were made of them.  Those that are the
    given tensors themselves are saved by autograd and may lie elsewhere when it hands them back (offloaded, gathered anew)."""
    return [u if (u is not None and u.data_ptr() != t.data_ptr()) else (t if t is None else t.stride()) for t, u in zip(given, used)]


def _moved(given, copies, pointers):
    """Whether a tensor that the descriptor points to directly lies elsewhere or otherwise by now"""
    for t, c, p in zip(given, copies, pointers):
        if type(c) is tuple and (t.data_ptr() != p or t.stride() != c):
            return True
    return False


def _norm_layout(cfg, x, f, out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift):
    """(the descriptor's fields up to the outputs, the tensors that they point to)"""
    who, layer, eps, with_in, constant = cfg
    B, C = x.size(0), x.size(-1)
    ow, _ = _param(who, "out_weight", out_weight, C)
    ob, _ = _param(who, "out_bias", out_bias, C)
    gt, gate_per = _param(who, "gate", gate, C, B)
    iw, _ = _param(who, "in_weight", in_weight, C)
    ib, _ = _param(who, "in_bias", in_bias, C)
    sc, ps = _param(who, "scale", scale, C, B)
    sh, qs = _param(who, "shift", shift, C, B)
    if sc is not None and sh is not None and ps != qs:
        _refuse(f"{who}: scale and shift must both be [C] or both [B, C]")
    mod_per, rt, per_channel = ps or qs, None, 0
    if rho is not None:
        n = rho.numel()
        if n not in (1, C) or rho.dim() > 1:
            _refuse(f"{who}: residual_scale must be a number, one element or [{C}], got {tuple(rho.shape)}")
        per_channel, rt = int(n == C and C > 1), _fp32(rho)
    shared = not (gate_per or mod_per)                  # nothing tells the samples apart: one run of rows where they lie so
    xr, xb, xs = _rows(x, shared)
    fr, fb, fs = _rows(f, shared) if f is not None else (None, 0, 0)
    rows = x.numel() // (B * C) if B else 0
    batch, per = B, rows
    if shared and (x.dim() == 2 or (xb == rows * xs and (fr is None or fb == rows * fs))):
        batch, per = 1, B * rows
    head = (batch, per, C, _code(who, x), layer, with_in, eps, constant, gate_per, mod_per, per_channel, 0, xb, xs, fb, fs, xr.data_ptr(), _p(fr),
            _p(ow), _p(ob), _p(gt), _p(rt), _p(iw), _p(ib), _p(sc), _p(sh))
    return head, (xr, fr, ow, ob, gt, rt, iw, ib, sc, sh)


def _norm_forward(cfg, tensors, stats_wanted):
    """(y or None, h or None, statistics or None, descriptor fields, the tensors they point to)"""
    x = tensors[0]
    with _on(x):
        head, used = _norm_layout(cfg, *tensors)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if tensors[1] is not None else None
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if cfg[3] else None
        stats = torch.empty(4 * (x.numel() // x.size(-1)), dtype=torch.float32, device=x.device) if stats_wanted else None
        if x.numel():
            rc = _lib.lib().gc_block_norm_fwd(_NORM.pack(*head, _p(y), _p(h), _p(stats), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), _stream(x))
            if rc:
                _lib.check(rc, "gc_block_norm_fwd")
    return y, h, stats, head, used


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, *tensors):
        y, h, ctx.stats, ctx.head, used = _norm_forward(cfg, tensors, True)
        ctx.copies = _copies(tensors, used)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*tensors)
        ctx.cfg = cfg
        return (y, h) if (y is not None and h is not None) else (y if y is not None else h)

    @staticmethod
    def backward(ctx, *gs):
        _no_second_order(ctx.cfg[0], *gs)
        tensors = ctx.saved_tensors                    # (raises if one of them was written since)
        x, f, *given = tensors
        head, stats, used = ctx.head, ctx.stats, None
        dy, dh = (gs if len(gs) == 2 else ((gs[0], None) if f is not None else (None, gs[0])))
        if dy is None and dh is None:
            return (None,) * 11
        dev, empty = x.device, x.numel() == 0
        with _on(x):
            if _moved(tensors, ctx.copies, head[16:]):
                head, used = _norm_layout(ctx.cfg, *tensors)
            dy, dh = (None if g is None else (g if g.dtype == x.dtype else g.to(x.dtype)).contiguous() for g in (dy, dh))
            make = torch.zeros if empty else torch.empty
            dx = make(x.shape, dtype=x.dtype, device=dev)
            df = make(x.shape, dtype=x.dtype, device=dev) if f is not None else None
            outs = _grad_buffers(given, ctx.needs_input_grad[3:], dev, empty)
            if not empty:
                L = _lib.lib()
                n = L.gc_block_norm_workspace_bytes(head[0], head[1], head[2])
                ws = torch.empty(n, dtype=torch.uint8, device=dev)
                rc = L.gc_block_norm_bwd(_NORM.pack(*head, 0, 0, stats.data_ptr(), _p(dy), _p(dh), dx.data_ptr(), _p(df), *[_p(t) for t in outs]),
                                         ws.data_ptr(), n, _stream(x))
                if rc:
                    _lib.check(rc, "gc_block_norm_bwd")
            outs = [t if t is None or g.dtype == torch.float32 else t.to(g.dtype) for t, g in zip(outs, given)]
        return (None, dx, df, *outs)


def block_norm(who, x, f, out_weight, out_bias, gate, residual_scale, in_weight, in_bias, scale, shift, kind, eps, with_input_norm):
    if kind not in _KINDS:
        _refuse(f"{who}: kind must be one of {list(_KINDS)}, got {kind!r}")
    if x.dim() < 2 or x.size(-1) == 0:
        _refuse(f"{who}: x must be [B, ..., C], got {tuple(x.shape)}")
    _code(who, x)
    if f is not None and (f.shape != x.shape or f.dtype != x.dtype):
        _refuse(f"{who}: f must have x's shape and dtype (got {tuple(f.shape)}, {f.dtype} and {tuple(x.shape)}, {x.dtype})")
    if x.size(-1) > 8192:
        _refuse(f"{who}: at most 8192 channels are supported, got {x.size(-1)}")
    eps = float(eps)
    if not eps > 0.0:
        _refuse(f"{who}: eps must be positive")
    rho, constant = (residual_scale, 1.0) if torch.is_tensor(residual_scale) else (None, float(residual_scale))
    tensors = (x, f, out_weight, out_bias, gate, rho, in_weight, in_bias, scale, shift)
    _same_gpu(who, *tensors)
    cfg = (who, _KINDS[kind], eps, int(with_input_norm), constant)
    if _graph_follows(*tensors):
        return _BlockNorm.apply(cfg, *tensors)
    y, h, *_ = _norm_forward(cfg, tensors, False)
    return (y, h) if (y is not None and h is not None) else (y if y is not None else h)


# ---- rotary positions with several axes ------------------------------------------------------------------------------------
class RotaryTable:
    """Frequencies of a rotary layer: per pair of elements the turns (2 pi radians) per unit of position and the axis it belongs
    to, on the device.  Made once by functional.rotary_table."""

    def __init__(self, turns, axis, axes, interleaved):
        self.turns, self.axis, self.axes, self.interleaved, self.pairs = turns, axis, axes, interleaved, turns.numel()

    def to(self, device):
        return RotaryTable(self.turns.to(device), self.axis.to(device), self.axes, self.interleaved)


_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


def _heads(t):
    """(t with contiguous heads, its three outer strides)"""
    if t.is_contiguous():
        _, N, H, D = t.shape
        return t, (N * H * D, H * D, D)
    if t.stride(-1) != 1 and t.size(-1) != 1:
        return _heads(t.contiguous())
    return t, tuple(_strides(t)[:3])


def _rotate(q, k, positions, table, inverse):
    q, qs = _heads(q)
    B, N, HQ, D = q.shape
    k, ks = _heads(k) if k is not None else (None, (0, 0, 0))
    with _on(q):
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
        if B and N:
            rc = _lib.lib().gc_axial_rotary(
                _ROTARY.pack(B, N, HQ, k.size(2) if k is not None else 0, D, table.pairs, table.axes, int(not table.interleaved), _code("axial_rotary", q),
                             _POSITIONS[positions.dtype], int(positions.dim() == 3), inverse, *qs, *ks, q.data_ptr(), _p(k), qo.data_ptr(), _p(ko),
                             positions.data_ptr(), table.turns.data_ptr(), table.axis.data_ptr()), _stream(q))
            if rc:
                _lib.check(rc, "gc_axial_rotary")
    return qo, ko


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table):
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        ctx.table, ctx.dtype = table, q.dtype
        qo, ko = _rotate(q, k, positions, table, 0)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, *gs):
        _no_second_order("axial_rotary", *gs)
        (positions,) = ctx.saved_tensors
        gq, gk = (None if g is None else (g if g.dtype == ctx.dtype else g.to(ctx.dtype)) for g in (gs[0], gs[1] if len(gs) == 2 else None))
        if gq is None and gk is None:
            return None, None, None, None
        if gq is None:                                  # a rotation's adjoint does not ask which of the two it turns
            return None, _rotate(gk, None, positions, ctx.table, 1)[0], None, None
        dq, dk = _rotate(gq, gk, positions, ctx.table, 1)
        return dq, dk, None, None


def axial_rotary(q, k, positions, table):
    who = "axial_rotary"
    if not isinstance(table, RotaryTable):
        _refuse(f"{who}: table must come from functional.rotary_table")
    if q.dim() != 4:
        _refuse(f"{who}: q must be [B, N, heads, dim], got {tuple(q.shape)}")
    _code(who, q)
    B, N, HQ, D = q.shape
    if HQ == 0:
        _refuse(f"{who}: q has no heads")
    if 2 * table.pairs > D:
        _refuse(f"{who}: the table turns {2 * table.pairs} elements, heads have {D}")
    if k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.size(3) != D or k.size(2) == 0 or k.dtype != q.dtype):
        _refuse(f"{who}: k must be [{B}, {N}, heads, {D}] in q's dtype, got {tuple(k.shape)}, {k.dtype}")
    if positions.dtype not in _POSITIONS:
        _refuse(f"{who}: positions must be int32, int64, float32 or float64, got {positions.dtype}")
    if tuple(positions.shape) not in ((N, table.axes), (B, N, table.axes)):
        _refuse(f"{who}: positions must be [{N}, {table.axes}] or [{B}, {N}, {table.axes}], got {tuple(positions.shape)}")
    _same_gpu(who, q, k, positions, table.turns)
    if not positions.is_contiguous() or positions.requires_grad:
        positions = positions.detach().contiguous()
    if _graph_follows(q, k):
        return _AxialRotary.apply(q, k, positions, table)
    qo, ko = _rotate(q, k, positions, table, 0)
    return qo if k is None else (qo, ko)


def rotary_table(dims, base=10000.0, interleaved=True, device=None):
    dims = (dims,) if isinstance(dims, int) else tuple(int(n) for n in dims)
    bases = (float(base),) * len(dims) if isinstance(base, (int, float)) else tuple(float(b) for b in base)
    if not (len(dims) > 0 and all(n > 0 and n % 2 == 0 for n in dims)):
        _refuse(f"rotary_table: dims must be positive even numbers, got {dims}")
    if not (len(bases) == len(dims) and all(b > 0 for b in bases)):
        _refuse("rotary_table: base must be a positive number or one per axis")
    if sum(dims) > 512:
        _refuse(f"rotary_table: at most 512 rotated elements are supported, got {sum(dims)}")
    turns = torch.tensor([b ** (-2.0 * i / n) / (2.0 * torch.pi) for n, b in zip(dims, bases) for i in range(n // 2)], dtype=torch.float64, device=device)
    axis = torch.tensor([a for a, n in enumerate(dims) for _ in range(n // 2)], dtype=torch.int32, device=device)
    return RotaryTable(turns, axis, len(dims), bool(interleaved))


# ---- differential attention ------------------------------------------------------------------------------------------------
def _aligned(t, width):
    """(t as the kernels take it -- contiguous heads, strides that are multiples of 8 elements, 16-byte aligned, rows apart --, its
    strides but the last)"""
    if t.is_contiguous():
        st, step = [], 1
        for n in reversed(t.shape[1:]):
            step *= n
            st.append(step)
        st.reverse()
    else:
        st = _strides(t)
        if st.pop() != 1:
            return _aligned(t.contiguous(), width)
    if t.data_ptr() % 16:
        return _aligned(t.clone(memory_format=torch.contiguous_format), width)
    if not t.is_contiguous() and not (width <= st[1] < (1 << 23) and all(s % 8 == 0 and s >= 0 for s in st)):
        return _aligned(t.contiguous(), width)
    return t, st


def _attention_layout(q, k, v, lam, lengths, causal, scale):
    """(the descriptor's fields up to the outputs, the tensors that they point to)"""
    B, NQ, H, _, d = q.shape
    _, NK, HK, dv = v.shape
    (qa, qs), (ka, ks), (va, vs), la = _aligned(q, d), _aligned(k, d), _aligned(v, dv), _fp32(lam)
    head = (*qs, *ks, *vs, B, NQ, NK, H, HK, d, dv, causal, scale, 0, qa.data_ptr(), ka.data_ptr(), va.data_ptr(), la.data_ptr(), _p(lengths))
    return head, (qa, ka, va, la, lengths)


def _attention_forward(q, k, v, lam, lengths, causal, scale, grads):
    B, NQ, H = q.shape[:3]
    NK, dv = v.size(1), v.size(3)
    with _on(q):
        head, used = _attention_layout(q, k, v, lam, lengths, causal, scale)
        out = (torch.empty if NK else torch.zeros)(B, NQ, H, dv, dtype=q.dtype, device=q.device)
        out2 = torch.empty(out.shape, dtype=q.dtype, device=q.device) if grads else None
        lse = torch.empty(B, H, 2, NQ, dtype=torch.float32, device=q.device) if grads else None
        if NK and out.numel():
            L = _lib.lib()
            desc = _ATTENTION.pack(*head, out.data_ptr(), _p(out2), _p(lse), 0, 0, 0, 0, 0)
            n = L.gc_diff_attention_workspace_bytes(desc, 0)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
            rc = L.gc_diff_attention_fwd(desc, _p(ws), n, _stream(q))
            if rc:
                _lib.check(rc, "gc_diff_attention_fwd")
    return out, out2, lse, head, used


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, lengths, causal, scale):
        out, ctx.out2, ctx.lse, ctx.head, used = _attention_forward(q, k, v, lam, lengths, causal, scale, True)
        ctx.copies = _copies((q, k, v, lam, lengths), used)
        ctx.save_for_backward(q, k, v, lam, lengths, out)
        ctx.cfg = (causal, scale)
        return out

    @staticmethod
    def backward(ctx, g):
        _no_second_order("differential_attention", g)
        q, k, v, lam, lengths, out = ctx.saved_tensors
        head, out2, lse, used = ctx.head, ctx.out2, ctx.lse, None
        with _on(q):
            if not (out.numel() and k.size(1)):
                return tuple(torch.zeros_like(t) for t in (q, k, v, lam)) + (None,) * 3
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
            dlam = torch.empty(lam.shape, dtype=torch.float32, device=q.device)
            if _moved((q, k, v, lam, lengths), ctx.copies, head[21:]):
                head, used = _attention_layout(q, k, v, lam, lengths, *ctx.cfg)
            g, out = ((t if t.dtype == q.dtype else t.to(q.dtype)).contiguous() for t in (g, out))
            g, out = (t.clone() if t.data_ptr() % 16 else t for t in (g, out))
            L = _lib.lib()
            desc = _ATTENTION.pack(*head, out.data_ptr(), out2.data_ptr(), lse.data_ptr(), g.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                   dlam.data_ptr())
            n = L.gc_diff_attention_workspace_bytes(desc, 1)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            rc = L.gc_diff_attention_bwd(desc, ws.data_ptr(), n, _stream(q))
            if rc:
                _lib.check(rc, "gc_diff_attention_bwd")
            return dq, dk, dv, dlam if lam.dtype == torch.float32 else dlam.to(lam.dtype), None, None, None


def differential_attention(q, k, v, lam, scale=None, causal=False, key_lengths=None):
    who = "differential_attention"
    if q.dim() != 5 or k.dim() != 5 or v.dim() != 4 or q.size(3) != 2 or k.size(3) != 2:
        _refuse(f"{who} takes q [B, NQ, H, 2, d], k [B, NK, HK, 2, d] and v [B, NK, HK, dv] (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    B, NQ, H, _, d = q.shape
    _, NK, HK, dv = v.shape
    if tuple(k.shape) != (B, NK, HK, 2, d) or v.size(0) != B or HK == 0 or H == 0 or H % HK:
        _refuse(f"{who}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together (heads of q: a multiple of those of k and v)")
    if not (0 < d <= 128 and d % 8 == 0 and 0 < dv <= 256 and dv % 8 == 0):
        _refuse(f"{who}: d must be a multiple of 8 up to 128 and dv one up to 256 (got d={d}, dv={dv})")
    if not (torch.is_tensor(lam) and lam.dim() == 1 and lam.numel() == H and lam.dtype in (torch.float32, torch.bfloat16)):
        _refuse(f"{who}: lam must be a float32 or bfloat16 tensor [{H}]")
    for t in (q, k, v):
        if t.dtype != torch.bfloat16:
            _refuse(f"{who}: operands are bf16, got {t.dtype}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        _refuse(f"{who}: scale must be positive and finite (1e-30 to 1e30), got {scale}")
    if key_lengths is not None and (key_lengths.dim() != 1 or key_lengths.numel() != B or key_lengths.dtype not in (torch.int32, torch.int64)):
        _refuse(f"{who}: key_lengths must be int32 or int64 [{B}]")
    _same_gpu(who, q, k, v, lam, key_lengths)
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or not key_lengths.is_contiguous()):
        key_lengths = key_lengths.clamp(0, NK).to(torch.int32).contiguous()
    if _graph_follows(q, k, v, lam):
        return _DiffAttention.apply(q, k, v, lam, key_lengths, int(bool(causal)), scale)
    return _attention_forward(q, k, v, lam, key_lengths, int(bool(causal)), scale, False)[0]
