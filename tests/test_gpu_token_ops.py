"""The operators of image / video transformer blocks (gan_amd.functional: block norms, axial rotary positions, differential
attention) against their definitions evaluated in float64 on the same operands.

Bounds are elementwise and counted, not chosen: a stored bf16 value is off by at most half a step (2^-8 of its value), an fp32
one by 2^-24; where a kernel rounds an intermediate to bf16 (the probabilities and score gradients of the attention), 2^-8 of every
addend's magnitude is carried through the formula with absolute values.  Sums of n fp32 addends are off by at most their depth
times 2^-24 of the sum of magnitudes; DEPTH bounds every summation depth in the kernels."""
import contextlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DEPTH = 512 * 2.0 ** -24


@pytest.fixture(scope="module")
def F():
    import gan_amd
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return gan_amd.functional


def _check(name, got, want, slack, dtype=None):
    """|got - want| <= half a step of got's type * |want| + slack (elementwise)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    slack = slack.detach().double().cpu() if torch.is_tensor(slack) else slack
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bound = HALF[dtype] * want.abs() + slack
    over = (got - want).abs() - bound
    assert torch.isfinite(got).all(), name
    assert float(over.max() if over.numel() else -1.0) <= 0.0, (name, float((got - want).abs().max()), float(over.max()), float(want.abs().max()))


# ---- norms ---------------------------------------------------------------------------------------------------------------
def _norm_reference(x, f, p, kind, eps, dy, dh):
    """(outputs, gradients by name, sums of magnitudes by name) in float64 by the formulas."""
    B, C = x.shape[0], x.shape[-1]
    xs, fs = x.double().reshape(B, -1, C), (None if f is None else f.double().reshape(B, -1, C))
    q = {n: (None if t is None else t.double()) for n, t in p.items()}

    def rows(n, neutral):
        return torch.full((B, 1, C), neutral, dtype=torch.float64) if q.get(n) is None else q[n].expand(B, C)[:, None, :]

    def std(t):
        mu = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
        r = 1.0 / ((t - mu).square().mean(-1, keepdim=True) + eps).sqrt()
        return (t - mu) * r, r

    def back(g, th, r):
        out = g - th * (g * th).mean(-1, keepdim=True)
        return (out - g.mean(-1, keepdim=True) if kind == "layer" else out) * r

    wo, bo, wi, bi, gate, sc, sh = (rows(n, v) for n, v in (("out_weight", 1.0), ("out_bias", 0.0), ("in_weight", 1.0), ("in_bias", 0.0), ("gate", 1.0),
                                                            ("scale", 0.0), ("shift", 0.0)))
    rho = q["residual_scale"] if torch.is_tensor(q.get("residual_scale")) else torch.tensor(1.0, dtype=torch.float64)
    outs, mags = {}, {}
    if f is not None:
        fh, rf = std(fs)
        u = fh * wo + bo
        y = rho * xs + gate * u
        outs["y"] = y
        mags["y"] = (rho * xs).abs() + (gate * fh * wo).abs() + (gate * bo).abs() + (gate * wo).abs() * rf * fs.abs()
    else:
        y = xs
    yh, ry = std(y)
    n = yh * wi + bi
    outs["h"] = n * (1 + sc) + sh
    mags["h"] = ((1 + sc) * wi).abs() * (yh.abs() + ry * mags.get("y", xs.abs()) + 1.0) + bi.abs() * (1 + sc).abs() + sh.abs()
    grads, gm = {}, {}
    g = torch.zeros_like(y) if dy is None else dy.double().reshape(y.shape)
    gmag = g.abs()
    if dh is not None:
        dhd = dh.double().reshape(y.shape)
        dn = dhd * (1 + sc)
        g = g + back(dn * wi, yh, ry)
        gmag = gmag + ry * ((dn * wi).abs() + (yh.abs() + ry * y.abs()) * (dn * wi * yh).abs().mean(-1, keepdim=True) + (dn * wi).abs().mean(-1, keepdim=True))
        grads["in_weight"], gm["in_weight"] = (dn * yh).sum((0, 1)), (dn.abs() * (yh.abs() + ry * y.abs())).sum((0, 1))
        grads["in_bias"], gm["in_bias"] = dn.sum((0, 1)), dn.abs().sum((0, 1))
        grads["scale"], gm["scale"] = (dhd * n).sum(1), (dhd.abs() * (wi.abs() * (yh.abs() + ry * y.abs()) + bi.abs())).sum(1)
        grads["shift"], gm["shift"] = dhd.sum(1), dhd.abs().sum(1)
    if f is not None:
        du = g * gate
        mdu = gmag * gate.abs()
        grads["x"], gm["x"] = rho * g, rho.abs() * gmag
        grads["f"] = back(du * wo, fh, rf)
        mp = mdu * wo.abs()
        gm["f"] = rf * (mp + (fh.abs() + rf * fs.abs()) * (mp * (fh.abs() + rf * fs.abs())).mean(-1, keepdim=True) + mp.mean(-1, keepdim=True))
        mf = fh.abs() + rf * fs.abs()
        grads["out_weight"], gm["out_weight"] = (du * fh).sum((0, 1)), (mdu * mf).sum((0, 1))
        grads["out_bias"], gm["out_bias"] = du.sum((0, 1)), mdu.sum((0, 1))
        grads["gate"], gm["gate"] = (g * u).sum(1), (gmag * (mf * wo.abs() + bo.abs())).sum(1)
        rs, rm = (g * xs).sum((0, 1)), (gmag * xs.abs()).sum((0, 1))
        grads["residual_scale"], gm["residual_scale"] = rs, rm
    else:
        grads["x"], gm["x"] = g, gmag
    for nme in ("gate", "scale", "shift"):
        if nme in grads and (q.get(nme) is None or q[nme].dim() == 1):
            grads[nme], gm[nme] = grads[nme].sum(0), gm[nme].sum(0)
    if torch.is_tensor(q.get("residual_scale")) and q["residual_scale"].numel() == 1 and "residual_scale" in grads and C > 1:
        grads["residual_scale"], gm["residual_scale"] = grads["residual_scale"].sum().reshape(1), gm["residual_scale"].sum().reshape(1)
    return outs, mags, grads, gm


NORM_CASES = [
    # shape, part, kind, per sample, parameters left out, residual_scale
    ((1, 1, 512), "both", "rms", False, (), "one"),
    ((3, 37, 128), "both", "rms", False, (), "one"),
    ((2, 65, 387), "both", "layer", True, (), "one"),
    ((4, 5, 64), "both", "layer", False, ("gate", "in_weight"), "channel"),
    ((2, 9, 4096), "both", "rms", True, (), "number"),
    ((2, 3, 2049), "both", "layer", True, (), "one"),
    ((2, 3, 8192), "both", "layer", False, (), "channel"),
    ((5, 1, 1), "both", "rms", False, (), "one"),
    ((2, 7, 20), "out", "layer", True, ("out_weight",), "channel"),
    ((3, 300, 72), "out", "rms", False, (), "number"),
    ((2, 11, 1000), "out", "layer", False, (), "one"),
    ((2, 8, 4, 96), "in", "rms", False, (), "number"),
    ((3, 50, 640), "in", "layer", True, ("in_bias",), "number"),
    ((7, 33), "in", "layer", True, (), "number"),
    ((700, 16), "both", "rms", False, (), "one"),
    ((2, 4100, 32), "both", "rms", True, (), "one"),
]


def _norm_inputs(case, dt, seed=5):
    shape, part, kind, per_sample, left_out, rs = case
    g = torch.Generator().manual_seed(seed)
    C, B = shape[-1], shape[0]
    r = lambda *s, scale=1.0, off=0.0: torch.randn(*s, generator=g) * scale + off
    x = r(*shape).to(dt)
    f = None if part == "in" else (r(*shape, scale=2.0, off=0.3)).to(dt)
    p = {}
    if part != "in":
        p["out_weight"], p["gate"] = r(C, scale=0.3, off=1.0), r(*((B, C) if per_sample else (C,)), scale=0.5)
        if kind == "layer":
            p["out_bias"] = r(C, scale=0.3)
    if part != "out":
        p["in_weight"] = r(C, scale=0.3, off=1.0)
        if kind == "layer":
            p["in_bias"] = r(C, scale=0.3)
        if per_sample:
            p["scale"], p["shift"] = r(B, C, scale=0.3), r(B, C, scale=0.3)
    p["residual_scale"] = {"one": r(1, scale=0.1, off=0.8), "channel": r(C, scale=0.1, off=0.8), "number": None}[rs] if part != "in" else None
    for n in left_out:
        p[n] = None
    dy = None if part == "in" else r(*shape).to(dt)
    dh = None if part == "out" else r(*shape).to(dt)
    return x, f, p, dy, dh


def _norm_call(F, part, x, f, p, kind, eps):
    rs = p.get("residual_scale")
    rs = 1.0 if rs is None else rs
    if part == "in":
        return (F.block_input_norm(x, p.get("in_weight"), p.get("in_bias"), scale=p.get("scale"), shift=p.get("shift"), kind=kind, eps=eps),)
    if part == "out":
        return (F.block_output_norm(x, f, p.get("out_weight"), p.get("out_bias"), gate=p.get("gate"), residual_scale=rs, kind=kind, eps=eps),)
    return F.block_boundary_norm(x, f, p.get("out_weight"), p.get("in_weight"), p.get("out_bias"), p.get("in_bias"), gate=p.get("gate"),
                                 residual_scale=rs, scale=p.get("scale"), shift=p.get("shift"), kind=kind, eps=eps)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "x".join(map(str, c[0])) + "-" + c[1] + "-" + c[2])
def test_block_norm_against_the_formulas(F, case, dt):
    shape, part, kind = case[:3]
    x, f, p, dy, dh = _norm_inputs(case, dt)
    leaves = {"x": x.cuda().requires_grad_(True)}
    if f is not None:
        leaves["f"] = f.cuda().requires_grad_(True)
    for n, t in p.items():
        if t is not None:
            leaves[n] = t.cuda().requires_grad_(True)
    out = _norm_call(F, part, leaves["x"], leaves.get("f"), {n: leaves.get(n) for n in p}, kind, 1e-5)
    seeds = [t.cuda() for t in (dy, dh) if t is not None]
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), seeds)))
    outs, mags, want, gm = _norm_reference(x, f, p, kind, 1e-5, dy, dh)
    for n, t in zip([m for m in ("y", "h") if (m == "y") <= (part != "in") and (m == "h") <= (part != "out")], out):
        _check(n, t.reshape(outs[n].shape), outs[n], DEPTH * mags[n], dt)
    for n, t in grads.items():
        _check("d " + n, t.reshape(want[n].shape), want[n], DEPTH * gm[n], t.dtype)
    again = torch.autograd.grad(_norm_call(F, part, leaves["x"], leaves.get("f"), {n: leaves.get(n) for n in p}, kind, 1e-5), list(leaves.values()), seeds)
    assert all(torch.equal(a, b) for a, b in zip(again, grads.values()))        # fixed summation order
    with torch.no_grad():                                                         # without a graph: the same values
        plain = _norm_call(F, part, leaves["x"], leaves.get("f"), {n: leaves.get(n) for n in p}, kind, 1e-5)
    assert all(torch.equal(a, b) for a, b in zip(plain, out))


def test_block_norm_gradients_against_differences(F):
    """Directional derivatives of a scalar of (y, h), central differences in the kernels' own fp32 arithmetic: the second-order
    remainder and the fp32 rounding of the two values (each about 2^-24 * |loss| / step) bound the difference by a few 1e-3."""
    g = torch.Generator().manual_seed(3)
    x, f, p, dy, dh = _norm_inputs(((2, 17, 96), "both", "layer", True, (), "one"), torch.float32)
    t = {"x": x.cuda(), "f": f.cuda(), **{n: v.cuda() for n, v in p.items()}}
    dy, dh = dy.cuda(), dh.cuda()

    def loss(v):
        y, h = _norm_call(F, "both", v["x"], v["f"], v, "layer", 1e-5)
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    leaves = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    y, h = _norm_call(F, "both", leaves["x"], leaves["f"], leaves, "layer", 1e-5)
    grads = dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (dy, dh))))
    for n in t:
        u = torch.randn(t[n].shape, generator=g).cuda()
        e = 2.0 ** -8
        up, down = dict(t), dict(t)
        up[n], down[n] = t[n] + e * u, t[n] - e * u
        with torch.no_grad():
            diff = float(loss(up) - loss(down)) / (2 * e)
        along = float((grads[n].double() * u.double()).sum())
        size = float((grads[n].double().norm() * u.double().norm()))
        assert abs(diff - along) < 4e-3 * size, (n, diff, along, size)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_block_norm_of_strided_and_shifted_tensors(F, dt):
    """Slices of wider tensors, a channels-last image, an odd offset, a transposed view: the definition on the view's values (an odd
    offset or stride takes narrower accesses and another order of the sums, which the counted bound covers)."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(3, 10, 200, generator=g).to(dt).cuda()
    w = torch.randn(64, generator=g).cuda()
    for view in (wide[:, 2:9, 64:128], wide[..., 3:67], wide[:, ::2, :64], wide[1:2].expand(3, 10, 200)[..., :64], wide.transpose(0, 1)[..., 64:128]):
        a = F.block_input_norm(view, w, kind="layer", eps=1e-5)
        outs, mags, _, _ = _norm_reference(view.cpu(), None, {"in_weight": w.cpu()}, "layer", 1e-5, None, view.cpu())
        assert a.is_contiguous()
        _check("h", a, outs["h"], DEPTH * mags["h"], dt)
        y = F.block_output_norm(view, view.flip(0), w, gate=w, eps=1e-5)
        outs, mags, _, _ = _norm_reference(view.cpu(), view.flip(0).cpu(), {"out_weight": w.cpu(), "gate": w.cpu()}, "rms", 1e-5, view.cpu(), None)
        _check("y", y, outs["y"], DEPTH * mags["y"], dt)
    same = wide[:, 2:9, 64:128]                                                  # the same accesses: the same bits
    assert torch.equal(F.block_input_norm(same, w), F.block_input_norm(same.contiguous(), w))
    img = torch.randn(2, 64, 6, 5, generator=g).to(dt).cuda().contiguous(memory_format=torch.channels_last)
    t = F.block_input_norm(img.permute(0, 2, 3, 1), w)
    assert t.permute(0, 3, 1, 2).is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(t, F.block_input_norm(img.permute(0, 2, 3, 1).contiguous(), w))


def test_block_norm_empty_rows_and_zero_rows(F):
    w = torch.ones(32, device="cuda", requires_grad=True)
    for shape in ((0, 4, 32), (3, 0, 32)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        h = F.block_input_norm(x, w)
        gx, gw = torch.autograd.grad(h.sum(), (x, w))
        assert h.shape == shape and gx.shape == shape and float(gw.abs().sum()) == 0.0
    x = torch.zeros(2, 3, 32, device="cuda", requires_grad=True)            # a row of zeros: eps alone under the root
    h = F.block_input_norm(x, w, kind="layer", eps=1e-6)
    (gx,) = torch.autograd.grad(h, x, torch.ones_like(h))
    assert float(h.abs().max()) == 0.0 and torch.isfinite(gx).all()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(150000, 16), (150000, 40), (20000, 256), (20002, 387), (9000, 1040), (5000, 4096)])
@pytest.mark.parametrize("part", ["in", "out", "both"])
def test_block_norm_of_many_rows_equals_a_few_alone(F, part, rows, C, dt, kind):
    """A workgroup walks many rows, asking for the next while it works on one: a row's outputs and gradients have to be those of a
    call on a few rows (the same kernel and the same order of sums), and the parameters' gradients the sum over three parts of the rows.
    Those are sums of n terms of size one: runs of m <= 1000 rows whose partial sums stay below 4 sqrt(m), each step off by half a unit
    of that with either sign, n / m of them: 4 x 2^-24 x sqrt(m n) < 128 x 2^-24 sqrt(n), and four times that for products of two or
    three normal factors."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, f = r(1, rows, C).to(dt).requires_grad_(True), r(1, rows, C).to(dt).requires_grad_(True)
    ow, gate, iw = (r(C).requires_grad_(True) for _ in range(3))
    dy, dh = r(1, rows, C).to(dt), r(1, rows, C).to(dt)

    def call(lo, hi):
        a, b = x[:, lo:hi], f[:, lo:hi]
        if part == "in":
            outs, seeds, leaves = (F.block_input_norm(a, iw, kind=kind),), (dh[:, lo:hi],), (x, iw)
        elif part == "out":
            outs, seeds, leaves = (F.block_output_norm(a, b, ow, gate=gate, kind=kind),), (dy[:, lo:hi],), (x, f, ow, gate)
        else:
            outs, seeds, leaves = F.block_boundary_norm(a, b, ow, iw, gate=gate, kind=kind), (dy[:, lo:hi], dh[:, lo:hi]), (x, f, ow, gate, iw)
        grads = torch.autograd.grad(outs, leaves, seeds)
        rowwise = [t.detach() for t in outs] + [t[:, lo:hi] for t in grads if t.dim() == 3]
        return rowwise, [t for t in grads if t.dim() == 1]

    whole, params = call(0, rows)
    step = 8 * ((rows // 3) // 8)
    sums = None
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        some, ps = call(lo, hi)
        sums = [p.double() for p in ps] if sums is None else [a + p.double() for a, p in zip(sums, ps)]
    for p, q in zip(params, sums):
        assert float((p.double() - q).abs().max()) <= 4 * 128 * 2.0 ** -24 * rows ** 0.5
    for lo in (0, 8 * (rows // 16), 8 * ((rows - 17) // 8)):
        few, _ = call(lo, min(rows, lo + 16))
        for n, (a, b) in enumerate(zip(whole, few)):
            assert torch.equal(a[:, lo:lo + 16], b), (n, lo)


# ---- rotary --------------------------------------------------------------------------------------------------------------
def _rotary_reference(t, positions, dims, bases, interleaved, sign):
    w = torch.cat([torch.tensor(b, dtype=torch.float64) ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n, b in zip(dims, bases)])
    axis = torch.cat([torch.full((n // 2,), i) for i, n in enumerate(dims)])
    ang = sign * positions.double()[..., axis] * w
    z = torch.polar(torch.ones_like(ang), ang)
    z = (z if z.dim() == 3 else z[None])[:, :, None]
    P = len(w)
    td = t.double()
    a, b = (td[..., 0:2 * P:2], td[..., 1:2 * P:2]) if interleaved else (td[..., :P], td[..., P:2 * P])
    r = torch.complex(a, b) * z
    head = torch.stack((r.real, r.imag), dim=-1).flatten(-2) if interleaved else torch.cat((r.real, r.imag), dim=-1)
    return torch.cat((head, td[..., 2 * P:]), dim=-1), torch.cat((torch.complex(a, b).abs().repeat_interleave(2, -1) if interleaved else
                                                                  torch.complex(a, b).abs().repeat(1, 1, 1, 2), 0 * td[..., 2 * P:]), dim=-1)


ROTARY_CASES = [
    # B, N, HQ, HK, dims, extra, positions dtype, per sample
    (1, 1, 1, 1, (2,), 0, torch.int64, False),
    (2, 65, 4, 2, (16, 16), 0, torch.int32, False),
    (3, 130, 2, 2, (16, 24, 24), 0, torch.int64, True),
    (2, 33, 8, 0, (32, 48, 48), 8, torch.float32, True),
    (1, 50, 3, 1, (6, 10), 3, torch.float64, False),
    (9, 17, 2, 1, (8, 12, 12), 0, torch.int64, False),
    (2, 40, 1, 1, (256, 256), 16, torch.int32, False),
]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", ROTARY_CASES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}+{c[3]}-{'_'.join(map(str, c[4]))}+{c[5]}")
def test_axial_rotary_against_complex_products(F, case, dt, interleaved):
    """Angle: turns formed in fp64, its fraction rounded to fp32 (2^-25 of a turn), sin and cos to a few units: 2^-20 of a pair's
    length covers both and the products."""
    B, N, HQ, HK, dims, extra, pdt, per = case
    g = torch.Generator().manual_seed(N)
    D = sum(dims) + extra
    q, k = torch.randn(B, N, HQ, D, generator=g).to(dt), (torch.randn(B, N, HK, D, generator=g).to(dt) if HK else None)
    shape = (B, N, len(dims)) if per else (N, len(dims))
    pos = torch.randint(-5, 1_000_000, shape, generator=g)
    pos = (pos.double() / 7).to(pdt) if pdt.is_floating_point else pos.to(pdt)
    bases = tuple(10000.0 / (1 + i) for i in range(len(dims)))
    table = F.rotary_table(dims, bases, interleaved, device="cuda")
    leaves = [q.cuda().requires_grad_(True)] + ([k.cuda().requires_grad_(True)] if HK else [])
    out = F.axial_rotary(leaves[0], leaves[1] if HK else None, pos.cuda(), table)
    out = out if HK else (out,)
    seeds = [torch.randn(t.shape, generator=g).to(dt) for t in out]
    grads = torch.autograd.grad(out, leaves, [s.cuda() for s in seeds])
    for src, got, seed, grad in zip((q, k), out, seeds, grads):
        want, size = _rotary_reference(src, pos, dims, bases, interleaved, 1.0)
        _check("out", got, want, 2.0 ** -20 * size, dt)
        want, size = _rotary_reference(seed, pos, dims, bases, interleaved, -1.0)
        _check("grad", grad, want, 2.0 ** -20 * size, dt)


def test_axial_rotary_strides_single_gradient_and_empty(F):
    g = torch.Generator().manual_seed(2)
    table = F.rotary_table((8, 8), device="cuda")
    pos = torch.randint(0, 50, (12, 2), generator=g).cuda()
    qkv = torch.randn(2, 12, 3, 4, 16, generator=g).cuda()
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    a, b = F.axial_rotary(q, k, pos, table)
    c, d = F.axial_rotary(q.contiguous(), k.contiguous(), pos, table)
    assert torch.equal(a, c) and torch.equal(b, d) and a.is_contiguous()
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    off = torch.randn(2 * 12 * 4 * 16 + 1, generator=g).cuda()[1:].view(2, 12, 4, 16)         # 4-byte aligned only
    assert torch.equal(F.axial_rotary(heads_first, None, pos, table), c)
    assert torch.equal(F.axial_rotary(off, None, pos, table), F.axial_rotary(off.clone(), None, pos, table))
    shared = q[:, :, :1].expand(2, 12, 4, 16).detach().requires_grad_(True)
    assert torch.equal(F.axial_rotary(shared, None, pos, table), F.axial_rotary(shared.detach().contiguous(), None, pos, table))
    kl = k.detach().clone().requires_grad_(True)
    _, kr = F.axial_rotary(q, kl, pos, table)                                                # only k is asked for
    (gk,) = torch.autograd.grad(kr, kl, torch.ones_like(kr))
    assert float((gk.double().norm() - torch.ones_like(kr).double().norm()).abs()) < 1e-3    # a rotation keeps lengths
    e, f_ = F.axial_rotary(q[:, :0], k[:, :0], pos[:0], table)
    assert e.shape == (2, 0, 4, 16) and f_.shape == (2, 0, 4, 16)


@pytest.mark.parametrize("extra", [0, 8, 3])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_axial_rotary_of_many_samples_equals_each_alone(F, dt, interleaved, extra):
    """Large batches with shared positions give a workgroup several samples: every sample has to come out as in a call of its own, its
    elements behind the turned pairs unchanged.  The last workgroup's run of samples is a short one."""
    B, N, D = 155, 1024, 16 + extra
    q = torch.randn(B, N, 1, D, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
    table = F.rotary_table((8, 8), interleaved=interleaved, device="cuda")
    pos = torch.arange(2 * N, device="cuda").view(N, 2)
    out = F.axial_rotary(q, None, pos, table)
    assert torch.equal(out[..., 16:], q[..., 16:])
    for b in (0, 1, 2, 3, 77, 151, 152, 153, 154):
        assert torch.equal(out[b:b + 1], F.axial_rotary(q[b:b + 1], None, pos, table)), b


# ---- differential attention ------------------------------------------------------------------------------------------------
def _attention_reference(q, k, v, lam, scale, causal, lengths, dout):
    """Output, gradients and their error bounds in float64.  u = 2^-8 * 1.06: a bf16 rounding of an intermediate, with room for the
    fp32 scores (|argument of exp| < 64 at a few 2^-24 of it)."""
    u = 2.0 ** -8 * 1.06
    B, NQ, H, _, d = q.shape
    NK, HK, dv = v.shape[1:]
    out, eo = torch.zeros(B, NQ, H, dv, dtype=torch.float64), torch.zeros(B, NQ, H, dv, dtype=torch.float64)
    gr = {n: torch.zeros(t.shape, dtype=torch.float64) for n, t in (("q", q), ("k", k), ("v", v), ("lam", lam))}
    er = {n: torch.zeros_like(t) for n, t in gr.items()}
    for b in range(B):
        n = NK if lengths is None else max(0, min(NK, int(lengths[b])))
        if n == 0:
            continue
        seen = torch.ones(NQ, n, dtype=torch.bool)
        if causal:
            seen = torch.arange(n)[None] <= torch.arange(NQ)[:, None] + (n - NQ)
        for h in range(H):
            c = h // (H // HK)
            l = float(lam[h].double())
            vv, go = v[b, :n, c].double(), dout[b, :, h].double()
            P, Q, K = [], [], []
            for m in range(2):
                Q.append(q[b, :, h, m].double())
                K.append(k[b, :n, c, m].double())
                s = (Q[m] @ K[m].t() * scale).masked_fill(~seen, float("-inf"))
                P.append(torch.nan_to_num(torch.softmax(s, -1)) * seen)
            O2 = P[1] @ vv
            o = P[0] @ vv - l * O2
            out[b, :, h] = o
            e1, e2 = u * (P[0] @ vv.abs()), u * (P[1] @ vv.abs())
            eo[b, :, h] = e1 + abs(l) * e2
            # delta from the STORED outputs: their own rounding on top
            E2 = (e2 + 2.0 ** -8 * O2.abs())
            E1 = (e1 + abs(l) * e2 + 2.0 ** -8 * o.abs()) + abs(l) * E2
            dP = go @ vv.t()
            delta = [(dP * P[m]).sum(-1, keepdim=True) for m in range(2)]
            Ed = [(go.abs() * E).sum(-1, keepdim=True) for E in (E1, E2)]
            mix = P[0] - l * P[1]
            gr["v"][b, :n, c] += mix.t() @ go
            er["v"][b, :n, c] += (u * mix.abs() + 2.0 ** -16 * (P[0] + abs(l) * P[1])).t() @ go.abs()
            size = go.abs() @ vv.abs().t()
            gr["lam"][h] -= delta[1].sum()
            er["lam"][h] += (P[1] * size).sum() * 2.0 ** -15
            for m, f in ((0, 1.0), (1, -l)):
                dS = P[m] * (dP - delta[m]) * f
                E = (P[m] * (Ed[m] + 2.0 ** -16 * (size + (P[m] * size).sum(-1, keepdim=True)))) * abs(f) + u * dS.abs()
                gr["q"][b, :, h, m] = scale * dS @ K[m]
                er["q"][b, :, h, m] = scale * E @ K[m].abs()
                gr["k"][b, :n, c, m] += scale * dS.t() @ Q[m]
                er["k"][b, :n, c, m] += scale * E.t() @ Q[m].abs()
    return out, eo, gr, er


ATTENTION_CASES = [
    # B, NQ, NK, H, HK, d, dv, causal, lengths, spread
    (1, 1, 1, 1, 1, 32, 64, False, None, 1.0),
    (2, 128, 128, 1, 1, 64, 128, False, None, 1.0),
    (2, 65, 130, 2, 1, 32, 64, False, (130, 77), 1.0),
    (4, 100, 100, 4, 2, 64, 128, True, (100, 0, 1, 63), 2.0),
    (2, 70, 33, 2, 2, 40, 80, True, None, 1.0),
    (2, 33, 257, 2, 1, 128, 256, True, (200, 257), 1.0),
    (1, 150, 90, 1, 1, 96, 200, False, None, 1.0),
    (2, 1, 4096, 4, 2, 64, 128, False, (4096, 1000), 1.0),
    (1, 7, 2050, 8, 2, 16, 64, True, None, 2.0),
    (2, 2, 1500, 2, 1, 128, 256, False, (0, 1500), 1.0),
    (1, 3, 600, 2, 1, 8, 8, False, None, 1.0),
    (1, 190, 190, 3, 1, 24, 48, True, None, 0.5),
    (1, 320, 320, 2, 2, 64, 128, True, None, 3.0),
    (1, 129, 129, 1, 1, 64, 64, True, (-3,), 1.0),
    (1, 8, 3000, 4, 1, 64, 128, True, (2990,), 1.0),
    (2, 4, 900, 2, 1, 32, 64, False, (900, 31), 1.0),
    (1, 40, 2100, 1, 1, 32, 64, True, None, 1.0),
    (1, 700, 700, 3, 1, 32, 64, True, None, 1.0),
    (1, 520, 300, 2, 1, 64, 128, False, None, 1.0),
    (1, 300, 520, 2, 2, 128, 256, False, (500,), 1.0),
    # a few shares of the keys for many rows (some of the shares without a visible key), and many shares for more rows than a short run
    (1, 600, 1100, 2, 1, 32, 64, True, (1000,), 1.0),
    (3, 260, 1030, 1, 1, 72, 136, False, (0, 1030, 70), 1.0),
    (1, 130, 2200, 2, 2, 64, 128, True, (40,), 1.0),
    (1, 40, 9000, 1, 1, 64, 128, True, None, 1.0),
    # few rows: the widest form, one workgroup per head (its waves' shares are all there is), a workgroup whose later waves see no key
    (1, 3, 400, 2, 1, 128, 256, False, None, 1.0),
    (70, 1, 300, 4, 4, 32, 64, False, None, 1.0),
    (64, 2, 260, 8, 4, 64, 128, True, None, 1.0),
    (2, 5, 700, 2, 1, 64, 128, True, (700, 33), 1.0),
    # grids of a quarter to one workgroup per CU in the backward pass: one share, several, shares without a visible key, odd widths
    (5, 200, 300, 8, 4, 64, 128, True, (300, 0, 1, 33, 170), 1.0),
    (9, 130, 700, 4, 2, 32, 64, False, (700, 31, 32, 33, 64, 65, 0, 1, 640), 1.0),
    (3, 90, 90, 24, 24, 40, 80, True, None, 2.0),
    (3, 129, 1100, 12, 3, 64, 128, True, (1100, 500, 64), 1.0),
]


def _attention_inputs(case, seed=11):
    B, NQ, NK, H, HK, d, dv, causal, lengths, spread = case
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(torch.bfloat16)
    a = math.sqrt(spread)
    q, k, v, lam, dout = r(B, NQ, H, 2, d, k=a), r(B, NK, HK, 2, d, k=a), r(B, NK, HK, dv), torch.rand(H, generator=g) * 1.2 - 0.2, r(B, NQ, H, dv)
    lam[1:2], lam[2:3] = -0.7, 0.0                       # a negative weight, none at all
    return q, k, v, lam, dout


@pytest.mark.parametrize("case", ATTENTION_CASES, ids=lambda c: "x".join(map(str, c[:7])) + ("-causal" if c[7] else "") + ("-lengths" if c[8] else ""))
def test_differential_attention_against_the_definition(F, case):
    causal, lengths = case[7:9]
    q, k, v, lam, dout = _attention_inputs(case)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, lam)]
    kl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = F.differential_attention(*leaves, causal=causal, key_lengths=kl)
    want, eo, gr, er = _attention_reference(q, k, v, lam, case[5] ** -0.5, causal, lengths, dout)
    _check("out", out, want, eo, torch.bfloat16)
    grads = torch.autograd.grad(out, leaves, dout.cuda())
    for n, got in zip(("v", "lam", "q", "k"), (grads[2], grads[3], grads[0], grads[1])):
        _check("d " + n, got, gr[n], er[n] + 1e-30, got.dtype)
    with torch.no_grad():
        assert torch.equal(F.differential_attention(*leaves, causal=causal, key_lengths=kl), out)
    again = torch.autograd.grad(F.differential_attention(*leaves, causal=causal, key_lengths=kl), leaves, dout.cuda())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))                  # no atomics


def test_differential_attention_layouts(F):
    """Views of a fused projection, heads-first storage, keys shared by expansion, int64 lengths, bf16 lam, an own scale: the values of
    contiguous operands; the gradient of an expanded tensor is the sum over its copies."""
    g = torch.Generator().manual_seed(9)
    B, N, H, d, dv = 2, 77, 2, 32, 64
    proj = torch.randn(B, N, H * (4 * d + dv), generator=g).to(torch.bfloat16).cuda()
    q, k, v = proj[..., :2 * H * d].view(B, N, H, 2, d), proj[..., 2 * H * d:4 * H * d].view(B, N, H, 2, d), proj[..., 4 * H * d:].view(B, N, H, dv)
    lam = torch.tensor([0.3, 0.9], device="cuda")
    want = F.differential_attention(q.contiguous(), k.contiguous(), v.contiguous(), lam)
    assert torch.equal(F.differential_attention(q, k, v, lam), want)
    hf = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(F.differential_attention(hf(q), hf(k), hf(v), lam), want)
    shifted = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(F.differential_attention(shifted, k, v, lam), want)
    assert torch.equal(F.differential_attention(q, k, v, lam.bfloat16().float()), F.differential_attention(q, k, v, lam.bfloat16()))
    ln = torch.tensor([50, 77], device="cuda")
    assert torch.equal(F.differential_attention(q, k, v, lam, key_lengths=ln), F.differential_attention(q, k, v, lam, key_lengths=ln.int()))
    assert not torch.equal(F.differential_attention(q, k, v, lam, scale=0.5), want)
    one = v[:1, :, :1].detach().clone().requires_grad_(True)
    full = one.expand(B, N, H, dv).detach().clone().requires_grad_(True)
    seed = torch.randn(B, N, H, dv, generator=g).to(torch.bfloat16).cuda()
    a = F.differential_attention(q, k, one.expand(B, N, H, dv), lam)
    b = F.differential_attention(q, k, full, lam)
    assert torch.equal(a, b)
    (ga,), (gb,) = torch.autograd.grad(a, one, seed), torch.autograd.grad(b, full, seed)
    assert float((ga.double() - gb.double().sum((0, 2), keepdim=True)).abs().max()) <= 2.0 ** -7 * float(gb.double().abs().sum((0, 2)).max())
    lq = q.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    out = F.differential_attention(lq, k, v, lam)
    (gq,) = torch.autograd.grad(out, lq, seed.transpose(1, 2).contiguous().transpose(1, 2))          # a gradient in another layout
    lq2 = q.detach().clone().requires_grad_(True)
    assert torch.equal(gq, torch.autograd.grad(F.differential_attention(lq2, k, v, lam), lq2, seed)[0])


def test_differential_attention_never_reads_behind_a_length(F):
    """NaN and infinities in keys and values behind a sample's length, also inside the last tile that is read."""
    case = (3, 70, 200, 2, 1, 64, 128, False, (0, 65, 130), 1.0)
    q, k, v, lam, dout = (t.cuda() for t in _attention_inputs(case))
    ln = torch.tensor(case[8], device="cuda")
    hidden = torch.arange(200, device="cuda")[None] >= ln[:, None]
    kn, vn = k.clone(), v.clone()
    kn[hidden], vn[hidden] = float("nan"), float("inf")
    res = []
    for kk, vv in ((k, v), (kn, vn)):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, kk, vv, lam)]
        out = F.differential_attention(*leaves, key_lengths=ln)
        res.append((out,) + torch.autograd.grad(out, leaves, dout))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert float(res[1][0][0].abs().max()) == 0.0                               # the empty sample
    assert float(res[1][2][hidden].abs().max()) == 0.0 and float(res[1][3][hidden].abs().max()) == 0.0
    # causal: a hidden key may hold anything finite, and a score of any size
    kb = k.clone()
    kb[:, -1] = 3e38
    a = F.differential_attention(q[:, :60], k[:, :100], v[:, :100], lam, causal=True)
    kb2 = k[:, :100].clone()
    kb2[:, 99] = 3e38
    b = F.differential_attention(q[:, :60], kb2, v[:, :100], lam, causal=True)
    assert torch.equal(a[:, :59], b[:, :59])
    # equal lowest scores everywhere: the mean of the values; one overwhelming score: its value alone
    qq = torch.full((1, 4, 1, 2, 32), 1e18, dtype=torch.bfloat16, device="cuda")
    kk = torch.full((1, 96, 1, 2, 32), -1e18, dtype=torch.bfloat16, device="cuda")
    vv = v[:1, :96, :1, :64].contiguous()
    out = F.differential_attention(qq, kk, vv, torch.zeros(1, device="cuda"))
    _check("mean", out[0, 0, 0], vv[0, :, 0].double().mean(0), 2.0 ** -8 * 1.06 * vv[0, :, 0].double().abs().mean(0).cpu(), torch.bfloat16)


# Both forward kernels on either side of each of the rule's limits: eight blocks of keys where every CU has a workgroup at most, 32 (64 in the
# narrow form) where more have to share one, and shares of four blocks and of eight.
WALK_CASES = [
    (2, 100, 448, 2, 1, 64, 128, True, (448, 384), 1.0),
    (2, 100, 449, 2, 1, 64, 128, True, (449, 63), 1.0),
    (3, 70, 512, 4, 4, 32, 64, False, (0, 1, 512), 1.0),
    (2, 40, 449, 2, 2, 40, 72, True, None, 2.0),
    (33, 40, 700, 8, 8, 64, 128, True, None, 1.0),
    (33, 40, 1984, 8, 8, 64, 128, False, None, 1.0),
    (33, 40, 1985, 8, 8, 64, 128, True, tuple((1985, 0, 1, 33, 700)[i % 5] for i in range(33)), 1.0),
    (33, 33, 4032, 8, 8, 32, 64, False, None, 1.0),
    (33, 33, 4033, 8, 8, 32, 64, True, None, 1.0),
    (1, 200, 2048, 1, 1, 64, 128, True, None, 1.0),
    (1, 130, 8000, 2, 1, 64, 128, True, (7000,), 1.0),
    # dQ: grids of a quarter to one workgroup per CU, on either side of walks of 12 blocks, whole and in shares
    (9, 130, 704, 8, 4, 64, 128, True, (704, 0, 1, 33, 700, 64, 65, 640, 641), 1.0),
    (9, 130, 705, 8, 4, 64, 128, True, (705, 0, 1, 33, 700, 64, 65, 640, 641), 1.0),
    (9, 130, 1600, 4, 2, 32, 64, False, (1600, 31, 32, 33, 64, 65, 0, 1, 1540), 1.0),
    (6, 90, 800, 24, 24, 40, 80, True, None, 2.0),
    (3, 129, 2400, 12, 3, 64, 128, True, (2400, 500, 64), 1.0),
]


@pytest.mark.parametrize("case", WALK_CASES, ids=lambda c: "x".join(map(str, c[:7])) + ("-causal" if c[7] else "") + ("-lengths" if c[8] else ""))
def test_differential_attention_of_short_and_long_walks(F, case):
    test_differential_attention_against_the_definition(F, case)


@pytest.mark.parametrize("B,NK,d,dv", [(3, 200, 32, 64), (3, 700, 64, 128), (3, 700, 32, 64), (140, 2000, 64, 128)])
def test_differential_attention_walks_never_read_behind_a_length(F, B, NK, d, dv):
    """As above, in a walk of every kernel that takes many rows."""
    ln = torch.tensor([(0, 65, NK - 70)[i % 3] for i in range(B)], device="cuda")
    q, k, v, lam, _ = (t.cuda() for t in _attention_inputs((B, 70, NK, 2, 2, d, dv, False, None, 1.0)))
    hidden = torch.arange(NK, device="cuda")[None] >= ln[:, None]
    kn, vn = k.clone(), v.clone()
    kn[hidden], vn[hidden] = float("nan"), float("inf")
    with torch.no_grad():
        for causal in (False, True):
            out = F.differential_attention(q, kn, vn, lam, causal=causal, key_lengths=ln)
            assert torch.equal(out, F.differential_attention(q, k, v, lam, causal=causal, key_lengths=ln))
            assert float(out[0].abs().max()) == 0.0


@pytest.mark.parametrize("slope", ["rising", "falling", "steps", "one"])
@pytest.mark.parametrize("B,NQ,H,HK,d,dv,causal", [(1, 5, 2, 1, 64, 128, False), (2, 150, 2, 1, 64, 128, True), (2, 150, 2, 2, 32, 64, False), (9, 130, 8, 4, 64, 128, True),
                                                   (1, 140, 1, 1, 128, 256, True)])
def test_differential_attention_of_steep_scores(F, B, NQ, H, HK, d, dv, causal, slope, NK=600):
    """Scores that run over a range of 300 along the keys, in a different direction in each map: the running maximum moves in every block, in
    none, now and then, or once.  fp32 scores of that size are off by 300 x 2^-23 at most, which the bounds' room beside a bf16 step covers."""
    q, k, v, lam, dout = _attention_inputs((B, NQ, NK, H, HK, d, dv, causal, None, 0.05))
    j = torch.arange(NK, dtype=torch.float64)
    f = {"rising": j * (300 / NK), "falling": (NK - j) * (300 / NK), "steps": (j // 97) * (30000 / NK), "one": 300.0 * (j == 431)}[slope]
    q[..., 0] = 8.0
    k[..., 0, 0] = (f * d ** 0.5 / 8).to(torch.bfloat16)[None, :, None]
    k[..., 1, 0] = (f.flip(0) * d ** 0.5 / 8).to(torch.bfloat16)[None, :, None]
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, lam)]
    out = F.differential_attention(*leaves, causal=causal)
    want, eo, gr, er = _attention_reference(q, k, v, lam, d ** -0.5, causal, None, dout)
    _check("out", out, want, eo, torch.bfloat16)
    grads = torch.autograd.grad(out, leaves, dout.cuda())
    for n, got in zip(("v", "lam", "q", "k"), (grads[2], grads[3], grads[0], grads[1])):
        _check("d " + n, got, gr[n], er[n] + 1e-30, got.dtype)


@pytest.mark.parametrize("slope", ["rising", "falling", "steps", "one"])
@pytest.mark.parametrize("B,NQ,H,HK,d,dv", [(9, 130, 8, 4, 64, 128), (9, 130, 8, 8, 32, 64), (33, 33, 8, 8, 64, 128)])
def test_differential_attention_of_steep_scores_in_long_walks(F, B, NQ, H, HK, d, dv, slope):
    test_differential_attention_of_steep_scores(F, B, NQ, H, HK, d, dv, True, slope, NK=2000 if B == 33 else 800)


def test_differential_attention_gradients_against_differences(F):
    """The output is linear in lam and in v: differences over whole steps are exact but for the stored roundings (2^-8 of the two
    outputs and of the probabilities)."""
    case = (2, 96, 96, 2, 1, 32, 64, True, None, 1.0)
    q, k, v, lam, dout = (t.cuda() for t in _attention_inputs(case))
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, lam)]
    gq, gk, gv, gl = torch.autograd.grad(F.differential_attention(*leaves, causal=True), leaves, dout)
    f = lambda *a: (F.differential_attention(*a, causal=True).double() * dout.double())
    up = lam.clone()
    up[0] += 1.0
    a, b = f(q, k, v, up), f(q, k, v, lam)
    room = 3 * 2.0 ** -8 * float((a[:, :, 0].abs() + b[:, :, 0].abs()).sum() + (F.differential_attention(q, k, v.abs(), torch.zeros_like(lam), causal=True).double() * dout.double()).abs().sum())
    assert abs(float((a - b).sum()) - float(gl[0])) < room
    dvv = torch.zeros_like(v)
    dvv[0, 17] = 1.0
    a, b = f(q, k, v + dvv, lam).sum(), f(q, k, v, lam).sum()
    step = (v + dvv).double() - v.double()
    assert abs(float(a - b) - float((gv.double() * step).sum())) < room
    # q and k: the definition in float64 stands in for the (bf16) kernel, whose own differences drown in rounding
    qd, kd, vd = (t.cpu().double() for t in (q, k, v))
    u = torch.randn(qd.shape, generator=torch.Generator().manual_seed(4), dtype=torch.float64)

    def plain(x):
        out, _, _, _ = _attention_reference(x, kd, vd, lam.cpu(), 32 ** -0.5, True, None, dout.cpu())
        return float((out * dout.cpu().double()).sum())

    diff = (plain(qd + 1e-4 * u) - plain(qd - 1e-4 * u)) / 2e-4
    along = float((gq.cpu().double() * u).sum())
    assert abs(diff - along) < 2.0 ** -7 * float(gq.double().norm()) * 4 + 1e-6 * abs(diff), (diff, along)


def test_differential_attention_of_a_cache_past_32_bits(F):
    """Keys and values of more than 4 GiB each: all but the last key are zeros, the last one's score in the first map (128 above the others')
    leaves e^-128 x 2^21 to them, the second map is uniform, so the result is the last value (and 2^-21 of it), rounded once, and the last
    value's gradient the sum of the incoming ones."""
    NK, H, d, dv = (1 << 21) + 70, 8, 64, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB")
    k = torch.zeros(1, NK, H, 2, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, NK, H, dv, dtype=torch.bfloat16, device="cuda")
    assert k.numel() * 2 > 1 << 32 and v.numel() * 2 > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(8)
    last = torch.randn(H, dv, generator=g, device="cuda").bfloat16()
    k[0, -1, :, 0], v[0, -1] = 4.0, last
    k.requires_grad_(True), v.requires_grad_(True)
    lam = torch.full((H,), 0.5, device="cuda")
    for NQ in (1, 40):                                     # the kernel for few rows, and the general one
        q = torch.full((1, NQ, H, 2, d), 4.0, dtype=torch.bfloat16, device="cuda")
        out = F.differential_attention(q, k, v, lam)
        assert float((out[0].float() - last.float()).abs().max()) <= 2.0 ** -8 * float(last.float().abs().max())
        dout = torch.randn(out.shape, generator=g, device="cuda").bfloat16()
        gk, gv = torch.autograd.grad(out, (k, v), dout)
        want = dout[0].double().sum(0)
        # each addend's probability and the sum are rounded to bf16
        assert bool(((gv[0, -1].double() - want).abs() <= 2.0 ** -8 * (want.abs() + dout[0].double().abs().sum(0)) + 1e-6).all())
        assert float(gv[0, :-1].abs().max()) <= 2.0 ** -20 * float(dout.float().abs().sum(1).max())
        assert bool(torch.isfinite(gk[0, -64:]).all()) and float(gk[0, :64].abs().max()) <= 1e-3
        del out, gk, gv


def test_differential_attention_weight_gradient_of_many_rows(F):
    """dlam is one sum over 131072 rows of either sign: a rounding that always goes one way would add up.  A row's term, dO . O2, is a
    difference of sums of fp32 values no larger than S = |delta1| + |delta2| + sum_j p2 |dP|, each step of them off by half of 2^-23 of S
    at most; three steps (the products' sum, the start value, the sum over the keys) and independent signs leave
    sqrt(sum S^2) x 3 x 2^-24, four times which nothing should pass."""
    B, N, d, dv = 32, 4096, 64, 128
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k = (torch.randn(B, N, 1, 2, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    v, dout = (torch.randn(B, N, 1, dv, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    lam = torch.tensor([0.4], device="cuda", requires_grad=True)
    got, = torch.autograd.grad(F.differential_attention(q, k, v, lam), lam, dout)
    want, spread = 0.0, 0.0
    for b in range(B):
        dP = dout[b, :, 0].double() @ v[b, :, 0].double().t().contiguous()
        P = [torch.softmax(q[b, :, 0, m].double() @ k[b, :, 0, m].double().t().contiguous() * d ** -0.5, -1) for m in range(2)]
        d1, d2 = ((p * dP).sum(-1) for p in P)
        want -= float(d2.sum())
        spread += float(((d1.abs() + d2.abs() + (P[1] * dP.abs()).sum(-1)) ** 2).sum())
    assert abs(float(got) - want) <= 4 * 3 * 2.0 ** -24 * math.sqrt(spread), (float(got) - want, math.sqrt(spread))


def test_differential_attention_empty_tensors(F):
    for B, NQ, NK in ((0, 4, 4), (2, 0, 5), (2, 3, 0)):
        q = torch.randn(B, NQ, 2, 2, 32, device="cuda").bfloat16().requires_grad_(True)
        k = torch.randn(B, NK, 1, 2, 32, device="cuda").bfloat16().requires_grad_(True)
        v = torch.randn(B, NK, 1, 64, device="cuda").bfloat16().requires_grad_(True)
        lam = torch.ones(2, device="cuda", requires_grad=True)
        out = F.differential_attention(q, k, v, lam)
        grads = torch.autograd.grad(out.float().sum(), (q, k, v, lam))
        assert out.shape == (B, NQ, 2, 64) and float(out.float().abs().sum()) == 0.0
        assert all(g.shape == t.shape and float(g.float().abs().sum()) == 0.0 for g, t in zip(grads, (q, k, v, lam)))


# ---- streams, graphs, refusals -------------------------------------------------------------------------------------------------
def _chain(F, t, table, pos):
    """norm -> projections -> rotary -> differential attention -> head norm -> boundary norm, as a block uses them."""
    x = t["x"]
    B, N, C = x.shape
    H, d, dv = 2, 32, 64
    h = F.block_input_norm(x, t["w1"])
    qkv = (h.reshape(B * N, C) @ t["proj"]).reshape(B, N, -1)
    q, k, v = qkv[..., :2 * H * d].view(B, N, 2 * H, d), qkv[..., 2 * H * d:4 * H * d].view(B, N, 2 * H, d), qkv[..., 4 * H * d:].view(B, N, H, dv)
    q, k = F.axial_rotary(q, k, pos, table)
    o = F.differential_attention(q.view(B, N, H, 2, d), k.view(B, N, H, 2, d), v, t["lam"])
    o = F.block_input_norm(o, t["wh"])
    return F.block_boundary_norm(x, o.reshape(B, N, C), t["w2"], t["w3"], gate=t["gate"], residual_scale=t["rho"])


def _chain_tensors(seed=0, B=2, N=80):
    g = torch.Generator().manual_seed(seed)
    C = 128
    r = lambda *s, k=1.0, o=0.0: torch.randn(*s, generator=g) * k + o
    t = {"x": r(B, N, C).bfloat16(), "w1": r(C, k=0.1, o=1), "proj": r(C, 2 * 2 * 32 * 2 + 128, k=C ** -0.5).bfloat16(), "lam": r(2, k=0.1, o=0.5),
         "wh": r(64, k=0.1, o=1), "w2": r(C, k=0.1, o=1), "w3": r(C, k=0.1, o=1), "gate": r(C, k=0.3), "rho": r(1, k=0.05, o=0.9)}
    return {n: v.cuda().requires_grad_(True) for n, v in t.items()}, torch.stack((torch.arange(N) // 8, torch.arange(N) % 8), 1).cuda()


def test_the_operators_together_against_plain_torch(F):
    """The block in float64 torch operations on the same operands; bf16 activations between the steps, so the bounds are those of a
    chain of roundings (the block's depth of 6 stored tensors, relative to the tensors' norms)."""
    t, pos = _chain_tensors()
    table = F.rotary_table((16, 16), device="cuda")
    y, h = _chain(F, t, table, pos)
    sy, sh = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).bfloat16().cuda(), torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    grads = torch.autograd.grad((y, h), list(t.values()), (sy, sh))
    r = {n: v.detach().cpu().double().requires_grad_(True) for n, v in t.items()}
    B, N, C = r["x"].shape
    rms = lambda z, w: z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * w
    qkv = rms(r["x"], r["w1"]) @ r["proj"]
    ang = torch.cat([pos.cpu().double()[:, a, None] * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16) for a in range(2)], -1)[None, :, None]

    def turn(z):
        a, b = z[..., 0::2], z[..., 1::2]
        return torch.stack((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()), -1).flatten(-2)

    q, k, v = turn(qkv[..., :128].reshape(B, N, 4, 32)), turn(qkv[..., 128:256].reshape(B, N, 4, 32)), qkv[..., 256:].reshape(B, N, 2, 64)
    P = torch.softmax(torch.einsum("bihd,bjhd->bhij", q, k) * 32 ** -0.5, -1)
    o = torch.einsum("bhij,bjhc->bihc", P[:, 0::2] - r["lam"][None, :, None, None] * P[:, 1::2], v)
    yr = r["rho"] * r["x"] + r["gate"] * rms(rms(o, r["wh"]).reshape(B, N, C), r["w2"])
    hr = rms(yr, r["w3"])
    want = torch.autograd.grad((yr, hr), list(r.values()), (sy.cpu().double(), sh.cpu().double()))
    rel = lambda a, b: float((a.detach().cpu().double() - b).norm() / b.norm())
    # 6 stored tensors forward, as many again backward; an independent rounding has an rms of 2^-8 / sqrt(3)
    assert rel(y, yr) < 2.0 ** -8 * 6 and rel(h, hr) < 2.0 ** -8 * 6
    for n, a, b in zip(t, grads, want):
        assert rel(a, b) < 2.0 ** -8 * 12, (n, rel(a, b))


def test_recorded_and_replayed_with_eager_work_between(F):
    """Forward and backward of the chain in one graph, replayed with other inputs while an eager graph of the same leaves lives and
    eager calls (their own workspaces) run between the replays: every replay equals the eager result."""
    t, pos = _chain_tensors()
    table = F.rotary_table((16, 16), device="cuda")
    live = _chain(F, t, table, pos)                                      # an eager graph of the same leaves, kept alive
    static = {n: v.detach().clone().requires_grad_(True) for n, v in t.items()}
    seed = torch.randn(t["x"].shape, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()

    def step(s):
        y, h = _chain(F, s, table, pos)
        return (y, h) + torch.autograd.grad((y, h), list(s.values()), (seed, seed))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                   # two recordings: their workspaces are their own
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(static)
        graphs.append((gr, out))
    for i in range(4):
        fresh, _ = _chain_tensors(seed=10 + i)
        with torch.no_grad():
            for n in static:
                static[n].copy_(fresh[n])
        want = step(fresh)
        for gr, out in graphs:
            gr.replay()
        again = step(fresh)
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    torch.autograd.grad(live, list(t.values()), (seed, seed))


def test_calls_on_another_stream(F):
    t, pos = _chain_tensors()
    table = F.rotary_table((16, 16), device="cuda")
    want = _chain(F, t, table, pos)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(F, t, table, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_order_and_changed_operands_are_refused(F):
    t, pos = _chain_tensors()
    x = t["x"].detach().float().requires_grad_(True)
    h = F.block_input_norm(x, t["w1"])
    (gx,) = torch.autograd.grad(h.square().sum(), x, create_graph=False)
    h = F.block_input_norm(x, t["w1"])
    with pytest.raises(RuntimeError, match="second-order"):
        torch.autograd.grad(h.square().sum(), x, create_graph=True)
    q = torch.randn(1, 8, 1, 2, 32, device="cuda").bfloat16().requires_grad_(True)
    v = torch.randn(1, 8, 1, 64, device="cuda").bfloat16()
    out = F.differential_attention(q, q.detach(), v, torch.ones(1, device="cuda"))
    v.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()


def test_saved_tensors_that_come_back_elsewhere(F):
    """Tensors offloaded between the passes (saved-tensor hooks) come back at other addresses, sliced ones with other strides, and a
    parameter's storage may be given up and gathered anew: the backward pass reads them where they are then."""
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    qkv = r(2, 70, 2, 2, 96).bfloat16().requires_grad_(True)
    lam, x, w, gate = r(2).requires_grad_(True), r(2, 70, 128).requires_grad_(True), r(128).requires_grad_(True), r(2, 128).bfloat16().requires_grad_(True)
    dout = r(2, 70, 128)
    table, places = F.rotary_table((16, 16), device="cuda"), torch.arange(140, device="cuda").view(70, 2)

    def grads(hooks, between=lambda: None):
        with hooks:
            q, k = F.axial_rotary(qkv[..., :32].reshape(2, 70, 4, 32), qkv[..., 32:64].reshape(2, 70, 4, 32), places, table)
            a = F.differential_attention(q.view(2, 70, 2, 2, 32), qkv[..., 32:64], qkv[:, :, :, 0, 32:], lam)
            y, h = F.block_boundary_norm(x, a.float().flatten(2), w, None, gate=gate, residual_scale=w)
            loss = ((y + h) * dout).sum()
        between()
        return torch.autograd.grad(loss, (qkv, lam, x, w, gate))

    class Elsewhere(torch.autograd.graph.saved_tensors_hooks):
        def __init__(self):
            super().__init__(lambda t: (t.cpu(), t.stride()), lambda p: torch.cat([p[0].flatten()[:1], p[0].flatten()]).cuda()[1:].view(p[0].shape))

    plain = grads(contextlib.nullcontext())
    assert all(torch.equal(a, b) for a, b in zip(plain, grads(torch.autograd.graph.save_on_cpu())))
    # off by one element the norm's kernel takes narrower accesses and adds in another order; the bf16 gradient that reaches the attention
    # then rounds to a neighbouring value here and there, 2^-7 of itself, and all others are linear in it
    for a, b in zip(plain, grads(Elsewhere())):
        assert float((a.float() - b.float()).norm()) <= 2.0 ** -7 * float(a.float().norm())

    def gather_anew():
        old = w.data
        w.data = old.clone()
        old.fill_(float("nan"))

    assert all(torch.equal(a, b) for a, b in zip(plain, grads(contextlib.nullcontext(), gather_anew)))
