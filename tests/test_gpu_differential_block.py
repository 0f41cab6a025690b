"""gan_amd.nn.DifferentialAttention2d and BigGAN with attention="differential": the block against plain torch operations in float64,
one training step eager and recorded."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gan():
    import gan_amd
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return gan_amd


def _reference(m, x, p):
    """The module's formula on float64 copies `p` of its parameters."""
    B, C, H, W = x.shape
    N = H * W
    rms = lambda z, w: z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * w
    y = x.permute(0, 2, 3, 1).reshape(B, N, C)
    n = torch.arange(N)
    pos = torch.stack((n // W, n % W), 1).double()
    for i, b in enumerate(m.blocks):
        heads, d = b.heads, b.head_dim
        dims = b.rotary.dims
        ang = torch.cat([pos[:, a, None] * 10000.0 ** (-torch.arange(0, k, 2, dtype=torch.float64) / k) for a, k in enumerate(dims)], -1)[None, :, None]

        def turn(z):
            u, v = z[..., 0::2], z[..., 1::2]
            return torch.stack((u * ang.cos() - v * ang.sin(), u * ang.sin() + v * ang.cos()), -1).flatten(-2)

        g = lambda name: p[f"blocks.{i}.{name}"]
        qkv = rms(y, p[f"in_norm.{i}"]) @ g("qkv.weight").flatten(1).t()
        q, k, v = turn(qkv[..., :C].reshape(B, N, 2 * heads, d)), turn(qkv[..., C:2 * C].reshape(B, N, 2 * heads, d)), qkv[..., 2 * C:].reshape(B, N, heads, 2 * d)
        P = torch.softmax(torch.einsum("bihd,bjhd->bhij", q, k) * d ** -0.5, -1)
        lam = (g("lambda_q1") * g("lambda_k1")).sum(1).exp() - (g("lambda_q2") * g("lambda_k2")).sum(1).exp() + b.lambda_init
        o = torch.einsum("bhij,bjhc->bihc", P[:, 0::2] - lam[None, :, None, None] * P[:, 1::2], v)
        f = rms(o, g("head_norm")).reshape(B, N, C) @ g("out.weight").flatten(1).t()
        y = y + p[f"gate.{i}"] * rms(f, p[f"out_norm.{i}"])
    return y.reshape(B, H, W, C).permute(0, 3, 1, 2)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C,heads,depth,H,W", [(64, None, 1, 8, 8), (128, 2, 2, 9, 7), (32, 1, 1, 5, 12)])
def test_block_against_float64(gan, C, heads, depth, H, W, dt):
    """Between x and the result lie up to 8 stored bf16 tensors per block (norm, weights and activations of two projections, q and k,
    the attention and its probabilities, the head norm), each off by an rms of 2^-8 / sqrt(3) at most; the gradients pass as many again."""
    torch.manual_seed(3)
    m = gan.nn.DifferentialAttention2d(C, heads, depth)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.startswith("gate"):
                p.uniform_(0.3, 1.0)
            elif "norm" in n:
                p.uniform_(0.7, 1.3)
    x = torch.randn(2, C, H, W).to(dt)
    seed = torch.randn(2, C, H, W).to(dt)
    p64 = {n: t.detach().double().requires_grad_(True) for n, t in m.named_parameters()}
    x64 = x.double().requires_grad_(True)
    want = _reference(m, x64, p64)
    wg = torch.autograd.grad(want, [x64, *p64.values()], seed.double())
    m.cuda()
    xg = x.cuda().contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = m(xg)
    assert y.dtype == dt and y.shape == x.shape
    got = torch.autograd.grad(y, [xg, *m.parameters()], seed.cuda())
    rel = lambda a, b: float((a.detach().cpu().double() - b).norm() / b.norm())
    u = 2.0 ** -8 / 3 ** 0.5
    assert rel(y, want) < 8 * depth * u, rel(y, want)
    for n, a, b in zip(["x", *p64], got, wg):
        # (the weights of lambda and of the q / k projections act through differences of probabilities, an order smaller than what they
        #  are differences of)
        room = 100 if "lambda" in n else (40 if "qkv" in n else 16)
        assert rel(a, b) < room * depth * u, (n, rel(a, b))
    plain = gan.nn.DifferentialAttention2d(C, heads, depth).cuda()
    assert torch.equal(plain(xg), xg)                                     # gate 0: the identity


def test_biggan_step_eager_and_recorded(gan):
    from gan_amd.harness import biggan as H
    torch.manual_seed(1)
    G, D = H.Generator(10, 16, attention="differential").cuda(), H.Discriminator(10, 16, attention="differential").cuda()
    with torch.no_grad():
        for net in (G, D):
            for n, p in net.named_parameters():
                if ".gate." in n:
                    p.fill_(0.5)
    H.set_activation_dtype(torch.bfloat16)
    try:
        real = torch.rand(4, 3, 128, 128, device="cuda").mul(2).sub(1).contiguous(memory_format=torch.channels_last)
        rl, fl = torch.tensor([1, 2, 3, 4], device="cuda"), torch.tensor([5, 6, 7, 8], device="cuda")
        z = torch.randn(4, 120, device="cuda")
        params = [*G.parameters(), *D.parameters()]
        buffers = {n: b.clone() for net in (G, D) for n, b in net.named_buffers()}

        def step():
            for p in params:
                p.grad = None
            a, b = H.discriminator_phase(G, D, real, rl, z, fl)
            c = H.generator_phase(G, D, z, fl)
            return [a, b, c] + [p.grad for p in params if p.grad is not None]

        eager = step()
        assert all(torch.isfinite(t).all() for t in eager)
        for net in (G, D):
            blocks = [b for b in net.main_sequence if isinstance(b, H.DifferentialAttentionBlock)]
            assert len(blocks) == 1 and buffers
            for p in blocks[0].parameters():
                assert p.grad is not None and float(p.grad.abs().sum()) > 0
        recorded = gan.GraphedStep(step)
        for _ in range(2):
            out = recorded()
            torch.cuda.synchronize()
            assert all(torch.isfinite(t).all() for t in out)
    finally:
        H.set_activation_dtype(None)
