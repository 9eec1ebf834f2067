"""8-bit activation checkpoints (ops.ckpt8_* / gelu_*_ckpt8 / layernorm_*_ckpt8) against their definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32, HALF_BF16 = 2.0 ** -24, 2.0 ** -8


def ops():
    from ssrs_amd import ops as o
    return o


def values64(x):
    """what the checkpoint of x [..., C] stands for, from the definition"""
    x = x.double().cpu()
    C = x.shape[-1]
    out = torch.empty_like(x)
    for lo in range(0, C, 32):
        b = x[..., lo:lo + 32]
        amax = b.abs().amax(-1, keepdim=True)
        mant, ex = torch.frexp(amax)
        e = torch.where(mant > 127 / 128, ex - 6, ex - 7)
        e = torch.where(amax == 0, torch.full_like(e, -126), e).clamp(-126, 121)
        step = torch.ldexp(torch.ones_like(amax), e)
        v = torch.round(b / step).clamp(-127, 127) * step
        out[..., lo:lo + 32] = torch.where(torch.isfinite(amax), v, torch.full_like(v, math.nan))
    return out


def tokens(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1:], generator=g))
    return x.to(dtype).cuda()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double().cpu(), nan=7e77), torch.nan_to_num(b, nan=7e77))


# rows of one element to long ones, widths that end inside a block, widths of the vector path and not
SHAPES = [(1,), (1, 1), (3, 31), (2, 32), (5, 33), (7, 40), (2, 3, 64), (4, 100), (977, 1003), (130, 1280), (33, 2056), (0, 64), (1, 70001), (70000, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_unpack_is_the_definition(shape, dtype):
    o = ops()
    x = tokens(shape, dtype)
    c = o.ckpt8_pack(x)
    blocks = (shape[-1] + 31) // 32
    assert 0 <= c.nbytes - x.numel() - (x.numel() // shape[-1]) * blocks < 16 and c.shape == tuple(shape)
    assert c.codes.shape == shape and c.codes.dtype == torch.int8 and c.exps.shape == tuple(shape[:-1]) + (blocks,)
    for dt in (torch.float32, torch.bfloat16):                  # the values are exact in both
        assert same(o.ckpt8_unpack(c, dt), values64(x))


def test_pack_edge_values():
    """zeros, ties, the step's border (127 * 2^k and the next number), subnormals, the largest numbers, infinities, NaN"""
    o = ops()
    rows = [torch.zeros(32), torch.full((32,), -0.0),
            torch.tensor([127.0] + [0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -126.5] + [0.0] * 24),
            torch.tensor([127.00001] + [1.0, 3.0, 5.0, -1.0, -3.0] + [0.0] * 26),
            torch.tensor([1.984375, 1e-3] + [0.0] * 30), torch.tensor([1.9843751, 1e-3] + [0.0] * 30),
            torch.tensor([1e-40, -3e-39, 1.2e-38] + [0.0] * 29), torch.tensor([2.0 ** -126 * 127, 2.0 ** -127] + [0.0] * 30),
            torch.tensor([3.4028234e38, -3.4028234e38, 1e38, 127 * 2.0 ** 121] + [0.0] * 28),
            torch.tensor([math.inf] + [1.0] * 31), torch.tensor([math.nan] + [1.0] * 31), torch.tensor([1.0] * 31 + [-math.inf])]
    x = torch.stack(rows)
    for t in (x, x.repeat(1, 3), torch.cat([x, x[:, :5]], 1)):      # vector path, several blocks, the one-element path with a short block
        v = o.ckpt8_unpack(o.ckpt8_pack(t.cuda()), torch.float32)
        assert same(v, values64(t))
        assert torch.isfinite(v[:9]).all() and torch.isnan(v[9:, :32]).all()


def test_pack_of_views():
    """row strides, column slices at odd offsets, transposed views, expanded rows: what torch calls the same values"""
    o = ops()
    x = tokens((70, 264), torch.bfloat16)
    for v in (x[:, 8:200], x[:, 3:100], x[::3], x.t(), x[5:6].expand(9, 264), x[:, :1], x.view(7, 10, 264)[:, 2:5], x[3]):
        assert same(o.ckpt8_unpack(o.ckpt8_pack(v), torch.float32), values64(v.contiguous()))
    f = tokens((40, 96), torch.float32)[:, 1:65]                 # fp32 rows that are not 16-byte aligned
    assert same(o.ckpt8_unpack(o.ckpt8_pack(f), torch.bfloat16), values64(f))


def gelu64(x):
    x = x.double()
    return x * 0.5 * torch.erfc(-x / math.sqrt(2))


def slope64(x):
    x = x.double()
    return 0.5 * torch.erfc(-x / math.sqrt(2)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (5, 64), (256, 1024), (19, 1003), (0, 32), (2, 3, 96)])
def test_gelu_forward_backward(shape, dtype):
    """Bounds. Phi's polynomial 3.8e-7 relative; exp(-x^2/2): three roundings of an argument of size x^2/2 (3 * 2^-24 * x^2/2 relative,
    doubled for the exponential's own steps) and 2^-22 of its own; the result's rounding. Below 1e-37 the exponential is flushed."""
    o = ops()
    half = HALF_BF16 if dtype == torch.bfloat16 else EPS32
    x = 3 * tokens(shape, dtype, 1)
    if x.numel() > 64:
        x.view(-1)[:6] = torch.tensor([0.0, -0.0, 12.5, -9.0, -4.0, 40.0], dtype=dtype, device="cuda")
    dy = tokens(shape, dtype, 2)
    act, c = o.gelu_fwd_ckpt8(x)
    assert same(o.ckpt8_unpack(c, torch.float32), values64(x))
    xd = x.double().cpu()
    rel = 1.2e-6 + 6 * EPS32 * xd * xd
    ref = gelu64(xd)
    assert ((act.double().cpu() - ref).abs() <= ref.abs() * (rel + half) + 1e-36).all()
    x8 = values64(x)
    dx, again = o.gelu_bwd_ckpt8(c, dy, want_act=True)
    assert torch.equal(dx, o.gelu_bwd_ckpt8(c, dy))
    rel8 = 1.2e-6 + 6 * EPS32 * x8 * x8
    ref8, d = gelu64(x8), dy.double().cpu()
    assert ((again.double().cpu() - ref8).abs() <= ref8.abs() * (rel8 + half) + 1e-36).all()
    # the slope is a sum of two terms that cancel near x = -0.75: its error is relative to the terms
    terms = 0.5 * torch.erfc(-x8 / math.sqrt(2)) + x8.abs() * torch.exp(-0.5 * x8 * x8) / math.sqrt(2 * math.pi)
    refd = d * slope64(x8)
    assert ((dx.double().cpu() - refd).abs() <= d.abs() * terms * (rel8 + 4 * EPS32) + refd.abs() * half + 1e-36).all()
    if dtype == torch.float32 and x.numel() > 64:               # the formula against differences of the formula, at the checkpoint's values
        h = 1e-6
        assert ((gelu64(x8 + h) - gelu64(x8 - h)) / (2 * h) - slope64(x8)).abs().max() < 1e-8


def test_gelu_nonfinite_reaches_the_gradient():
    o = ops()
    x = torch.ones(2, 64, device="cuda")
    x[1, 40] = math.inf
    act, c = o.gelu_fwd_ckpt8(x)
    assert torch.isinf(act[1, 40]) and torch.isfinite(act[0]).all()
    dx = o.gelu_bwd_ckpt8(c, torch.ones_like(x))
    assert torch.isnan(dx[1, 32:]).all() and torch.isfinite(dx[0]).all() and torch.isfinite(dx[1, :32]).all()


def ln64(x, gamma, beta, eps):
    x = x.double().cpu()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    return mean, rstd, (x - mean) * rstd * gamma + beta


LN_CASES = [(1, 32, torch.float32, torch.bfloat16), (5, 64, torch.bfloat16, torch.float32), (33, 128, torch.float32, torch.float32),
            (512, 768, torch.float32, torch.bfloat16), (70, 1024, torch.bfloat16, torch.bfloat16), (4200, 1280, torch.float32, torch.bfloat16),
            (9, 2048, torch.float32, torch.bfloat16), (0, 96, torch.float32, torch.bfloat16), (6, 1760, torch.bfloat16, torch.bfloat16),
            (10, 1376, torch.float32, torch.float32), (2048, 96, torch.bfloat16, torch.float32), (2049, 96, torch.float32, torch.float32),
            (2100, 1760, torch.float32, torch.bfloat16), (65, 32, torch.float32, torch.float32)]


@pytest.mark.parametrize("rows,C,xdt,ddt", LN_CASES)
def test_layernorm_forward_backward(rows, C, xdt, ddt):
    """Bounds: the row sums add at most 32 terms per lane and 6 in the tree: 40 * 2^-24 of the sum of magnitudes; a few roundings more
    per element. u is the error of a normalised value, from the mean's error and the subtraction."""
    o = ops()
    x = tokens((rows, C), xdt, 3) + 0.5
    g = torch.Generator().manual_seed(4)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    dy, dres = tokens((rows, C), ddt, 5), tokens((rows, C), torch.float32, 6)
    y, mean, rstd, c = o.layernorm_fwd_ckpt8(x, gamma.cuda(), beta.cuda(), 1e-6)
    assert same(o.ckpt8_unpack(c, torch.float32), values64(x))
    mean64, rstd64, y64 = ln64(x, gamma.double(), beta.double(), 1e-6)
    k = 48 * EPS32
    xd = x.double().cpu()
    big = xd.abs().amax(-1, keepdim=True) if rows else xd.abs()[:, :1]
    u = k * big * rstd64 + k * (xd - mean64).abs() * rstd64
    assert ((y.double().cpu() - y64).abs() <= y64.abs() * HALF_BF16 + (u + EPS32) * (gamma.abs() + beta.abs()) * 2).all()
    assert ((mean.double().cpu() - mean64[:, 0]).abs() <= k * big[:, 0]).all()
    assert ((rstd.double().cpu() / rstd64[:, 0] - 1).abs() <= 4 * k).all()
    xh = (values64(x) - mean64) * rstd64
    d, t = dy.double().cpu(), dy.double().cpu() * gamma.double()
    m1, m2 = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    ref = rstd64 * (t - m1 - xh * m2) + dres.double().cpu()
    u8 = k * big * rstd64 + 5 * k * xh.abs()
    a1, a2 = t.abs().mean(-1, keepdim=True), (t * xh).abs().mean(-1, keepdim=True)
    tol = rstd64 * (k * (t.abs() + a1 + xh.abs() * a2) * 2 + u8 * a2 + xh.abs() * (t.abs() * u8).mean(-1, keepdim=True)) * 2 + 4 * EPS32 * (ref.abs() + dres.double().cpu().abs())
    dx, dxb, y2, dg, db = o.layernorm_bwd_ckpt8(dy, c, mean, rstd, gamma.cuda(), beta.cuda(), dres.cuda(), want_bf16=True, want_y=True, want_weights=True)
    assert ((dx.double().cpu() - ref).abs() <= tol).all()
    assert torch.equal(dxb, dx.to(torch.bfloat16))
    y8 = xh * gamma.double() + beta.double()
    assert ((y2.double().cpu() - y8).abs() <= y8.abs() * HALF_BF16 + (u8 + EPS32) * (gamma.abs() + beta.abs()) * 2).all()
    # sums over the rows: per wave, then 8 waves, then up to 128 slabs and 4 quarters
    depth = rows / 4096 + 8 + 128 + 4 + 8
    assert ((dg.double().cpu() - (d * xh).sum(0)).abs() <= depth * EPS32 * (d * xh).abs().sum(0) + (d.abs() * u8).sum(0)).all()
    assert ((db.double().cpu() - d.sum(0)).abs() <= depth * EPS32 * d.abs().sum(0)).all()
    # fewer results are the same results; without the residual gradient the sum is that much smaller
    assert torch.equal(o.layernorm_bwd_ckpt8(dy, c, mean, rstd, gamma.cuda(), dres=dres.cuda()), dx)
    only = o.layernorm_bwd_ckpt8(dy, c, mean, rstd, gamma.cuda(), want_f32=False, want_bf16=True)
    refn = ref - dres.double().cpu()
    assert ((only.double().cpu() - refn).abs() <= tol + refn.abs() * HALF_BF16).all()


def test_layernorm_views_and_gradient_by_differences():
    """strided inputs; and the backward against differences of the forward where the checkpoint is exact (inputs on its grid)"""
    o = ops()
    wide = tokens((40, 200), torch.float32, 7)
    x, gamma, beta = wide[:, 4:132], torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")
    a = o.layernorm_fwd_ckpt8(x, gamma, beta, 1e-6)
    b = o.layernorm_fwd_ckpt8(x.contiguous(), gamma, beta, 1e-6)
    assert torch.equal(a[0], b[0]) and torch.equal(a[3].codes, b[3].codes)
    odd = wide[:, 1:129]                                            # not 16-byte aligned: copied
    assert torch.equal(o.layernorm_fwd_ckpt8(odd, gamma, beta, 1e-6)[0], o.layernorm_fwd_ckpt8(odd.contiguous(), gamma, beta, 1e-6)[0])
    g = torch.Generator().manual_seed(8)
    xs = torch.randint(-126, 127, (3, 64), generator=g).float() / 16
    xs[:, ::32] = 127 / 16
    dy = torch.randn(3, 64, generator=g)
    ga = (1 + torch.rand(64, generator=g)).double()
    assert torch.equal(values64(xs), xs.double())
    y, mean, rstd, c = o.layernorm_fwd_ckpt8(xs.cuda(), ga.float().cuda(), torch.zeros(64, device="cuda"), 1e-6)
    dx = o.layernorm_bwd_ckpt8(dy.cuda(), c, mean, rstd, ga.float().cuda()).double().cpu()

    def loss(v):
        return (ln64(v, ga, 0.0, 1e-6)[2] * dy.double()).sum()
    for i, j in ((0, 0), (1, 17), (2, 63), (0, 32)):
        h = 1e-5
        e = torch.zeros(3, 64, dtype=torch.float64)
        e[i, j] = h
        # third-order term of the difference and the fp32 arithmetic of dx
        assert abs(((loss(xs.double() + e) - loss(xs.double() - e)) / (2 * h)).item() - dx[i, j].item()) < 1e-5


def test_streams_and_graph_replays():
    """on a stream of its own, and captured: every replay on new inputs equals the eager call"""
    o = ops()
    x, dy = tokens((300, 768), torch.float32, 9), tokens((300, 768), torch.bfloat16, 10)
    gamma, beta = torch.rand(768, device="cuda") + 0.5, torch.rand(768, device="cuda")

    def step(x, dy):
        y, mean, rstd, c = o.layernorm_fwd_ckpt8(x, gamma, beta, 1e-6)
        dx, dg, db = o.layernorm_bwd_ckpt8(dy, c, mean, rstd, gamma, want_weights=True)
        act, k = o.gelu_fwd_ckpt8(y)
        return y, dx, dg, db, act, o.gelu_bwd_ckpt8(k, dy), o.ckpt8_unpack(o.ckpt8_pack(x))
    ref = step(x, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x, dy)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    sx, sd = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out = step(sx, sd)
    for k in range(3):
        sx.copy_(tokens((300, 768), torch.float32, 20 + k))
        sd.copy_(tokens((300, 768), torch.bfloat16, 30 + k))
        graph.replay()
        torch.cuda.synchronize()
        ref = step(sx, sd)
        assert all(torch.equal(a, b) for a, b in zip(ref, out)), k


def test_refusals():
    o = ops()
    from ssrs_amd._lib import MfnetError
    x = torch.randn(4, 64, device="cuda")
    c = o.ckpt8_pack(x)
    v = torch.ones(64, device="cuda")
    m = torch.ones(4, device="cuda")
    for bad in (lambda: o.ckpt8_pack(x.double()), lambda: o.ckpt8_pack(x.half()), lambda: o.ckpt8_pack(x.cpu()), lambda: o.ckpt8_pack(x[:, :0]),
                lambda: o.ckpt8_pack(torch.tensor(1.0, device="cuda")), lambda: o.ckpt8_unpack(c, torch.float16),
                lambda: o.gelu_bwd_ckpt8(c, x[:3]), lambda: o.gelu_bwd_ckpt8(c, x.double()), lambda: o.gelu_bwd_ckpt8(c, x.cpu()),
                lambda: o.layernorm_fwd_ckpt8(x[:, :40], v[:40], v[:40], 1e-6), lambda: o.layernorm_fwd_ckpt8(x, v[:32], v, 1e-6),
                lambda: o.layernorm_fwd_ckpt8(torch.randn(2, 2080, device="cuda"), torch.ones(2080, device="cuda"), torch.ones(2080, device="cuda"), 1e-6),
                lambda: o.layernorm_fwd_ckpt8(x, v.double(), v, 1e-6), lambda: o.layernorm_bwd_ckpt8(x[:3], c, m, m, v),
                lambda: o.layernorm_bwd_ckpt8(x, c, m[:3], m, v), lambda: o.layernorm_bwd_ckpt8(x, c, m, m, v, want_y=True),
                lambda: o.layernorm_bwd_ckpt8(x, c, m, m, v, want_f32=False), lambda: o.layernorm_bwd_ckpt8(x, c, m, m, v, dres=x.double())):
        with pytest.raises(MfnetError):
            bad()


def test_offsets_past_32_bits():
    """more elements than 2^31, as one dense tensor and as far-apart rows: the same as the rows by themselves"""
    from ssrs_amd import ops
    rows, C = 1100000, 2048
    x = torch.empty(rows, C, device="cuda", dtype=torch.bfloat16)
    x.view(-1)[:1 << 22].normal_()
    x[2048:] = x[:2048].repeat(rows // 2048 + 1, 1)[:rows - 2048]
    x[-70:] = torch.randn(70, C, device="cuda", dtype=torch.bfloat16)
    g, b = torch.rand(C, device="cuda") + 0.5, torch.randn(C, device="cuda")
    tail = x[-100:].contiguous()
    c, ct = ops.ckpt8_pack(x), ops.ckpt8_pack(tail)
    assert torch.equal(c.codes[-100:], ct.codes) and torch.equal(c.exps[-100:], ct.exps)
    assert torch.equal(ops.ckpt8_unpack(c)[-100:], ops.ckpt8_unpack(ct))
    act, cg = ops.gelu_fwd_ckpt8(x)
    act_t, cgt = ops.gelu_fwd_ckpt8(tail)
    assert torch.equal(act[-100:], act_t) and torch.equal(cg.codes[-100:], ct.codes)
    assert torch.equal(ops.gelu_bwd_ckpt8(cg, x)[-100:], ops.gelu_bwd_ckpt8(cgt, tail))
    del act, cg
    y, mean, rstd, cl = ops.layernorm_fwd_ckpt8(x, g, b, 1e-6)
    yt, mt, rt, clt = ops.layernorm_fwd_ckpt8(tail, g, b, 1e-6)
    assert torch.equal(y[-100:], yt) and torch.equal(mean[-100:], mt) and torch.equal(cl.codes[-100:], clt.codes)
    dx = ops.layernorm_bwd_ckpt8(y, cl, mean, rstd, g, want_f32=False, want_bf16=True)
    assert torch.equal(dx[-100:], ops.layernorm_bwd_ckpt8(yt, clt, mt, rt, g, want_f32=False, want_bf16=True))
    del x, y, dx, cl, c
    far = torch.empty(40000, 65541, device="cuda", dtype=torch.bfloat16)      # (rows at odd addresses: an element per lane)
    for width in (96, 77):
        v = far[:, 5:5 + width]
        v.copy_(torch.randn(40000, width, device="cuda"))
        a, b = ops.ckpt8_pack(v), ops.ckpt8_pack(v.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.exps, b.exps)
