"""Pooled low-rank adapters (ops.lora_pool*) against their formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23          # one step of an fp32 accumulation (matrix instructions need not round to nearest)
HALF_BF16 = 2.0 ** -8


def ops():
    from ssrs_amd import ops as o
    return o


def make(M, K, N, n, r, ids="runs", seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    x, w, dy = rn(M, K).bfloat16(), (rn(N, K) / math.sqrt(K)).bfloat16(), rn(M, N).bfloat16()
    A, B = (rn(n, r, K) / math.sqrt(K)).to(dtype), (0.3 * rn(n, N, r)).to(dtype)
    scale, bias = 0.5 + torch.rand(n, generator=g, device="cuda"), rn(N)
    if ids == "mixed":          # row by row, some without an adapter: below and above the range
        idx = torch.randint(-2, n + 2, (M,), generator=g, device="cuda", dtype=torch.int32)
    elif ids == "one":          # a single adapter's rows
        idx = torch.full((M,), n - 1, dtype=torch.int32, device="cuda")
    elif ids == "none":
        idx = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    else:                       # runs of ragged lengths, an adapter may come again
        cuts = torch.randint(0, M + 1, (max(1, min(M, 2 * n)),), generator=g, device="cuda").sort().values
        per = torch.randint(-1, n, (cuts.numel() + 1,), generator=g, device="cuda", dtype=torch.int32)
        idx = per[torch.searchsorted(cuts, torch.arange(M, device="cuda"), right=True)].contiguous()
    return dict(x=x, w=w, dy=dy, A=A, B=B, scale=scale, bias=bias, ids=idx, w_t=w.t().contiguous())


def formulas(t, x=None):
    """out, dx, dA, dB in 64 bits and a bound of each one's fp32 arithmetic. Sums of k products: k U of the sum of magnitudes; the
    fp32 factors (down, p) carry the error of theirs, and 2^-16 of their own where they enter a bf16 result split in two parts."""
    d = {k: v.double() for k, v in t.items() if k != "ids"}
    A, B = t["A"].bfloat16().double(), t["B"].bfloat16().double()        # the MFMA operands
    n, r, K = A.shape
    N = B.shape[1]
    M = t["x"].shape[0]
    xs = d["x"] if x is None else x
    out, eout = d["x"] @ d["w"].t() + d["bias"], (K + 2) * U * (d["x"].abs() @ d["w"].abs().t() + d["bias"].abs())
    dx, edx = d["dy"] @ d["w"], (N + 2) * U * (d["dy"].abs() @ d["w"].abs())
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    eA, eB = torch.zeros_like(A), torch.zeros_like(B)
    split = 2.0 ** -16
    for i in range(n):
        rows = (t["ids"] == i).nonzero().flatten()
        if not rows.numel():
            continue
        s, X, D, Xs = d["scale"][i], d["x"][rows], d["dy"][rows], xs[rows]
        a, ea = s * X @ A[i].t(), (K + 4) * U * s * X.abs() @ A[i].abs().t()
        p, ep = s * D @ B[i], (N + 4) * U * s * D.abs() @ B[i].abs()
        out[rows] += a @ B[i].t()
        eout[rows] += (ea + (split + (r + 2) * U) * a.abs()) @ B[i].abs().t()
        dx[rows] += p @ A[i]
        edx[rows] += (ep + (split + (r + 2) * U) * p.abs()) @ A[i].abs()
        k = rows.numel() + 8
        dA[i], eA[i] = p.t() @ Xs, (ep + k * U * p.abs()).t() @ Xs.abs()
        dB[i], eB[i] = D.t() @ a, D.abs().t() @ (ea + k * U * a.abs())
    return (out, dx, dA, dB), (eout, edx, eA, eB)


def close(got, ref, tol, half=0.0):
    return bool(((got.double() - ref).abs() <= tol + half * ref.abs() + 1e-30).all())


# single rows, odd and ragged sizes, ranks of every padding, widths that end inside k-tiles and column tiles, each tile shape of the product
CASES = [(1, 64, 64, 1, 1, "one"), (1, 8, 8, 3, 5, "mixed"), (2, 72, 24, 2, 4, "mixed"), (15, 768, 768, 4, 4, "mixed"), (16, 136, 264, 16, 8, "mixed"), (32, 1288, 768, 5, 64, "mixed"), (33, 264, 72, 2, 20, "runs"), (64, 776, 128, 9, 16, "mixed"), (256, 72, 200, 11, 8, "mixed"),
         (16, 1096, 200, 5, 32, "mixed"), (9, 3840, 72, 2, 20, "mixed"), (12, 264, 136, 3, 64, "mixed"), (17, 768, 2304, 70, 16, "mixed"), (128, 136, 264, 40, 16, "mixed"), (100, 72, 520, 3, 48, "runs"), (63, 128, 40, 3, 17, "runs"), (65, 1280, 128, 5, 64, "mixed"), (130, 200, 392, 24, 33, "mixed"),
         (257, 264, 520, 7, 16, "runs"), (509, 768, 768, 2, 5, "runs"), (700, 1024, 1032, 300, 8, "mixed"), (1200, 64, 1000, 3, 16, "none"),
         (3907, 520, 1160, 24, 16, "runs"), (6000, 328, 2312, 5, 16, "mixed"), (8192, 768, 2304, 8, 8, "runs"), (4000, 1096, 4104, 6, 16, "mixed"), (33000, 24, 520, 3, 16, "mixed"), (4100, 64, 4096, 3, 40, "runs"), (3800, 136, 4000, 4, 20, "mixed"), (16900, 72, 776, 3, 12, "runs"),
         (100, 264, 4104, 3, 16, "mixed"), (192, 776, 2312, 3, 32, "runs"), (1024, 264, 136, 9, 20, "mixed"), (1025, 264, 136, 9, 20, "mixed"), (1030, 1288, 264, 20, 64, "mixed"), (16, 1288, 72, 3, 16, "mixed"), (3, 2568, 72, 2, 9, "mixed"), (1, 5120, 136, 2, 32, "one"), (512, 264, 776, 3, 40, "one"), (512, 72, 136, 2, 5, "one"), (513, 72, 136, 2, 5, "one"), (400, 520, 72, 20, 20, "mixed")]


@pytest.mark.parametrize("M,K,N,n,r,ids", CASES)
def test_forward_and_backward(M, K, N, n, r, ids):
    o = ops()
    t = make(M, K, N, n, r, ids)
    pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(t["ids"], n)
    out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
    out32 = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], out_dtype=torch.float32)
    dx, dA, dB = o.lora_pool_bwd(t["dy"], t["x"], t["w_t"], pool, plan, down)
    ref, tol = formulas(t)
    assert close(out, ref[0], tol[0], HALF_BF16) and close(out32, ref[0], tol[0])
    assert close(dx, ref[1], tol[1], HALF_BF16)
    assert dA.dtype == dB.dtype == torch.float32 and dA.shape == t["A"].shape and dB.shape == t["B"].shape
    assert close(dA, ref[2], tol[2]) and close(dB, ref[3], tol[3])
    # again: the same bits; and without dx
    assert all(torch.equal(a, b) for a, b in zip((dx, dA, dB), o.lora_pool_bwd(t["dy"], t["x"], t["w_t"], pool, plan, down)))
    none, dA2, dB2 = o.lora_pool_bwd(t["dy"], t["x"], None, pool, plan, down, want_dx=False)
    assert none is None and torch.equal(dA2, dA) and torch.equal(dB2, dB)
    # the input kept in 8 bits: dA sums what the checkpoint stands for, the rest does not change
    kept = o.ckpt8_pack(t["x"])
    dx8, dA8, dB8 = o.lora_pool_bwd(t["dy"], kept, t["w_t"], pool, plan, down)
    ref8, tol8 = formulas(t, o.ckpt8_unpack(kept, torch.float32).double())
    assert torch.equal(dx8, dx) and torch.equal(dB8, dB) and close(dA8, ref8[2], tol8[2])


def test_rows_without_an_adapter_take_the_projection_alone():
    o = ops()
    t = make(300, 128, 136, 4, 8, "mixed")
    pool = o.lora_pool(t["A"], t["B"], t["scale"])
    out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
    off = (t["ids"] < 0) | (t["ids"] >= 4)
    assert off.any() and (down[off] == 0).all()
    plain = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, torch.full_like(t["ids"], -1))
    assert torch.equal(out[off], plain[off])
    nobias = o.lora_pool_fwd(t["x"], t["w"], None, pool, t["ids"], out_dtype=torch.float32)
    ref = formulas(dict(t, bias=torch.zeros_like(t["bias"])))
    assert close(nobias, ref[0][0], ref[1][0])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("M,K,N", [(40, 128, 136), (700, 256, 264), (6000, 136, 2312)])
def test_one_requests_nonfinite_values_stay_its_own(M, K, N, bad):
    """an adapter with infinities or NaN, and rows that hold them, change nothing for the other requests' rows and gradients"""
    o = ops()
    t = make(M, K, N, 3, 8, "mixed", seed=5)
    ids = t["ids"]

    def run(t):
        pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(ids, 3)
        out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, ids, want_down=True)
        return (out, down) + o.lora_pool_bwd(t["dy"], t["x"], t["w_t"], pool, plan, down)
    clean = run(t)
    for what in ("A", "B", "x", "dy"):
        s = dict(t)
        s[what] = t[what].clone()
        if what in ("A", "B"):
            s[what][1] = bad
        else:
            s[what][ids == 1] = bad
        got = run(s)
        ok = ids != 1
        assert torch.equal(got[0][ok], clean[0][ok]) and torch.equal(got[1][ok], clean[1][ok]) and torch.equal(got[2][ok], clean[2][ok]), what
        for i in (0, 2):
            assert torch.equal(got[3][i], clean[3][i]) and torch.equal(got[4][i], clean[4][i]), what
        assert not torch.isfinite(got[0][ids == 1].float()).all() or what == "dy"


def test_layouts_and_types():
    """row strides, column slices, transposed and misaligned views; fp32 factors (rounded once to bf16); default scale"""
    o = ops()
    t = make(130, 128, 72, 3, 8, "runs", seed=3, dtype=torch.float32)
    pool = o.lora_pool(t["A"], t["B"], t["scale"])
    ref = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"])
    assert torch.equal(ref, o.lora_pool_fwd(t["x"], t["w"], t["bias"], o.lora_pool(t["A"].bfloat16(), t["B"].bfloat16(), t["scale"]), t["ids"]))
    r64, tol = formulas(t)
    assert close(ref, r64[0], tol[0], HALF_BF16)
    wide = torch.randn(130, 300, device="cuda").bfloat16()
    for lo in (0, 8, 3):                                     # 3: rows not 16-byte aligned
        v = wide[:, lo:lo + 128]
        v.copy_(t["x"])
        assert torch.equal(o.lora_pool_fwd(v, t["w"], t["bias"], pool, t["ids"]), ref)
    xt = t["x"].t().contiguous().t()
    big_w = torch.zeros(72, 160, device="cuda", dtype=torch.bfloat16)
    big_w[:, :128] = t["w"]
    bias = torch.zeros(73, device="cuda")[1:]
    bias.copy_(t["bias"])
    assert torch.equal(o.lora_pool_fwd(xt, big_w[:, :128], bias, pool, t["ids"]), ref)
    plan = o.lora_pool_plan(t["ids"], 3)
    down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)[1]
    a = o.lora_pool_bwd(t["dy"], t["x"], t["w_t"], pool, plan, down)
    b = o.lora_pool_bwd(t["dy"].t().contiguous().t(), wide[:, 3:131], t["w"].t(), pool, plan, down)
    wide[:, 3:131].copy_(t["x"])
    b = o.lora_pool_bwd(t["dy"].t().contiguous().t(), wide[:, 3:131], t["w"].t(), pool, plan, down)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    ones = o.lora_pool_fwd(t["x"], t["w"], t["bias"], o.lora_pool(t["A"], t["B"]), t["ids"])
    assert torch.equal(ones, o.lora_pool_fwd(t["x"], t["w"], t["bias"], o.lora_pool(t["A"], t["B"], torch.ones(3, device="cuda")), t["ids"]))


def test_no_rows():
    o = ops()
    t = make(0, 64, 72, 2, 4, "none")
    pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(t["ids"], 2)
    out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
    dx, dA, dB = o.lora_pool_bwd(t["dy"], t["x"], t["w_t"], pool, plan, down)
    assert out.shape == (0, 72) and dx.shape == (0, 64) and (dA == 0).all() and (dB == 0).all() and dA.shape == (2, 4, 64)


def test_plan_groups_every_row():
    o = ops()
    for M, n in ((1, 1), (255, 3), (257, 300), (5000, 7), (40000, 2)):
        ids = torch.randint(-1, n + 1, (M,), device="cuda", dtype=torch.int32)
        p = o.lora_pool_plan(ids, n)
        offs, perm = p.offs.tolist(), p.perm
        for i in {0, n // 2, n - 1}:
            assert torch.equal(perm[offs[i]:offs[i + 1]].long(), (ids == i).nonzero().flatten())
        assert offs[0] == 0 and offs[n] == int(((ids >= 0) & (ids < n)).sum())
        table = [e for e in p.table.tolist() if e[0] >= 0]
        assert sum(e[2] - e[1] for e in table) == offs[n] and len(table) == p.base.tolist()[n]


def test_streams_and_graph_replays():
    """on another stream; captured with its plan and pool, replayed on new rows, indices and factors between eager calls"""
    o = ops()
    t = make(600, 256, 264, 4, 8, "mixed")

    def step(t):
        pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(t["ids"], 4)
        out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
        return (out,) + o.lora_pool_bwd(t["dy"], o.ckpt8_pack(t["x"]), t["w_t"], pool, plan, down)
    ref = step(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(t)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    st = {k: v.clone() for k, v in t.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out = step(st)
    for k in range(3):
        for key, v in make(600, 256, 264, 4, 8, ("runs", "one", "mixed")[k], seed=50 + k).items():
            st[key].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        ref = step(st)
        assert all(torch.equal(a, b) for a, b in zip(ref, out)), k


def test_refusals():
    o = ops()
    from ssrs_amd._lib import MfnetError
    t = make(40, 64, 72, 2, 4)
    pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(t["ids"], 2)
    out, down = o.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
    f, b = o.lora_pool_fwd, o.lora_pool_bwd
    for bad in (lambda: o.lora_pool(t["A"], t["B"][:1]), lambda: o.lora_pool(t["A"][:, :3], t["B"]), lambda: o.lora_pool(t["A"].half(), t["B"].half()), lambda: o.lora_pool(t["A"].float(), t["B"]),
                lambda: o.lora_pool(t["A"][:, :, :60], t["B"]), lambda: o.lora_pool(t["A"], t["B"], t["scale"][:1]), lambda: o.lora_pool(t["A"].cpu(), t["B"]),
                lambda: o.lora_pool(torch.zeros(1, 65, 64, device="cuda"), torch.zeros(1, 64, 65, device="cuda")),
                lambda: o.lora_pool_plan(t["ids"].long(), 2), lambda: o.lora_pool_plan(t["ids"], 0), lambda: o.lora_pool_plan(t["ids"].view(2, 20), 2),
                lambda: f(t["x"][0], t["w"], t["bias"], pool, t["ids"]), lambda: f(t["x"].float(), t["w"], t["bias"], pool, t["ids"]), lambda: f(t["x"][:, :56], t["w"], t["bias"], pool, t["ids"]),
                lambda: f(t["x"], t["w"].t(), t["bias"], pool, t["ids"]), lambda: f(t["x"], t["w"], t["bias"][:64], pool, t["ids"]),
                lambda: f(t["x"], t["w"], t["bias"], pool, t["ids"][:39]), lambda: f(t["x"], t["w"], t["bias"], pool, t["ids"].long()),
                lambda: f(t["x"], t["w"], t["bias"], pool, t["ids"], out_dtype=torch.float16), lambda: f(t["x"].cpu(), t["w"], t["bias"], pool, t["ids"]),
                lambda: b(t["dy"][:39], t["x"], t["w_t"], pool, plan, down), lambda: b(t["dy"], t["x"][:39], t["w_t"], pool, plan, down),
                lambda: b(t["dy"], t["x"], t["w"], pool, plan, down), lambda: b(t["dy"], t["x"], None, pool, plan, down),
                lambda: b(t["dy"], t["x"], t["w_t"], pool, plan, down[:, :8]), lambda: b(t["dy"], t["x"], t["w_t"], pool, o.lora_pool_plan(t["ids"], 3), down),
                lambda: b(t["dy"], o.ckpt8_pack(t["x"][:39]), t["w_t"], pool, plan, down), lambda: b(t["dy"].float(), t["x"], t["w_t"], pool, plan, down)):
        with pytest.raises(MfnetError):
            bad()


def test_copied_and_stored_pools():
    """a copy and a stored pool hold addresses of their own buffer, not of the one they were made from"""
    import copy
    import io
    import pickle
    from ssrs_amd import ops
    g = torch.Generator().manual_seed(0)
    A, B = torch.randn(3, 5, 72, generator=g).cuda(), torch.randn(3, 40, 5, generator=g).cuda()
    x, w = torch.randn(33, 72, generator=g).bfloat16().cuda(), torch.randn(40, 72, generator=g).bfloat16().cuda()
    ids = torch.randint(-1, 3, (33,), generator=g, dtype=torch.int32).cuda()
    pool = ops.lora_pool(A, B, torch.tensor([0.5, 1.0, 2.0], device="cuda"))
    want = ops.lora_pool_fwd(x, w, None, pool, ids)
    stored = io.BytesIO()
    torch.save(pool, stored)
    stored.seek(0)
    others = [copy.deepcopy(pool), pickle.loads(pickle.dumps(pool)), torch.load(stored, weights_only=False)]
    for other in others:
        assert other.a_down == other.buf.data_ptr() != pool.a_down and other.scale - other.a_down == pool.scale - pool.a_down
    pool.buf.fill_(float("nan"))                                 # (nothing may read it any more)
    for other in others:
        assert torch.equal(ops.lora_pool_fwd(x, w, None, other, ids), want)


def test_offsets_past_32_bits():
    """rows whose byte or element offsets pass 32 bits: far-apart rows of x, dy and w, and more output elements than 2^31"""
    o = ops()
    t = make(40000, 64, 72, 3, 8, "mixed", seed=2)
    far = torch.empty(40000, 65544, device="cuda", dtype=torch.bfloat16)
    x, dy = far[:, 8:72], far[:, 128:200]
    x.copy_(t["x"])
    dy.copy_(t["dy"])
    w = torch.empty(72, (1 << 22) + 8, device="cuda", dtype=torch.bfloat16)[:, :64]
    w.copy_(t["w"])
    pool, plan = o.lora_pool(t["A"], t["B"], t["scale"]), o.lora_pool_plan(t["ids"], 3)

    def run(x, w, dy):
        out, down = o.lora_pool_fwd(x, w, t["bias"], pool, t["ids"], want_down=True)
        return (out, down) + o.lora_pool_bwd(dy, x, t["w_t"], pool, plan, down)
    ref, tol = formulas(t)
    for got in (run(x, t["w"], dy), run(x, w, dy)):
        assert close(got[0], ref[0], tol[0], HALF_BF16) and close(got[2], ref[1], tol[1], HALF_BF16) and close(got[3], ref[2], tol[2]) and close(got[4], ref[3], tol[3])
    del far, x, dy, w
    t = make(3000, 1280, 5120, 3, 8, "mixed", seed=4)            # the largest tile, rows as far apart as it takes and a little further
    pool = o.lora_pool(t["A"], t["B"], t["scale"])
    ref, tol = formulas(t)
    for ld in (1 << 22, (1 << 22) + 8):
        x = torch.empty(3000, ld, device="cuda", dtype=torch.bfloat16)[:, -1280:]
        x.copy_(t["x"])
        assert close(o.lora_pool_fwd(x, t["w"], t["bias"], pool, t["ids"]), ref[0], tol[0], HALF_BF16), ld
        del x
    M, N = 300000, 8192
    t = make(M, 64, N, 2, 4, "mixed", seed=3)
    out = o.lora_pool_fwd(t["x"], t["w"], t["bias"], o.lora_pool(t["A"], t["B"], t["scale"]), t["ids"])
    for rows in (slice(0, 64), slice(M - 100, M)):
        part = {k: (v[rows] if k in ("x", "dy", "ids") else v) for k, v in t.items()}
        ref, tol = formulas(part)
        assert close(out[rows], ref[0], tol[0], HALF_BF16), rows
