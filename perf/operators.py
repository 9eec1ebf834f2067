"""The pooled low-rank adapters and the 8-bit activation checkpoints, as a user's program calls them.

Five operators, each in a plain form (elementary torch operations in 32 bits, `own = False`) and as the framework's own calls
(`own = True`):

  lora_serve   out = x W^T + bias + s_i (x A_i^T) B_i^T, the adapter i of every row given by an index of its own
  lora_train   the same with its backward pass: dx, and dA / dB of every adapter; `ckpt` keeps x in 8 bits for dA
  ckpt8        a tensor into the 8-bit checkpoint and back
  layernorm    LayerNorm with its input kept in 8 bits, forward and backward
  gelu         GELU with its input kept in 8 bits, forward and backward

The 8-bit checkpoint of a row: blocks of 32 consecutive elements (the last one may be shorter); with amax the largest magnitude of a
block, e is the smallest integer in [-126, 121] with amax <= 127 * 2^e (121 if none), an element is held as the whole number
rint(x / 2^e) in [-127, 127] and stands for that number times 2^e.
"""
import math
import random

import torch

own = False

EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # sixteen rows of as many requests, an adapter each, through a qkv projection: latency alone
        dict(name="serve_16_rows", op="lora_serve", rows=16, requests=16, adapters=16, K=768, N=2304, rank=8, order="mixed"),
        # requests of ragged lengths over 24 adapters of rank 16, rows of other models' requests between them (index -1), row count odd
        dict(name="serve_ragged", op="lora_serve", rows=3907, requests=61, adapters=24, K=1024, N=4096, rank=16, order="runs"),
        # 4 pairs of 1024 x 1024 tiles (4096 tokens each) of eight fine-tunes through the widest encoder's first MLP layer
        dict(name="serve_large", op="lora_serve", rows=32768, requests=8, adapters=8, K=1280, N=5120, rank=16, order="runs"),
        # two small tiles of two jobs, inputs kept in bf16; odd row count and rank
        dict(name="train_small", op="lora_train", rows=509, requests=2, adapters=2, K=768, N=768, rank=5, order="runs", ckpt=False),
        # 16 pairs of 256 x 256 tiles of eight jobs through the qkv projection, inputs kept in 8 bits
        dict(name="train_tiles", op="lora_train", rows=8192, requests=32, adapters=8, K=768, N=2304, rank=8, order="runs", ckpt=True),
        # 4 pairs of 1024 x 1024 tiles through the widest encoder's qkv projection, inputs kept in 8 bits
        dict(name="train_large", op="lora_train", rows=32768, requests=8, adapters=8, K=1280, N=3840, rank=16, order="runs", ckpt=True),
        # an odd-sized fp32 map: rows that end inside a block
        dict(name="ckpt8_odd", op="ckpt8", rows=977, C=1003, dtype="f32"),
        # the MLP's hidden activations of 4 pairs of 1024 x 1024 tiles
        dict(name="ckpt8_large", op="ckpt8", rows=32768, C=5120, dtype="bf16"),
        # one pair of 256 x 256 tiles
        dict(name="layernorm_small", op="layernorm", rows=512, C=768),
        # 4 pairs of 1024 x 1024 tiles in the widest encoder
        dict(name="layernorm_large", op="layernorm", rows=32768, C=1280),
        # one tile, hidden width of the middle encoder
        dict(name="gelu_small", op="gelu", rows=256, C=4096, dtype="bf16"),
        # 4 pairs of 1024 x 1024 tiles, hidden width of the widest encoder
        dict(name="gelu_large", op="gelu", rows=32768, C=5120, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["lora_serve", "lora_serve", "lora_train", "lora_train", "ckpt8", "layernorm", "gelu"])
    rows = _log_int(rng, 1, 24000)
    if op in ("lora_serve", "lora_train"):
        c = dict(op=op, rows=rows, requests=rng.randint(1, min(rows, 96)), adapters=_log_int(rng, 1, 48), K=8 * _log_int(rng, 8, 160),
                 N=8 * _log_int(rng, 8, 480), rank=_log_int(rng, 1, 32), order=rng.choice(["runs", "runs", "mixed"]))
        if op == "lora_train":
            c["ckpt"] = rng.random() < 0.6
        return c
    if op == "layernorm":
        return dict(op=op, rows=rows, C=32 * _log_int(rng, 1, 40))
    return dict(op=op, rows=rows, C=_log_int(rng, 1, 5120), dtype=rng.choice(["f32", "bf16"]))


# ----------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 12345)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, C):
    """tokens as a ViT block sees them: channels of different spread, a few of them far larger than the rest"""
    gain = torch.exp(0.5 * _randn(g, C))
    gain[torch.randint(0, C, (1 + C // 256,), generator=g, device="cuda")] *= 12.0
    return _randn(g, rows, C) * gain + 0.2 * _randn(g, C)


def _row_ids(g, case):
    """int32 adapter index of every row: runs of ragged lengths (or, "mixed", row by row), about one request in twelve without one"""
    rows, n = case["rows"], case["adapters"]
    k = rows if case["order"] == "mixed" else case["requests"]
    ids = torch.randint(0, n, (k,), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.rand(k, generator=g, device="cuda") < 1 / 12] = -1
    if case["order"] == "mixed":
        return ids
    cuts = torch.randint(0, rows + 1, (k - 1,), generator=g, device="cuda").sort().values
    return ids[torch.searchsorted(cuts, torch.arange(rows, device="cuda"), right=True)].contiguous()


def _inputs(case, seed):
    g = _gen(seed)
    bf = torch.bfloat16
    if case["op"] in ("lora_serve", "lora_train"):
        rows, n, K, N, r = case["rows"], case["adapters"], case["K"], case["N"], case["rank"]
        s = dict(x=_activations(g, rows, K).to(bf), w=(_randn(g, N, K) / math.sqrt(K)).to(bf), bias=0.1 * _randn(g, N),
                 A=(_randn(g, n, r, K) / math.sqrt(K)).to(bf), B=(0.1 * _randn(g, n, N, r)).to(bf),
                 scale=(0.5 + torch.rand(n, generator=g, device="cuda")), ids=_row_ids(g, case))
        if case["op"] == "lora_train":
            s["dy"] = (0.01 * _randn(g, rows, N)).to(bf)
            s["w_t"] = s["w"].t().contiguous()          # operand of the gradient product: the shared weight is frozen
        return s
    rows, C = case["rows"], case["C"]
    dt = torch.float32 if case.get("dtype", "f32") == "f32" else bf
    s = dict(x=_activations(g, rows, C).to(dt))
    if case["op"] == "layernorm":
        s.update(gamma=1.0 + 0.2 * _randn(g, C), beta=0.1 * _randn(g, C), dy=(0.01 * _randn(g, rows, C)).to(bf), dres=0.01 * _randn(g, rows, C))
    elif case["op"] == "gelu":
        s["dy"] = (0.01 * _randn(g, rows, C)).to(dt)
    return s


def prepare(case, seed):
    state = dict(case=case, t=_inputs(case, seed))
    if own and case["op"] in ("lora_serve", "lora_train"):
        from ssrs_amd import ops
        t = state["t"]
        if case["op"] == "lora_serve":
            state["pool"] = ops.lora_pool(t["A"], t["B"], t["scale"])             # the adapters' images: laid out once, served often
        else:
            state["plan"] = ops.lora_pool_plan(t["ids"], case["adapters"])        # one per batch, kept for all of its layers
    return state


# ------------------------------------------------------------------------------------------------------------- plain forms
def _ckpt_plain(x):
    """the values the 8-bit checkpoint of x [rows, C] stands for (fp32)"""
    x = x.float()
    rows, C = x.shape
    nb = -(-C // 32)
    b = torch.nn.functional.pad(x, (0, nb * 32 - C)).view(rows, nb, 32)
    u = b.abs().amax(-1, keepdim=True).view(torch.int32)
    # mantissa above that of 127 / 64 needs the next power of two
    e = ((u >> 23) - 6 + ((u & 0x7FFFFF) > 0x7E0000).to(torch.int32)).clamp(1, 248)       # exponent byte
    step = (e << 23).view(torch.float32)
    inv = ((254 - e) << 23).view(torch.float32)
    return (torch.round(b * inv).clamp(-127, 127) * step).view(rows, nb * 32)[:, :C]


def _pool_mask(ids, n, r):
    """[rows, n * r]: the rank columns that belong to the row's adapter"""
    return ids.view(-1, 1) == torch.arange(n, device=ids.device, dtype=torch.int32).repeat_interleave(r)


def _lora_fwd_plain(t):
    n, r, K = t["A"].shape
    x = t["x"].float()
    mask = _pool_mask(t["ids"], n, r)
    down = x @ t["A"].float().reshape(n * r, K).t()
    down = torch.where(mask, down * t["scale"].repeat_interleave(r), 0.0)
    up = t["B"].float().permute(0, 2, 1).reshape(n * r, -1)
    return x @ t["w"].float().t() + t["bias"] + down @ up, down, up, mask


def _lora_train_plain(t, ckpt):
    n, r, K = t["A"].shape
    out, down, up, mask = _lora_fwd_plain(t)
    dy = t["dy"].float()
    p = torch.where(mask, (dy @ up.t()) * t["scale"].repeat_interleave(r), 0.0)
    dx = dy @ t["w"].float() + p @ t["A"].float().reshape(n * r, K)
    xs = _ckpt_plain(t["x"]) if ckpt else t["x"].float()
    dA = (p.t() @ xs).view(n, r, K)
    dB = (down.t() @ dy).view(n, r, -1).permute(0, 2, 1).contiguous()
    return out.to(torch.bfloat16), dx.to(torch.bfloat16), dA, dB


def _cdf_plain(x):
    return 0.5 * torch.erfc(x * -0.7071067811865476)


def _run_plain(case, t):
    op = case["op"]
    if op == "lora_serve":
        return _lora_fwd_plain(t)[0].to(torch.bfloat16)
    if op == "lora_train":
        return _lora_train_plain(t, case["ckpt"])
    x = t["x"].float()
    if op == "ckpt8":
        return _ckpt_plain(x).to(t["x"].dtype)
    if op == "layernorm":
        mean = x.mean(-1, keepdim=True)
        rstd = torch.rsqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
        y = (x - mean) * rstd * t["gamma"] + t["beta"]
        xh = (_ckpt_plain(x) - mean) * rstd
        dy = t["dy"].float()
        g = dy * t["gamma"]
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) + t["dres"]
        return y.to(torch.bfloat16), dx, (dy * xh).sum(0), dy.sum(0)
    act = x * _cdf_plain(x)
    x8 = _ckpt_plain(x)
    dx = t["dy"].float() * (_cdf_plain(x8) + x8 * 0.3989422804014327 * torch.exp(-0.5 * x8 * x8))
    return act.to(t["x"].dtype), dx.to(t["x"].dtype)


# --------------------------------------------------------------------------------------------------- the framework's calls
def _run_own(state):
    from ssrs_amd import ops
    case, t = state["case"], state["t"]
    op = case["op"]
    if op == "lora_serve":
        return ops.lora_pool_fwd(t["x"], t["w"], t["bias"], state["pool"], t["ids"])
    if op == "lora_train":
        pool = ops.lora_pool(t["A"], t["B"], t["scale"])                          # the factors change with every step
        kept = ops.ckpt8_pack(t["x"]) if case["ckpt"] else t["x"]
        out, down = ops.lora_pool_fwd(t["x"], t["w"], t["bias"], pool, t["ids"], want_down=True)
        dx, dA, dB = ops.lora_pool_bwd(t["dy"], kept, t["w_t"], pool, state["plan"], down)
        return out, dx, dA, dB
    if op == "ckpt8":
        return ops.ckpt8_unpack(ops.ckpt8_pack(t["x"]), t["x"].dtype)
    if op == "layernorm":
        y, mean, rstd, kept = ops.layernorm_fwd_ckpt8(t["x"], t["gamma"], t["beta"], EPS)
        dx, dgamma, dbeta = ops.layernorm_bwd_ckpt8(t["dy"], kept, mean, rstd, t["gamma"], dres=t["dres"], want_weights=True)
        return y, dx, dgamma, dbeta
    act, kept = ops.gelu_fwd_ckpt8(t["x"])
    return act, ops.gelu_bwd_ckpt8(kept, t["dy"])


def run(state):
    return _run_own(state) if own else _run_plain(state["case"], state["t"])


# ---------------------------------------------------------------------------------------------------------- work and truth
def work(case):
    op, m = case["op"], case["rows"]
    if op in ("lora_serve", "lora_train"):
        n, K, N, r = case["adapters"], case["K"], case["N"], case["rank"]
        fwd_bytes = 2 * (m * K + N * K + m * N + n * r * (K + N)) + 4 * (N + n + m)
        fwd_flops = 2 * m * N * K + 2 * m * r * (K + N)
        if op == "lora_serve":
            return {"bytes": fwd_bytes, "flops": fwd_flops}
        # backward: dy, the kept x, the transposed weight and the factors once, dx and the gradients once
        bwd_bytes = 2 * (m * N + m * K + N * K + n * r * (K + N)) + (m * K * 33 // 32 if case["ckpt"] else 2 * m * K) + 4 * n * r * (K + N)
        return {"bytes": fwd_bytes + bwd_bytes, "flops": 2 * fwd_flops + 2 * m * r * (K + N)}
    C = case["C"]
    el = m * C
    size = 4 if case.get("dtype", "f32") == "f32" else 2
    kept = el + m * (-(-C // 32))
    if op == "ckpt8":
        return {"bytes": 2 * (el * size + kept), "flops": 4 * el}
    if op == "layernorm":
        return {"bytes": el * (4 + 2 + 2 + 4 + 4) + 2 * kept + 16 * m + 16 * C, "flops": 24 * el}
    return {"bytes": 4 * el * size + 2 * kept, "flops": 60 * el}


def _ckpt_exact(x):
    """the checkpoint's values from its definition, in 64 bits"""
    x = x.double()
    out = torch.empty_like(x)
    C = x.shape[1]
    full = C // 32 * 32
    for lo, hi, width in ((0, full, 32), (full, C, C - full)):
        if lo == hi:
            continue
        blk = x[:, lo:hi].reshape(x.shape[0], -1, width)
        mant, ex = torch.frexp(blk.abs().amax(-1, keepdim=True))           # amax = mant * 2^ex, mant in [1/2, 1)
        e = torch.where(mant > 127.0 / 128.0, ex - 6, ex - 7).clamp(-126, 121)
        e = torch.where(mant == 0, torch.full_like(e, -126), e)
        step = ((e.to(torch.int64) + 1023) << 52).view(torch.float64)          # 2^e by its bits: a power function rounds
        out[:, lo:hi] = (torch.round(blk / step).clamp(-127, 127) * step).reshape(x.shape[0], -1)
    return out


def exact(case, seed):
    t = {k: (v.double() if v.is_floating_point() else v) for k, v in _inputs(case, seed).items()}
    op = case["op"]
    if op in ("lora_serve", "lora_train"):
        out = t["x"] @ t["w"].t() + t["bias"]
        train = op == "lora_train"
        if train:
            dx = t["dy"] @ t["w"]
            xs = _ckpt_exact(t["x"]) if case["ckpt"] else t["x"]
            dA, dB = torch.zeros_like(t["A"]), torch.zeros_like(t["B"])
        for i in range(case["adapters"]):
            rows = (t["ids"] == i).nonzero().flatten()
            if rows.numel() == 0:
                continue
            a = t["scale"][i] * (t["x"][rows] @ t["A"][i].t())
            out[rows] += a @ t["B"][i].t()
            if train:
                p = t["scale"][i] * (t["dy"][rows] @ t["B"][i])
                dx[rows] += p @ t["A"][i]
                dA[i] = p.t() @ xs[rows]
                dB[i] = t["dy"][rows].t() @ a
        return (out, dx, dA, dB) if train else out
    x = t["x"]
    if op == "ckpt8":
        return _ckpt_exact(x)
    x8 = _ckpt_exact(x)
    if op == "layernorm":
        mean = x.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
        xh = (x8 - mean) * rstd
        g = t["dy"] * t["gamma"]
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) + t["dres"]
        return (x - mean) * rstd * t["gamma"] + t["beta"], dx, (t["dy"] * xh).sum(0), t["dy"].sum(0)
    root = 1.0 / math.sqrt(2.0)
    slope = 0.5 * torch.erfc(-x8 * root) + x8 * torch.exp(-0.5 * x8 * x8) / math.sqrt(2.0 * math.pi)
    return x * 0.5 * torch.erfc(-x * root), t["dy"] * slope
