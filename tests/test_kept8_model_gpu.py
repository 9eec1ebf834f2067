"""MMLoRA blocks that keep 8-bit activations: the forward against the usual one, the gradients against the usual backward formulas on the kept
values themselves (only roundings are left between the two)."""
import argparse
import functools

import pytest
import torch
import torch.nn as nn

from ssrs_amd import detfill

pytestmark = pytest.mark.gpu
HALF_BF16 = 2.0 ** -8
U = 2.0 ** -23


def _block(mid_dim=None, ws=14, dim=128):
    from ssrs_amd.vit import LoraBlock
    args = argparse.Namespace(mod="sam_lora", mid_dim=mid_dim, image_size=1024, multimask_output=1)
    blk = LoraBlock(args=args, dim=dim, num_heads=2, mlp_ratio=4.0, norm_layer=functools.partial(nn.LayerNorm, eps=1e-6), use_rel_pos=True,
                    window_size=ws, input_size=(64, 64))
    blk.load_state_dict(detfill.fill_state_dict(blk.state_dict(), "kept8/"))
    blk = blk.cuda()
    for name, p in blk.named_parameters():
        p.requires_grad = "lora_" in name
    return blk


@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("mid_dim", [None, 6])
def test_gelu_sees_the_sum_and_not_its_rounding(monkeypatch, kept8, mid_dim):
    """What lin2 is given is GELU of lin1's fp32 sum, rounded once, whether activations are kept in 8 bits or not (training and evaluation
    of one model agree). Bound: a bf16 rounding; GELU's slope (below 1.13) times K + 2 R fp32 additions and 2^-16 of the low-rank
    terms (their factors are split in two bf16 parts each); 2e-7 of the error function's own, on x."""
    from ssrs_amd import ops
    blk = _block(mid_dim)
    blk.checkpoint8 = kept8
    h = torch.randn(2, 2, 16, 16, 128, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    seen, gemm = [], ops.gemm

    def record(a, w, **kw):
        seen.append((a, w, kw))
        return gemm(a, w, **kw)
    monkeypatch.setattr(ops, "gemm", record)
    blk.forward_stacked(h)
    (x, w, kw), (act, w2, _) = seen[-2:]
    assert x.shape == (1024, 128) and act.shape == (1024, 512) and w2.shape == (128, 512)
    d = lambda t: t.detach().double()      # noqa: E731
    Uf, V = d(kw["U"]), d(kw["V"])
    pre = d(x) @ d(w).t() + d(kw["bias"]) + Uf @ V.t()
    size = d(x).abs() @ d(w).abs().t() + d(kw["bias"]).abs()
    lr = Uf.abs() @ V.abs().t()
    ref = 0.5 * pre * torch.erfc(-pre / 2 ** 0.5)
    tol = HALF_BF16 * ref.abs() + 1.13 * ((128 + 2 * Uf.shape[1] + 4) * U * (size + lr) + 3 * 2.0 ** -16 * lr) + 2e-7 * pre.abs()
    assert ((act.double() - ref).abs() <= tol).all()


class KeptValues:
    """Inside it, a block WITHOUT 8-bit checkpoints saves what a block with them keeps: the LayerNorm inputs and lin1's output as their
    checkpoints' values, LayerNorm outputs and GELU values made of those in 64 bits and rounded to bf16. Its backward pass is the usual
    one. Per branch the saved tensors come in the order (h, mean, rstd, LN(h), ...) and (h, mean, rstd, LN(h), GELU, lin1, ...)."""

    def __init__(self, blk):
        self.blk = blk

    def __enter__(self):
        from ssrs_amd import ops
        saved = []

        def value(t):
            return ops.ckpt8_unpack(ops.ckpt8_pack(t), torch.float32)

        def pack(t):
            i = len(saved)
            saved.append(t)
            return i

        def unpack(i):
            base, norm = (0, self.blk.norm1) if i < 8 else (8, self.blk.norm2)
            k, t = i - base, saved[i]
            if k == 0:
                return value(t)
            if k == 3:
                xh = (value(saved[base]).double() - saved[base + 1].double()[:, None]) * saved[base + 2].double()[:, None]
                return (xh * norm.weight.double() + norm.bias.double()).to(t.dtype)
            if base and k == 4:
                x = value(saved[base + 5]).double()
                return (0.5 * x * torch.erfc(-x / 2 ** 0.5)).to(t.dtype)
            if base and k == 5:
                return value(t).to(t.dtype)
            return t
        self.saved = saved
        self.hooks = torch.autograd.graph.saved_tensors_hooks(pack, unpack)
        self.hooks.__enter__()
        return self

    def __exit__(self, *exc):
        return self.hooks.__exit__(*exc)


def _l2(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


# Against that reference a gradient differs by roundings alone: the kept path rounds dGELU to bf16 before it multiplies with the slope, and
# the bf16 tensors made of it behind that (dlin1, dLN, dO, dqkv, dLN) may each fall to the other side. A bf16 rounding is at most 2^-8 and
# in a sum of squares 2^-8 / sqrt(3); seven of them: sqrt(7 / 3) 2^-8, below 2 2^-8 for a block.
ROUNDINGS = 2 * HALF_BF16
# That is relative to a gradient's norm, the norm of what it sums up. lora_wx and lora_wy are single sums of P_m . a_m over the rows m, whose
# terms cancel: their error is the sum of dP_m . a_m, in a row at most |dP_m| |a_m|, of independent rows
# with |dP| <= ROUNDINGS |P| in norm: a standard deviation of ROUNDINGS |P| |a| / sqrt(rows), of which four are allowed.


@pytest.mark.parametrize("mid_dim,ws", [(None, 14), (2, 0), (6, 14), (8, 0)])
def test_block_gradients_are_those_of_the_kept_values(monkeypatch, mid_dim, ws):
    from ssrs_amd import ops
    blk = _block(mid_dim, ws)
    mixes, mix_bwd = [], ops.lora_mix_bwd
    monkeypatch.setattr(ops, "lora_mix_bwd", lambda P, a, *w: (mixes.append((P, a)), mix_bwd(P, a, *w))[1])
    g = torch.Generator().manual_seed(3)
    h0, dh = torch.randn(2, 2, 16, 16, 128, generator=g).cuda(), torch.randn(2, 2, 16, 16, 128, generator=g).cuda()
    grads = {}
    for kept8 in (False, True):
        blk.checkpoint8 = kept8
        blk.zero_grad()
        h = h0.clone().requires_grad_()
        if kept8:
            out = blk.forward_stacked(h)
        else:
            with KeptValues(blk) as kv:
                out = blk.forward_stacked(h)
            assert len(kv.saved) == 18
        out.backward(dh)
        grads[kept8] = {"h": h.grad, **{k: p.grad for k, p in blk.named_parameters() if p.grad is not None}}
    assert set(grads[True]) == set(grads[False]) and len(grads[True]) == 17
    allowed = {}
    for lin, (P, a) in zip(("lin2", "lin1"), mixes):             # in the order of the backward pass
        for w in ("wx", "wy"):
            allowed[f"mlp.{lin}.lora_{w}"] = 4 * ROUNDINGS * (P.double().norm() * a.double().norm() / P.shape[0] ** 0.5).item()
    for k, want in grads[False].items():
        assert (grads[True][k].double() - want.double()).norm().item() < allowed.get(k, ROUNDINGS * want.double().norm().item()), (k, _l2(grads[True][k], want))


@pytest.mark.parametrize("use_graph", [False, True])
def test_step_gradients_of_every_encoder_parameter(use_graph):
    """the train step of the tiny model: each encoder parameter's slice of the flat gradient against the same step of a model without
    8-bit checkpoints that saves the kept values. Two blocks of two branches: the roundings of both, 2 ROUNDINGS; a scalar's terms
    are the other parameters' business (the block's test), here it is held to that share of the branch's largest scalar gradient."""
    import warnings
    from ssrs_amd.trainer import TrainEngine
    from ssrs_amd.unetformer_mmsam import UNetFormer
    rgb, dsm, tgt = (t.cuda() for t in detfill.tiles("kept8s", 2, 256, 6))
    grads = {}
    for kind in ("bf16", "int8"):
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            m = UNetFormer(num_classes=6, encoder="vit_tiny_test", args=argparse.Namespace(mod="sam_lora", mid_dim=None, image_size=1024, multimask_output=1), checkpoints=kind)
        m.load_state_dict(detfill.fill_state_dict(m.state_dict(), "kept8s/"))
        m = m.cuda().eval()
        m.decoder.segmentation_head[1].p = 0.0
        graph = use_graph and kind == "int8"
        if kind == "bf16":
            for blk in m.image_encoder.blocks:
                def keeps(h, blk=blk, plain=blk.forward_stacked):
                    with KeptValues(blk):
                        return plain(h)
                blk.forward_stacked = keeps
        eng = TrainEngine(m, lr=0.0, momentum=0.9, weight_decay=5e-4, class_weight=torch.ones(6, device="cuda"), use_graph=graph)
        for _ in range(4 if graph else 1):
            eng.step(rgb, dsm, tgt)
        torch.cuda.synchronize()
        grads[kind] = {k: p._mfnet_sink[0].clone() for k, p in m.image_encoder.named_parameters() if p.requires_grad}
    assert len(grads["int8"]) == 2 * 16
    for k, want in grads["bf16"].items():
        size = want.double().norm().item() if want.numel() > 1 else max(v.abs().item() for n, v in grads["bf16"].items() if v.numel() == 1 and n.split(".")[1] == k.split(".")[1])
        assert (grads["int8"][k].double() - want.double()).norm().item() < 2 * ROUNDINGS * size, (k, _l2(grads["int8"][k], want))
