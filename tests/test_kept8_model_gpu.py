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
