"""fp32 mode: the depthwise convolutions' weight gradients have the same bits in every run."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,k,ext,collected", [(2, 16, 8, True, False), (2, 64, 8, True, True), (2, 64, 3, False, False), (3, 20, 3, True, True), (1, 130, 5, False, False)])
def test_depthwise_weight_gradient_repeats(B, S, k, ext, collected):
    from ssrs_amd import ops
    g = torch.Generator().manual_seed(1)
    dy, x, w = (torch.randn(*s, generator=g).cuda() for s in ((B * S * S, 64), (B * S * S, 64), (64, k * k)))
    first = None
    with ops.precision("fp32"):
        for _ in range(6):
            if collected:
                ops.TN_QUEUE = []
            try:
                _, dw, db = ops.dwconv_bwd(dy, x, w, B, S, S, k, ext, want_bias=True)
                got = dw.materialize(), db.materialize()
            finally:
                ops.TN_QUEUE = None
            first = first or got
            assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    ref = ops.dwconv_bwd(dy, x, w, B, S, S, k, ext, want_bias=True)      # fewer copies: another order of the same sums
    # every addition rounds by at most 2^-24 of a partial sum: B S^2 + copies of them on terms of size |dy| |x|
    for a, b, terms in ((first[0], ref[1].materialize(), (dy.abs().max() * x.abs().max()).item()), (first[1], ref[2].materialize(), dy.abs().max().item())):
        assert (a - b).abs().max().item() <= 2 * B * S * S * terms * 2.0 ** -24 * 4
