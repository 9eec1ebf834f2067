"""Column reductions write their outputs and their workspace and nothing beside them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
MARK = 12345.0


def _guarded(n, fill):
    """n floats inside a larger tensor whose other elements hold a mark"""
    t = torch.full((n + 8192,), MARK, device="cuda")
    t[4096:4096 + n] = fill
    return t, t[4096:4096 + n]


def _untouched(t, n):
    return bool((t[:4096] == MARK).all()) and bool((t[4096 + n:] == MARK).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [12, 512, 516, 768, 1000, 1020, 1024])
def test_sums_and_weight_gradients_stay_inside(C, dtype):
    """two sums per column (sum and sum of squares; LayerNorm's dbeta and dgamma): widths of one pass, of whole passes and of a last
    pass that is not full"""
    from ssrs_amd import _lib, ops
    P = 700
    g = torch.Generator().manual_seed(C)
    x, dy = (torch.randn(P, C, generator=g).to(dtype).cuda() for _ in range(2))
    mean, rstd = x.float().mean(-1), torch.rsqrt(x.float().var(-1, unbiased=False) + 1e-6)
    n = int(_lib.lib().mfnet_colreduce_workspace_floats(1, P, C))
    st = torch.cuda.current_stream().cuda_stream
    dt = ops._DT[dtype]
    for kind in ("sums", "layernorm"):
        (a, out0), (b, out1), (w, ws) = _guarded(C, 0.0), _guarded(C, 0.0), _guarded(n, 0.0)
        tickets = torch.zeros(1, dtype=torch.int32, device="cuda")
        if kind == "sums":
            ops.call("mfnet_colsum", x.data_ptr(), dt, out0.data_ptr(), out1.data_ptr(), 1, P, C, ws.data_ptr(), tickets.data_ptr(), st)
            ref0, ref1 = x.double().sum(0), (x.double() ** 2).sum(0)
            size0, size1 = x.double().abs().sum(0), ref1
        else:
            ops.call("mfnet_layernorm_bwd_weights", dy.data_ptr(), dt, x.data_ptr(), dt, mean.data_ptr(), rstd.data_ptr(), out1.data_ptr(), out0.data_ptr(), P, C,
                     ws.data_ptr(), tickets.data_ptr(), st)
            xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
            ref0, ref1 = dy.double().sum(0), (dy.double() * xh).sum(0)
            size0, size1 = dy.double().abs().sum(0), (dy.double() * xh).abs().sum(0)
        torch.cuda.synchronize()
        assert _untouched(a, C) and _untouched(b, C) and _untouched(w, n), kind
        # every addition rounds by 2^-24 of a partial sum: at most P of them, and a few roundings per term
        assert ((out0.double() - ref0).abs() <= (P + 8) * 2.0 ** -24 * size0).all() and ((out1.double() - ref1).abs() <= (P + 8) * 2.0 ** -24 * size1 + 4 * 2.0 ** -24 * size1).all(), kind
