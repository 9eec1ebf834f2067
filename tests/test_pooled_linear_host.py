"""lora.PooledLinear before any launch (no GPU): the pool made of fine-tuned layers."""
import pytest
import torch


def _merged(g, alpha, first=None, bias=True, r=4):
    from ssrs_amd.medsam.models.common import loralib as lora
    m = lora.MergedLinear(64, 192, r=r, lora_alpha=alpha, enable_lora=[True, False, True], bias=bias)
    with torch.no_grad():
        for p in (m.lora_Ax, m.lora_Ay, m.lora_Bx, m.lora_By):
            p.copy_(torch.randn(p.shape, generator=g))
        if first is not None:
            m.weight.copy_(first.weight)
            if bias:
                m.bias.copy_(first.bias)
    return m


def _update(m, A, B):
    """a layer's low-rank update of its [3 D, in] weight (q and v thirds), from its definition in 64 bits"""
    r, D = m.r, m.out_features // 3
    dw = torch.zeros(3 * D, m.in_features, dtype=torch.float64)
    dw[:D] = m.scaling * B[:D].double() @ A[:r].double()
    dw[2 * D:] = m.scaling * B[D:].double() @ A[r:].double()
    return dw.detach()


def test_pool_of_layers_keeps_each_layers_scaling():
    from ssrs_amd.medsam.models.common import loralib as lora
    g = torch.Generator().manual_seed(0)
    layers = [_merged(g, 1)]
    layers += [_merged(g, alpha, layers[0]) for alpha in (16, 3)]
    pool = lora.PooledLinear.from_merged(layers)
    assert pool.scaling.tolist() == [0.25, 0.25, 4.0, 4.0, 0.75, 0.75]
    for i, m in enumerate(layers):
        for j, (A, B) in enumerate(((m.lora_Ax, m.lora_Bx), (m.lora_Ay, m.lora_By))):
            k = 2 * i + j
            got = pool.scaling[k].double() * pool.lora_B[k].double() @ pool.lora_A[k].double()
            assert torch.allclose(got.detach(), _update(m, A, B), rtol=1e-12, atol=1e-12), k


def test_pool_of_layers_without_a_bias():
    """no layer has a bias: the pool has none; some have one: refused like any other difference of the shared projection"""
    from ssrs_amd.medsam.models.common import loralib as lora
    g = torch.Generator().manual_seed(1)
    layers = [_merged(g, 1, bias=False)]
    layers.append(_merged(g, 1, layers[0], bias=False))
    pool = lora.PooledLinear.from_merged(layers)
    assert pool.bias is None and torch.equal(pool.weight, layers[0].weight) and torch.equal(pool.lora_A[3], layers[1].lora_Ay)
    with_bias = _merged(g, 1)
    with torch.no_grad():
        with_bias.weight.copy_(layers[0].weight)
    for mixed in ([layers[0], with_bias], [with_bias, layers[0]]):
        with pytest.raises(ValueError, match="bias"):
            lora.PooledLinear.from_merged(mixed)


def test_cast_of_nothing():
    """a batch without rows has no address"""
    from ssrs_amd import _lib
    L = _lib.lib()
    assert L.mfnet_cast(None, 0, None, 1, 0, None) == 0
    assert L.mfnet_cast(None, 0, None, 1, 8, None) == -1 and b"null" in L.mfnet_last_error()
    assert L.mfnet_cast(None, 0, None, 1, 4, None) == -1 and b"multiple" in L.mfnet_last_error()


def test_import_with_a_torch_that_has_no_gpu_backend():
    """ops is imported by code that runs on the host alone (state dicts, plans of rasters); only calls need the GPU backend"""
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    delattr(torch._C, n)\n"
            "from ssrs_amd import ops\n"
            "from ssrs_amd.vit import PooledLinear\n"
            "PooledLinear(64, 64, 2, 4)\n"
            "try:\n"
            "    ops.ckpt8_pack(torch.zeros(4, 64))\n"
            "except ops.MfnetError as e:\n"
            "    assert 'CPU tensor' in str(e)\n"
            "else:\n"
            "    raise SystemExit(1)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
