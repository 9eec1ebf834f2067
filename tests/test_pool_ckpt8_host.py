"""Refusals of the pooled-adapter and 8-bit-checkpoint entry points before any launch (no GPU), and their host-side sizes."""
import pytest
import torch


def _L():
    from ssrs_amd import _lib
    return _lib.lib()


def test_entry_points_refuse_bad_arguments_before_a_launch():
    L = _L()
    E = L.mfnet_last_error
    assert L.mfnet_ckpt8_pack(None, 0, 64, 16, 16, 4, 64, None) == -1 and b"null" in E()
    assert L.mfnet_ckpt8_pack(16, 2, 64, 16, 16, 4, 64, None) == -1 and b"dtype" in E()
    assert L.mfnet_ckpt8_pack(16, 0, 63, 16, 16, 4, 64, None) == -1 and b"stride" in E()
    assert L.mfnet_ckpt8_pack(18, 0, 64, 16, 16, 4, 64, None) == -1 and b"misaligned" in E()
    assert L.mfnet_ckpt8_pack(16, 0, 64, 16, 16, -1, 64, None) == -1 and b"shape" in E()
    assert L.mfnet_ckpt8_pack(16, 0, 64, 16, 16, 1 << 39, 64, None) == -1 and b"shape" in E()
    assert L.mfnet_ckpt8_pack(None, 0, 64, None, None, 0, 64, None) == 0                    # no rows: nothing to do
    assert L.mfnet_gelu_fwd_ckpt8(16, 1, 64, None, 64, 16, 16, 4, 64, None) == -1 and b"null" in E()
    assert L.mfnet_gelu_bwd_ckpt8(16, 16, None, 1, 64, 16, None, 64, 4, 64, None) == -1 and b"null" in E()
    assert L.mfnet_layernorm_fwd_ckpt8(16, 0, 48, 16, 16, 16, 16, 16, 16, 16, 4, 48, 1e-6, None) == -1 and b"multiple of 32" in E()
    assert L.mfnet_layernorm_fwd_ckpt8(16, 0, 2080, 16, 16, 16, 16, 16, 16, 16, 4, 2080, 1e-6, None) == -1
    bwd = [16, 1, 64, 16, 16, 16, 16, 16, None, None, 16, None, None, None, None, None, 0, 4, 64, None]
    for k, v, msg in ((13, 16, b"go together"), (10, None, b"null"), (12, 16, b"beta"), (2, 62, b"lddy")):
        a = list(bwd)
        a[k] = v
        assert L.mfnet_layernorm_bwd_ckpt8(*a) == -1 and msg in E(), msg
    a = list(bwd)
    a[13] = a[14] = 16
    assert L.mfnet_layernorm_bwd_ckpt8(*a) == -1 and b"workspace" in E()
    assert L.mfnet_lora_pool_pack(16, 0, 0, 2, 64, 20, 16, 16, 16, None) == -1 and b"sizes" in E()
    assert L.mfnet_lora_pool_pack(16, 0, 0, 2, 60, 4, 16, 16, 16, None) == -1
    assert L.mfnet_lora_pool_pack(16, 0, 0, 2, 64, 4, 24, 16, 16, None) == -1
    assert L.mfnet_lora_pool_plan(16, 1 << 31, 2, 16, 16, 16, 16, None) == -1 and b"sizes" in E()
    assert L.mfnet_lora_pool_plan(None, 8, 2, 16, 16, 16, 16, None) == -1 and b"null" in E()
    assert L.mfnet_lora_pool_down(16, 60, 16, 16, 16, 2, 16, 16, 8, 64, None) == -1 and b"stride" in E()
    assert L.mfnet_lora_pool_down(16, 64, 16, 16, 16, 2, 17, 16, 8, 64, None) == -1 and b"sizes" in E()
    assert L.mfnet_lora_pool_gemm(16, 64, 16, 64, None, 16, None, None, 2, 16, 16, 1, 64, 8, 64, 64, None) == -1 and b"null" in E()
    assert L.mfnet_lora_pool_gemm(16, 64, 24, 64, None, None, None, None, 0, 0, 16, 1, 64, 8, 64, 64, None) == -1 and b"weight" in E()
    assert L.mfnet_lora_pool_gemm(16, 64, 16, 64, None, None, None, None, 0, 0, 16, 1, 64, 8, 60, 64, None) == -1 and b"out" in E()
    assert L.mfnet_lora_pool_tn(16, 64, 16, 16, 16, 16, 16, 16, 16, 8, 2, 64, 4, 0, 16, 16, 1 << 20, None) == -1 and b"null" in E()     # rows twice
    assert L.mfnet_lora_pool_tn(16, 64, None, None, 16, 16, 16, 16, 16, 8, 2, 64, 4, 0, 16, 16, 8, None) == -1 and b"workspace" in E()
    assert L.mfnet_lora_pool_tn(16, 64, None, None, 16, 16, 16, 16, 16, 8, 2, 64, 17, 0, 16, 16, 1 << 20, None) == -1


def test_sizes():
    L = _L()
    assert L.mfnet_layernorm_ckpt8_workspace_floats(1, 64) == 128 and L.mfnet_layernorm_ckpt8_workspace_floats(1 << 20, 64) == 512 * 128
    assert L.mfnet_lora_pool_chunks(0, 5) == 0 and L.mfnet_lora_pool_chunks(3, 100) == 3
    for M in (1, 127, 128, 129, 5000, 16384, 16385, 100000):      # every split of M rows over n adapters fits
        for n in (1, 3, 50):
            c = L.mfnet_lora_pool_chunks(M, n)
            ch = 128 if M <= 16384 else 512
            one_each = min(n, M)
            worst = (one_each - 1) + -(-(M - one_each + 1) // ch)
            assert c >= worst
            assert L.mfnet_lora_pool_tn_workspace_floats(M, n, 64, 32) == c * 64 * 32


def test_wrappers_refuse_host_tensors():
    from ssrs_amd import ops
    from ssrs_amd._lib import MfnetError
    x = torch.zeros(4, 64)
    for bad in (lambda: ops.ckpt8_pack(x), lambda: ops.gelu_fwd_ckpt8(x), lambda: ops.layernorm_fwd_ckpt8(x, torch.ones(64), torch.ones(64), 1e-6),
                lambda: ops.lora_pool(torch.zeros(1, 4, 64), torch.zeros(1, 64, 4)), lambda: ops.lora_pool_plan(torch.zeros(4, dtype=torch.int32), 1)):
        with pytest.raises(MfnetError, match="CPU tensor"):
            bad()
