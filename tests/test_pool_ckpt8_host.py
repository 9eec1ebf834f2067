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
    for k, v, msg in ((13, 16, b"go together"), (10, None, b"null"), (0, None, b"null"), (3, None, b"null"), (12, 16, b"beta"), (2, 62, b"lddy")):
        a = list(bwd)
        a[k] = v
        assert L.mfnet_layernorm_bwd_ckpt8(*a) == -1 and msg in E(), msg
    a = list(bwd)
    a[13] = a[14] = 16
    a[17] = 2049                               # (up to 2048 rows need none)
    assert L.mfnet_layernorm_bwd_ckpt8(*a) == -1 and b"workspace" in E()
    pack = dict(A=16, B=16, dt=0, scale=None, n=2, K=64, N=64, r=4, RP=16, a_down=16, a_up=16, b_down=16, b_up=16, so=16, s=None)
    for key, v, msg in (("r", 20, b"sizes"), ("K", 60, b"sizes"), ("N", 4, b"sizes"), ("RP", 24, b"sizes"), ("n", 0, b"sizes"), ("b_down", None, b"null"), ("so", None, b"null"), ("a_up", 24, b"misaligned"),
                        ("A", 18, b"misaligned"), ("dt", 3, b"dtype")):
        assert L.mfnet_lora_pool_pack(*dict(pack, **{key: v}).values()) == -1 and msg in E(), key
    assert L.mfnet_lora_pool_plan(16, 1 << 27, 2, 16, 16, 16, 16, None) == -1 and b"sizes" in E()
    assert L.mfnet_lora_pool_plan(None, 8, 2, 16, 16, 16, 16, None) == -1 and b"null" in E()
    fwd = dict(X=16, ldx=64, W=16, ldw=64, bias=None, scale=16, a_down=16, b_up=16, ids=16, n=2, RP=16, down=16, nd=8 * 16, out=16, dt=1, ldo=64, M=8, N=64, K=64, s=None)
    for key, v, msg in (("ldx", 60, b"row stride"), ("K", 60, b"multiple of 8"), ("X", 24, b"16-byte"), ("W", None, b"null"), ("ldw", 56, b"weight"), ("ldo", 62, b"out"),
                        ("nd", 8 * 16 - 1, b"too few"), ("RP", 17, b"sizes"), ("n", 0, b"sizes"), ("M", 1 << 27, b"sizes"), ("dt", 2, b"dtype"), ("down", None, b"null"), ("b_up", 24, b"misaligned"), ("ids", None, b"null")):
        assert L.mfnet_lora_pool_fwd(*dict(fwd, **{key: v}).values()) == -1 and msg in E(), key
    assert L.mfnet_lora_pool_fwd(*dict(fwd, M=0).values()) == 0
    bwd = dict(dy=16, lddy=64, X=16, ldx=64, codes=None, exps=None, Wt=16, ldwt=64, scale=16, b_down=16, a_up=16, ids=16, offs=16, perm=16, base=16, table=16, n=2, r=4, RP=16, down=16,
               dx=16, lddx=64, dA=16, dB=16, ws=16, nws=1 << 20, M=8, N=64, K=64, s=None)
    for key, v, msg in (("codes", 16, b"either"), ("X", None, b"either"), ("lddy", 60, b"dy"), ("ldx", 60, b"(x)"), ("ldwt", 56, b"weight"), ("lddx", 60, b"dx"), ("r", 17, b"sizes"),
                        ("nws", 100, b"workspace"), ("dA", None, b"null"), ("table", 24, b"misaligned"), ("K", 68, b"multiples of 8"), ("Wt", None, b"null"), ("down", None, b"null")):
        assert L.mfnet_lora_pool_bwd(*dict(bwd, **{key: v}).values()) == -1 and msg in E(), key


def test_sizes():
    L = _L()
    assert [L.mfnet_layernorm_ckpt8_workspace_floats(r, 64) for r in (0, 1, 2048, 2049, 1 << 20)] == [0, 0, 0, 257 * 128, 512 * 128]
    assert L.mfnet_lora_pool_chunks(0, 5) == 0 and L.mfnet_lora_pool_chunks(3, 100) == 3
    for M in (1, 127, 128, 129, 512, 513, 5000, 5001, 12288, 12289, 100000):      # every split of M rows over n adapters fits
        for n in (1, 3, 50):
            c = L.mfnet_lora_pool_chunks(M, n)
            ch = 512 if M <= 512 or M > 12288 else 128 if M <= 5000 else 256
            one_each = min(n, M)
            worst = (one_each - 1) + -(-(M - one_each + 1) // ch)
            assert c >= worst
            assert L.mfnet_lora_pool_bwd_workspace_floats(M, n, 64, 72, 32) == L.mfnet_lora_pool_down_floats(M, 32, 1) + (c * (64 + 72) * 32 if M > 512 else 0)


def test_room_behind_the_down_products():
    L = _L()
    for M in (0, 1, 64, 65, 5000):      # fp32 [M, RP]; above 64 rows two bf16 parts of it for a bf16 result, three for an fp32 one
        for RP in (16, 64):
            for dt, parts in ((1, 2), (0, 3)):
                assert L.mfnet_lora_pool_down_floats(M, RP, dt) == M * RP + (M * RP * parts // 2 if M > 64 else 0)


def test_wrappers_refuse_host_tensors():
    from ssrs_amd import ops
    from ssrs_amd._lib import MfnetError
    x = torch.zeros(4, 64)
    for bad in (lambda: ops.ckpt8_pack(x), lambda: ops.gelu_fwd_ckpt8(x), lambda: ops.layernorm_fwd_ckpt8(x, torch.ones(64), torch.ones(64), 1e-6),
                lambda: ops.lora_pool(torch.zeros(1, 4, 64), torch.zeros(1, 64, 4)), lambda: ops.lora_pool_plan(torch.zeros(4, dtype=torch.int32), 1)):
        with pytest.raises(MfnetError, match="CPU tensor"):
            bad()
