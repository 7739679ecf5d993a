"""CPU: what the e4m3 products, their expert layers and the routing refuse before anything is launched, and the sizes of their workspaces."""
import pytest
import torch

import muxi_native_layout_kernels_amd as mlk
from muxi_native_layout_kernels_amd import _lib

BF, F8, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8


def refused(match, f, *args, **kw):
    with pytest.raises((RuntimeError, ValueError), match=match):
        f(*args, **kw)


def test_quantize_refuses():
    refused("CUDA", mlk.quantize_fp8, torch.zeros(4, 128, dtype=BF))
    refused("fp16, bf16 or fp32", mlk.quantize_fp8, torch.zeros(4, 128, dtype=torch.float64))
    refused("multiple of 128", mlk.quantize_fp8, torch.zeros(4, 96, dtype=BF))
    refused("multiple of 128", mlk.quantize_fp8, torch.zeros(4, 0, dtype=BF))
    refused("multiple of 128", mlk.quantize_fp8, torch.zeros((), dtype=BF))


def test_product_refuses():
    A, S, x = torch.zeros(2, 32, 16, 8, dtype=U8), torch.zeros(1, 2), torch.zeros(4, 256, dtype=BF)
    q, a = torch.zeros(4, 256, dtype=U8), torch.zeros(4, 2)
    refused("CUDA", mlk.gemm_layoutA_fp8, A, S, x)
    refused("4D", mlk.gemm_layoutA_fp8, A[0], S, x)
    refused("e4m3", mlk.gemm_layoutA_fp8, A.to(BF), S, x)
    refused("k % 128", mlk.gemm_layoutA_fp8, A[:, :8], S, x)
    refused("A_Scale", mlk.gemm_layoutA_fp8, A, S.to(BF), x)
    refused("A_Scale", mlk.gemm_layoutA_fp8, A, torch.zeros(2, 2), x)
    refused("2D", mlk.gemm_layoutA_fp8, A, S, x[0])
    refused("same k", mlk.gemm_layoutA_fp8, A, S, x[:, :128])
    refused("B must be fp16 or bf16", mlk.gemm_layoutA_fp8, A, S, x.float())
    refused("B must be fp16 or bf16", mlk.gemm_layoutA_fp8, A, S, q)
    refused("out_dtype is that of B", mlk.gemm_layoutA_fp8, A, S, x, out_dtype=torch.float16)
    refused("e4m3 codes where there is a B_Scale", mlk.gemm_layoutA_fp8, A, S, x, a)
    refused("B_Scale must be fp32", mlk.gemm_layoutA_fp8, A, S, q, a[:, :1])
    refused("B_Scale must be fp32", mlk.gemm_layoutA_fp8, A, S, q, a.to(BF))
    refused("B_Scale must be on", mlk.gemm_layoutA_fp8, A, S, q, a)
    refused("bias", mlk.gemm_layoutA_fp8, A, S, x, bias=torch.zeros(1, 32))
    refused("bias", mlk.gemm_layoutA_fp8, A, S, x, bias=torch.zeros(1, 16, dtype=BF))
    refused("[bB]eta", mlk.gemm_layoutA_fp8, A, S, x, beta=1)


def layer(E=4, H=256, I=128):
    return (torch.zeros(E, 2 * I // 16, H // 8, 16, 8, dtype=U8), torch.zeros(E, H // 16, I // 8, 16, 8, dtype=U8),
            torch.zeros(E, 2 * I // 128, H // 128), torch.zeros(E, H // 128, I // 128))


def test_experts_refuse():
    w1, w2, s1, s2 = layer()
    x, ids, wts = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=BF)
    f = mlk.fused_experts_fp8
    refused("CUDA", f, x, w1, w2, ids, wts, s1, s2)
    refused("e4m3", f, x, w1.to(BF), w2, ids, wts, s1, s2)
    refused("layout-A", f, x, w1[0], w2[0], ids, wts, s1, s2)
    refused("w1 must be", f, x, w1[:2], w2, ids, wts, s1, s2)
    refused("w1 must be", f, x, w1, w2[:, :8], ids, wts, s1, s2)
    refused("w1_scale", f, x, w1, w2, ids, wts, s1[:, :1], s2)
    refused("w2_scale", f, x, w1, w2, ids, wts, s1, s2[:1])
    refused("scales must be float32", f, x, w1, w2, ids, wts, s1.to(BF), s2)
    refused("hidden_states must be \\[T, H\\]", f, x[:, :128], w1, w2, ids, wts, s1, s2)
    refused("fp16 or bf16", f, x.float(), w1, w2, ids, wts, s1, s2)
    refused("topk_ids", f, x, w1, w2, ids.long(), wts, s1, s2)
    refused("topk_ids", f, x, w1, w2, ids[:2], wts, s1, s2)
    refused("topk_weights", f, x, w1, w2, ids, wts.float(), s1, s2)
    refused("topK", f, x, w1, w2, ids[:, :0], wts[:, :0], s1, s2)
    refused("topK", f, x, w1, w2, torch.zeros(3, 33, dtype=torch.int32), torch.zeros(3, 33, dtype=BF), s1, s2)
    refused("experts_map", f, x, w1, w2, ids, wts, s1, s2, torch.zeros(8))
    big = layer(257, 128, 128)
    refused("256 experts", f, torch.zeros(3, 128, dtype=BF), big[0], big[1], ids, wts, big[2], big[3])


def test_moe_layer_refuses():
    from muxi_native_layout_kernels_amd.moe_planC import fused_moe_fp8
    w1, w2, s1, s2 = layer()
    x, logits = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 4, dtype=BF)
    refused("CUDA", fused_moe_fp8, x, w1, w2, logits, 2, True, s1, s2)
    refused("Number of tokens", fused_moe_fp8, x, w1, w2, logits[:2], 2, True, s1, s2)
    refused("num_expert_group must be 1", fused_moe_fp8, x, w1, w2, logits, 2, True, s1, s2, num_expert_group=2)
    refused("activation dtype or be fp32", fused_moe_fp8, x, w1, w2, logits.half(), 2, True, s1, s2)
    refused("one column per expert", fused_moe_fp8, x, w1, w2, logits[:, :3], 2, True, s1, s2)


def test_routing_refuses():
    x = torch.zeros(4, 16, dtype=BF)
    f = mlk.moe_routing
    refused("CUDA", f, x, 2)
    refused("512 experts", f, torch.zeros(4, 513), 2)
    refused("512 experts", f, x[0], 2)
    refused("fp16, bf16 or fp32", f, x.double(), 2)
    refused("topk must be", f, x, 0)
    refused("topk must be", f, x, 17)
    refused("topk must be", f, torch.zeros(4, 64), 33)
    refused("num_expert_group", f, x, 2, "softmax", True, 3)
    refused("topk_group must be", f, x, 2, "softmax", True, 4, 5)
    refused("kept groups hold", f, x, 5, "softmax", True, 4, 1)
    refused("gating_bias", f, x, 2, gating_bias=torch.zeros(16, dtype=BF))
    refused("gating_bias", f, x, 2, gating_bias=torch.zeros(8))
    refused("token_mask", f, x, 2, token_mask=torch.zeros(4))
    refused("token_mask", f, x, 2, token_mask=torch.zeros(3, dtype=torch.bool))


def test_library_refuses_by_itself():
    """What a caller of the C interface may get wrong, with pointers that are never read."""
    lib = _lib.load()
    p, odd = 4096, 4100
    for args, word in (((p, 2, p, p, 1, 1, 1, 128, None), b"fp16, bf16 or fp32"), ((p, 1, p, p, 1, 1, -1, 128, None), b"2^27"), ((p, 1, p, p, 1, 1, 1, 100, None), b"K % 128"),
                       ((None, 1, p, p, 1, 1, 1, 128, None), b"null"), ((odd, 1, p, p, 1, 1, 1, 128, None), b"16 bytes"), ((p, 1, odd, p, 1, 1, 1, 128, None), b"16 bytes")):
        assert lib.mlk_quantize_fp8(*args) < 0 and word in lib.mlk_last_error()
    big = 1 << 40
    good = [p, p, p, 1, None, 0, 0, p, 1, 100, 32, 256, 1.0, None, p, big, None]
    for at, value, word in ((8, 2, b"fp16 or bf16"), (3, 0, b"output's kind"), (9, -1, b"tokens"), (9, (1 << 21) + 1, b"tokens"), (10, 24, b"N % 16"), (11, 192, b"K % 128"), (0, None, b"null"), (1, None, b"null"),
                            (2, odd, b"16 bytes"), (7, odd, b"16 bytes"), (15, 64, b"too small"), (14, odd, b"workspace")):
        bad = list(good)
        bad[at] = value
        assert lib.mlk_gemm_layout_a_fp8(*bad) < 0 and word in lib.mlk_last_error(), (at, lib.mlk_last_error())
    good = [p, p, p, p, p, 3, 4, 4, 2, 256, 128, 1, p, p, None, p, p, big, None]
    for at, value, word in ((11, 2, b"fp16 or bf16"), (5, -1, b"negative"), (6, 257, b"256 experts"), (7, 8, b"experts_map"), (8, 33, b"topk"), (9, 100, b"multiples of 128"),
                            (10, 0, b"multiples of 128"), (0, None, b"null"), (4, odd, b"16 bytes"), (17, 64, b"too small")):
        bad = list(good)
        bad[at] = value
        assert lib.mlk_fused_experts_fp8(*bad) < 0 and word in lib.mlk_last_error(), (at, lib.mlk_last_error())
    good = [p, 1, 0, 3, 16, 1, 1, 2, None, 1, 1.0, None, p, p, None]
    for at, value, word in ((1, 2, b"fp16, bf16 or fp32"), (2, 2, b"score function"), (3, -1, b"tokens"), (4, 513, b"512"), (5, 3, b"divide"), (6, 2, b"topk_groups"), (7, 33, b"picks"),
                            (0, None, b"null"), (12, None, b"null")):
        bad = list(good)
        bad[at] = value
        assert lib.mlk_moe_routing(*bad) < 0 and word in lib.mlk_last_error(), (at, lib.mlk_last_error())
    assert lib.mlk_moe_routing_grad(p, 1, 0, 3, 16, 2, 1, 1.0, None, p, p, None) < 0 and b"null" in lib.mlk_last_error()
    # nothing to do is not an error
    assert lib.mlk_quantize_fp8(None, 1, None, None, 1, 1, 0, 128, None) == 0
    assert lib.mlk_moe_routing(None, 1, 0, 0, 16, 1, 1, 2, None, 1, 1.0, None, None, None, None) == 0


def test_workspaces_grow_with_the_call():
    lib = _lib.load()
    assert lib.mlk_gemm_fp8_workspace_bytes(100, 32, 256, 1) >= lib.mlk_gemm_counter_bytes() + 100 * 256 + 100 * 2 * 4
    assert lib.mlk_gemm_fp8_workspace_bytes(0, 32, 256, 1) == 0 and lib.mlk_gemm_fp8_workspace_bytes(4, 32, 200, 1) == 0
    last = 0
    for t in (1, 2, 17, 300, 1024, 5000, 100000):
        need = lib.mlk_experts_fp8_workspace_bytes(t, 16, 16, 4, 512, 256)
        assert need >= last or t == 100000
        last = max(last, need)
    assert lib.mlk_experts_fp8_workspace_bytes(100000, 16, 16, 4, 512, 256) < 2 * lib.mlk_experts_fp8_workspace_bytes(4096, 16, 16, 4, 512, 256)
    assert lib.mlk_experts_fp8_workspace_bytes(4, 257, 257, 4, 512, 256) == 0
