"""CPU: what the 4-bit products, their expert layers, the balance loss and the expert counts refuse before anything is launched, and the sizes of their workspaces."""
import pytest
import torch

import muxi_native_layout_kernels_amd as mlk
from muxi_native_layout_kernels_amd import _lib

BF, U8 = torch.bfloat16, torch.uint8


def packed(n=32, k=256, group=128, lead=(), dtype=BF):
    per = max(1, 128 // group)
    return (torch.zeros(lead + (n // 16, k // 128, 64, 16), dtype=U8), torch.zeros(lead + (n // 16, k // max(128, group), 16, per), dtype=dtype),
            torch.zeros(lead + (n // 16, k // max(128, group), 16, per), dtype=U8))


def refused(match, f, *args, **kw):
    with pytest.raises((RuntimeError, ValueError), match=match):
        f(*args, **kw)


def test_pack_refuses():
    codes, s, z = torch.zeros(32, 128, dtype=U8), torch.zeros(32, 2, dtype=BF), torch.zeros(32, 2, dtype=U8)
    refused("CUDA", mlk.pack_layout_a_w4, codes, s, z)
    refused("uint8", mlk.pack_layout_a_w4, codes.int(), s)
    refused("fp16 or bf16", mlk.pack_layout_a_w4, codes, s.float())
    refused("zeros must be uint8", mlk.pack_layout_a_w4, codes, s, z.int())
    refused("shape of scales", mlk.pack_layout_a_w4, codes, s, z[:, :1])
    refused("N % 16", mlk.pack_layout_a_w4, codes[:30], s[:30])
    refused("K % 128", mlk.pack_layout_a_w4, codes[:, :96], s)
    refused("scales must be", mlk.pack_layout_a_w4, codes, s[:16])
    refused("scales must be", mlk.pack_layout_a_w4, codes, torch.zeros(32, 3, dtype=BF))
    refused("group", mlk.pack_layout_a_w4, codes, torch.zeros(32, 16, dtype=BF))
    refused("group", mlk.pack_layout_a_w4, torch.zeros(32, 192, dtype=U8), torch.zeros(32, 2, dtype=BF))      # groups of 192
    refused("uint8 \\[N, K/2\\]", mlk.pack_layout_a_w4, torch.zeros(128, dtype=U8), s)
    A, S, Z = packed()
    refused("CUDA", mlk.unpack_layout_a_w4, A, S, Z)
    refused("scales of A", mlk.unpack_layout_a_w4, A, S[:1])
    refused("zero points of A", mlk.unpack_layout_a_w4, A, S, Z[:1])


def test_product_refuses():
    A, S, Z = packed()
    x = torch.zeros(4, 256, dtype=BF)
    refused("CUDA", mlk.gemm_layoutA_w4, A, S, x)
    refused("same k", mlk.gemm_layoutA_w4, A, S, x[:, :128])
    refused("2D", mlk.gemm_layoutA_w4, A, S, x[0])
    refused("Unsupported data type", mlk.gemm_layoutA_w4, A, S, x.float())
    refused("activation dtype", mlk.gemm_layoutA_w4, A, S, x.half())
    refused("A must be uint8", mlk.gemm_layoutA_w4, A.float(), S, x)
    refused("A must be uint8", mlk.gemm_layoutA_w4, A[0], S, x)
    refused("scales of A", mlk.gemm_layoutA_w4, A, S[:, :, :8], x)
    refused("scales of A", mlk.gemm_layoutA_w4, A, S.float(), x)
    refused("scales of A", mlk.gemm_layoutA_w4, A, torch.zeros(2, 2, 16, 3, dtype=BF), x)
    refused("scales of A", mlk.gemm_layoutA_w4, A, torch.zeros(2, 0, 16, 1, dtype=BF), x)
    refused("zero points of A", mlk.gemm_layoutA_w4, A, S, x, Z.int())
    refused("bias", mlk.gemm_layoutA_w4, A, S, x, Z, bias=torch.zeros(1, 16, dtype=BF))
    refused("bias", mlk.gemm_layoutA_w4, A, S, x, Z, bias=torch.zeros(1, 32))
    refused("[bB]eta", mlk.gemm_layoutA_w4, A, S, x, beta=1)
    refused("vector", mlk.gemv_layoutA_w4, A, S, x)


def test_experts_refuse():
    (w1, s1, z1), (w2, s2, z2) = packed(512, 128, 64, (4,)), packed(128, 256, 64, (4,))
    x, ids, wts = torch.zeros(3, 128, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=BF)

    def call(x=x, w1=w1, w2=w2, ids=ids, wts=wts, s1=s1, s2=s2, z1=z1, z2=z2, m=None):
        return mlk.fused_experts_w4(x, w1, w2, ids, wts, s1, s2, z1, z2, m)
    refused("CUDA", call)
    refused("\\[E, 2I, H\\]", call, w2=w2[:3], s2=s2[:3], z2=z2[:3])
    refused("both w1 and w2", call, z2=None)
    refused("\\[T, H\\]", call, x=x[:, :64])
    refused("fp16 or bf16", call, x=x.float())
    refused("activation dtype", call, x=x.half())
    refused("int32", call, ids=ids.long())
    refused("int32", call, ids=ids[:2])
    refused("topk_weights", call, wts=wts.float())
    refused("topk_weights", call, wts=wts[:, :1])
    refused("1..32", call, ids=torch.zeros(3, 33, dtype=torch.int32), wts=torch.zeros(3, 33, dtype=BF))
    refused("experts_map", call, m=torch.zeros(4))
    refused("experts_map", call, m=torch.zeros(0, dtype=torch.int32))
    v2, t2, y2 = packed(128, 256, 128, (4,))
    refused("same group", call, w2=v2, s2=t2, z2=y2)
    from muxi_native_layout_kernels_amd.moe_planC import fused_moe_w4
    refused("CUDA", fused_moe_w4, x, w1, w2, torch.zeros(3, 4, dtype=BF), 2, True, s1, s2, z1, z2)
    refused("tokens", fused_moe_w4, x, w1, w2, torch.zeros(2, 4, dtype=BF), 2, True, s1, s2, z1, z2)
    refused("num_expert_group", fused_moe_w4, x, w1, w2, torch.zeros(3, 4, dtype=BF), 2, True, s1, s2, z1, z2, num_expert_group=2)
    refused("scoring", fused_moe_w4, x, w1, w2, torch.zeros(3, 4, dtype=BF), 2, True, s1, s2, z1, z2, score_func="relu")


def test_balance_and_counts_refuse():
    logits, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int32)
    refused("CUDA", mlk.moe_balance_loss, logits, ids)
    refused("256", mlk.moe_balance_loss, torch.zeros(5, 257), ids)
    refused("256", mlk.moe_balance_loss, torch.zeros(8), ids)
    refused("fp16, bf16 or fp32", mlk.moe_balance_loss, logits.double(), ids)
    refused("int32", mlk.expert_counts, ids.long(), 8)
    refused("int32", mlk.expert_counts, ids[0], 8)
    refused("int32", mlk.expert_counts, ids[:, :0], 8)
    refused("token_mask", mlk.expert_counts, ids, 8, torch.ones(4, dtype=torch.bool))
    refused("token_mask", mlk.expert_counts, ids, 8, torch.ones(5))
    refused("CUDA", mlk.expert_counts, ids, 8)


FAKE = 4096          # an aligned address that is never read: every call below is refused ahead of any launch


def said(lib, rc, word, code=-1):
    assert rc == code and word in lib.mlk_last_error(), (rc, lib.mlk_last_error())


def test_c_interface_of_the_products_refuses():
    lib = _lib.load()

    def gemm(a=FAKE, s=FAKE, z=None, b=FAKE, c=FAKE, m=4, n=32, k=256, group=128, kind=1, ws=None, ws_bytes=0):
        return lib.mlk_gemm_layout_a_w4(a, s, z, b, c, m, n, k, group, kind, 1.0, None, ws, ws_bytes, None)
    said(lib, gemm(m=-1), b"negative")
    said(lib, gemm(n=24), b"N % 16")
    said(lib, gemm(k=192), b"K % 128")
    said(lib, gemm(k=0), b"negative")
    said(lib, gemm(group=16), b"group")
    said(lib, gemm(group=384), b"group")
    said(lib, gemm(k=1 << 23), b"2^23")
    said(lib, gemm(kind=2), b"fp16 or bf16")
    said(lib, gemm(a=None), b"null")
    for p in ("a", "b", "c", "ws"):
        said(lib, gemm(**{p: FAKE + 8}), b"16 bytes")
    said(lib, gemm(s=FAKE + 4), b"8 bytes")
    said(lib, gemm(z=FAKE + 2), b"on 4")
    assert gemm(m=0) == 0 and gemm(n=0) == 0
    scratch = 0
    for m, n, k, group in ((16, 4096, 14336, 128), (100, 512, 1024, 32), (2000, 1024, 1024, 64), (100, 512, 7168, 128), (500, 11008, 4096, 64), (4000, 4096, 4096, 32)):
        need = lib.mlk_gemm_w4_workspace_bytes(m, n, k, group)
        if need == 0:                                    # runs whole
            continue
        assert need > 64 * 1024
        scratch += 1
        said(lib, gemm(m=m, n=n, k=k, group=group, ws=FAKE, ws_bytes=need - 1), b"workspace", -3)
        said(lib, gemm(m=m, n=n, k=k, group=group), b"workspace", -3)
    assert scratch >= 4
    assert lib.mlk_gemm_w4_workspace_bytes(1, 4096, 4096, 128) == 0
    for bad in ((0, 16, 128, 128), (1, 0, 128, 128), (1, 16, 0, 128), (1, 16, 128, 48), (1, 16, 128, 256), (-5, 16, 128, 128)):
        assert lib.mlk_gemm_w4_workspace_bytes(*bad) == 0
    said(lib, lib.mlk_pack_layout_a_w4(FAKE, FAKE, 1, 24, 128, None), b"N % 16")
    said(lib, lib.mlk_pack_layout_a_w4(FAKE, FAKE + 2, 1, 16, 128, None), b"4 bytes")
    said(lib, lib.mlk_unpack_layout_a_w4(None, FAKE, 1, 16, 128, None), b"4 bytes")
    said(lib, lib.mlk_pack_scales_w4(FAKE, FAKE, 1, 16, 128, 96, 2, None), b"group")
    said(lib, lib.mlk_pack_scales_w4(FAKE, FAKE, 1, 16, 128, 64, 4, None), b"2 bytes")
    said(lib, lib.mlk_unpack_scales_w4(FAKE, None, 1, 16, 128, 64, 1, None), b"null")
    assert lib.mlk_pack_layout_a_w4(None, None, 0, 16, 128, None) == 0 and lib.mlk_pack_scales_w4(None, None, 1, 0, 128, 64, 1, None) == 0


def test_c_interface_of_the_experts_refuses():
    lib = _lib.load()

    def experts(w1=FAKE, s1=FAKE, z1=None, w2=FAKE, s2=FAKE, z2=None, x=FAKE, t=4, e=8, er=8, k=2, h=256, i=128, group=128, kind=0, ids=FAKE, wts=FAKE,
                m=None, y=FAKE, ws=FAKE, ws_bytes=1 << 40):
        return lib.mlk_fused_experts_w4(w1, s1, z1, w2, s2, z2, x, t, e, er, k, h, i, group, kind, ids, wts, m, y, ws, ws_bytes, None)
    for kw, word in ((dict(kind=3), b"fp16 or bf16"), (dict(t=-1), b"negative"), (dict(e=257, er=257), b"256"), (dict(e=0, er=0), b"256"),
                     (dict(er=9), b"experts_map"), (dict(k=0), b"topk"), (dict(k=33), b"topk"), (dict(h=192), b"multiples of 128"),
                     (dict(i=0), b"multiples of 128"), (dict(h=1 << 23), b"2^23"), (dict(group=256), b"group"), (dict(group=16), b"group"),
                     (dict(z1=FAKE), b"zero points"), (dict(y=None), b"null"), (dict(ws=None), b"null"), (dict(x=FAKE + 8), b"16 bytes"),
                     (dict(s2=FAKE + 4), b"8 bytes"), (dict(z1=FAKE + 2, z2=FAKE), b"on 4")):
        said(lib, experts(**kw), word)
    assert experts(t=0) == 0
    for t in (1, 4, 500, 20000):
        need = lib.mlk_experts_w4_workspace_bytes(t, 8, 8, 2, 256, 128, 128)
        assert need > 0
        said(lib, experts(t=t, ws_bytes=need - 1), b"workspace", -3)
    # passes of 16384 pairs: a long prompt needs no more than its longest pass
    assert lib.mlk_experts_w4_workspace_bytes(1 << 20, 8, 8, 2, 256, 128, 128) == lib.mlk_experts_w4_workspace_bytes(8192, 8, 8, 2, 256, 128, 128)
    for bad in ((0, 8, 8, 2, 256, 128, 128), (4, 0, 8, 2, 256, 128, 128), (4, 257, 257, 2, 256, 128, 128), (4, 8, 8, 33, 256, 128, 128), (4, 8, 8, 2, 0, 128, 128),
                (4, 8, 8, 2, 256, 128, 0), (4, 8, 0, 2, 256, 128, 128)):
        assert lib.mlk_experts_w4_workspace_bytes(*bad) == 0


def test_c_interface_of_the_balance_loss_refuses():
    lib = _lib.load()

    def loss(x=FAKE, kind=3, fun=0, t=10, e=8, k=2, ids=FAKE, mask=None, cu=None, s=1, out=FAKE, counts=FAKE, share=FAKE, ws=FAKE, ws_bytes=1 << 40):
        return lib.mlk_balance_loss(x, kind, fun, t, e, k, ids, mask, cu, s, 1.0, out, counts, share, ws, ws_bytes, None)
    for kw, word in ((dict(kind=2), b"fp16, bf16 or fp32"), (dict(fun=2), b"score"), (dict(t=-1), b"tokens"), (dict(t=(1 << 30) + 1), b"tokens"),
                     (dict(t=1 << 29, k=4), b"pairs"), (dict(k=0), b"pick"), (dict(e=0), b"experts"), (dict(e=257), b"experts"), (dict(s=2), b"sequences"),
                     (dict(s=0), b"sequences"), (dict(cu=FAKE, s=65536), b"sequences"), (dict(x=None), b"null"), (dict(ids=None), b"null"), (dict(out=None), b"null"),
                     (dict(ws=None), b"null"), (dict(ws=FAKE + 8), b"16 bytes")):
        said(lib, loss(**kw), word)
    need = lib.mlk_balance_workspace_bytes(10, 8, 1)
    said(lib, loss(ws_bytes=need - 1), b"workspace", -3)
    assert lib.mlk_balance_workspace_bytes(-1, 8, 1) == 0 and lib.mlk_balance_workspace_bytes(1, 300, 1) == 0
    assert lib.mlk_balance_workspace_bytes(1, 8, 65536) == 0 and lib.mlk_balance_workspace_bytes((1 << 30) + 1, 8, 1) == 0
    assert lib.mlk_balance_counter_bytes() <= lib.mlk_balance_workspace_bytes(1, 1, 1)

    def grad(x=FAKE, kind=3, t=10, e=8, s=1, share=FAKE, g=FAKE, d=FAKE):
        return lib.mlk_balance_loss_grad(x, kind, 0, t, e, None, None, s, share, g, d, None)
    for kw, word in ((dict(kind=2), b"fp16, bf16 or fp32"), (dict(t=(1 << 30) + 1), b"tokens"), (dict(s=3), b"sequences"), (dict(share=None), b"null"),
                     (dict(g=None), b"null"), (dict(d=None), b"null")):
        said(lib, grad(**kw), word)
    assert grad(t=0) == 0
    for kw, word in ((dict(n_tokens=-1), b"negative"), (dict(topk=0), b"picks"), (dict(n_experts=300), b"256"), (dict(counts=None), b"null"), (dict(topk_ids=None), b"null"),
                     (dict(n_tokens=2049), b"workspace"), (dict(n_tokens=2049, workspace=FAKE + 8), b"16 bytes")):
        a = dict(topk_ids=FAKE, token_mask=None, n_tokens=4, topk=2, n_experts=8, accumulate=0, counts=FAKE, workspace=None, stream=None)
        a.update(kw)
        said(lib, lib.mlk_expert_counts(*a.values()), word)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_zero_points_that_take_more_than_four_bits_are_refused(device):
    codes, s = torch.zeros(3, 32, 128, dtype=U8, device=device), torch.ones(3, 32, 2, dtype=BF, device=device)
    for wrong in (16, 255):
        z = torch.full((3, 32, 2), 15, dtype=U8, device=device)
        z[2, 31, 1] = wrong
        refused("0..15", mlk.pack_layout_a_w4, codes, s, z)


def test_balance_loss_refuses_forward_mode():
    from torch.autograd import forward_ad
    logits, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int32)
    with forward_ad.dual_level():
        refused("forward-mode", mlk.moe_balance_loss, forward_ad.make_dual(logits, torch.ones(5, 8)), ids)
        refused("CUDA", mlk.moe_balance_loss, logits, ids)


def test_router_refuses_a_bias_that_it_would_read_past():
    """Short, strided, of another type or elsewhere: said before the logits are looked at on the device."""
    logits, ids, wts = torch.zeros(3, 8, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=BF)

    def call(bias):
        return mlk.fused_routing_gate(logits, 0, 3, 128, 1, 1, ids, wts, 2, bias, True)
    refused("every expert", call, torch.zeros(7, dtype=BF))
    refused("contiguous", call, torch.zeros(16, dtype=BF)[::2])
    refused("contiguous", call, torch.zeros(8, dtype=BF, device="meta"))
    refused("Mismatched dtypes", call, torch.zeros(8))
    refused("CUDA", call, torch.zeros(8, dtype=BF))
    refused("CUDA", call, torch.zeros(1, 8, dtype=BF))


def test_layer_refuses_its_own_arguments():
    from muxi_native_layout_kernels_amd.moe_planC import fused_moe_w4
    (w1, s1, z1), (w2, s2, z2) = packed(512, 128, 64, (4,)), packed(128, 256, 64, (4,))
    x, logits = torch.zeros(3, 128, dtype=BF), torch.zeros(3, 4, dtype=BF)

    def call(**kw):
        return fused_moe_w4(x, w1, w2, logits, 2, True, s1, s2, z1, z2, **kw)
    refused("n_experts", call, expert_load=torch.zeros(3, dtype=torch.int32))
    refused("n_experts", call, expert_load=torch.zeros(4, dtype=torch.int64))
    refused("n_experts", call, expert_load=torch.zeros(1, 4, dtype=torch.int32))
    refused("every expert", call, gating_bias=torch.zeros(3, dtype=BF))
    refused("CUDA", call, gating_bias=torch.zeros(4, dtype=BF), expert_load=torch.zeros(4, dtype=torch.int32))


def test_counters_in_front_of_the_workspace_are_those_of_the_other_products():
    """One buffer serves them all: behind the counters, 16 tokens through 4096 rows of 14336 keep the partial sums of each slice of k, a whole number of outputs in fp32."""
    lib = _lib.load()
    partial = lib.mlk_gemm_w4_workspace_bytes(16, 4096, 14336, 128) - lib.mlk_gemm_counter_bytes()
    assert partial > 0 and partial % (16 * 4096 * 4) == 0
