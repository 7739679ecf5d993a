"""CPU: sizes at the ends of what the e4m3 products, their expert layers and the routing promise."""
from muxi_native_layout_kernels_amd import _lib


def test_scales_of_an_intermediate_stay_within_32_bits():
    """The down panels address the scales [I/128, slots] of a pass with 32 bits: codes of slots * I bytes and scales of a 32nd of that, at most 2^37 and 2^32.  Beside them one token's row, sums and tables are small."""
    lib = _lib.load()
    hidden, inter = 128, (1 << 23) - 128
    for tokens, experts, picks in ((16384, 1, 1), (16384, 16, 1), (8192, 16, 2), (100000, 8, 4)):
        need = lib.mlk_experts_fp8_workspace_bytes(tokens, experts, experts, picks, hidden, inter)
        assert (1 << 36) < need <= (1 << 37) + (1 << 32) + (1 << 26), (tokens, experts, picks)


def test_scratch_of_an_expert_layer_serves_every_shorter_call():
    lib = _lib.load()
    for experts, router, picks, hidden, inter in ((8, 8, 2, 4096, 14336), (16, 16, 4, 512, 256), (64, 128, 8, 2048, 768), (1, 1, 1, 256, 128), (3, 300, 32, 256, 8192), (2, 2, 1, 128, (1 << 23) - 128),
                                                  (32, 256, 8, 7168, 2048), (4, 4, 2, 1 << 20, 128)):
        last = 0
        for tokens in list(range(1, 2101)) + [2600, 4096, 5000, 8192, 8193, 16384, 16385, 20000, 100000]:
            need = lib.mlk_experts_fp8_workspace_bytes(tokens, experts, router, picks, hidden, inter)
            assert need >= last > -1, (experts, router, picks, hidden, inter, tokens)
            last = need


def test_arrivals_fit_the_counters():
    """k past the panels' offsets, so that thousands of tokens stream: 16 sets of rows x tokens / 32 workgroups count their arrivals in 16384 counters, if k is in slices; from 32769 tokens on they do not fit."""
    lib = _lib.load()
    few = lib.mlk_gemm_fp8_workspace_bytes(256, 1024, 1 << 23, 2)
    for tokens in (257, 32768, 32769, 40000):
        assert lib.mlk_gemm_fp8_workspace_bytes(tokens, 1024, 1 << 23, 2) <= few, tokens


def test_scratch_of_a_product_serves_every_shorter_call():
    lib = _lib.load()
    for n, k in ((8192, 8192), (4096, 14336), (512, 7168), (28672, 8192), (13824, 5120), (16, 128), (1040, 12416), (37888, 3584), (272, 640), (1024, 1 << 23), (4096, (1 << 23) - 128)):
        for kind in (0, 1, 2):
            last = 0
            for tokens in list(range(1, 700)) + list(range(700, 4500, 37)) + [8191, 8192, 16384, 16385, 30000, 1 << 20, 1 << 21]:
                need = lib.mlk_gemm_fp8_workspace_bytes(tokens, n, k, kind)
                assert need >= last, (n, k, kind, tokens)
                assert need > 0 or not lib.mlk_gemm_fp8_needs_workspace(tokens, n, k, kind)
                last = need
    assert lib.mlk_gemm_fp8_needs_workspace(100, 32, 256, 1) and not lib.mlk_gemm_fp8_needs_workspace(8, 4096, 4096, 2)


def test_one_limit_of_k():
    """Quantising and the product that quantises its activations refuse the same k, with pointers that are never read."""
    lib = _lib.load()
    p, big = 4096, 1 << 60
    for k in (65535 * 512 + 128, (1 << 25) - 128, 1 << 25):
        assert lib.mlk_quantize_fp8(p, 1, p, p, 1, 1, 1, k, None) < 0 and b"33553920" in lib.mlk_last_error()
        for kind in (1, 2):
            assert lib.mlk_gemm_layout_a_fp8(p, p, p, kind, p, 1, 1, p, 1, 100, 32, k, 1.0, None, p, big, None) < 0 and b"33553920" in lib.mlk_last_error(), (k, kind)
    # the last one that is taken is refused for its workspace, which is checked behind it
    assert lib.mlk_gemm_layout_a_fp8(p, p, p, 1, None, 0, 0, p, 1, 100, 32, 65535 * 512, 1.0, None, p, 64, None) < 0 and b"too small" in lib.mlk_last_error()


def test_rows_of_weights_that_a_launch_has_threads_for():
    lib = _lib.load()
    p, big = 4096, 1 << 60
    for n in ((1 << 27) + 16, 1 << 29, (1 << 31) - 16):
        for kind in (1, 2):
            assert lib.mlk_gemm_layout_a_fp8(p, p, p, kind, p, 1, 1, p, 1, 1, n, 128, 1.0, None, p, big, None) < 0 and b"2^27 rows" in lib.mlk_last_error(), (n, kind)
