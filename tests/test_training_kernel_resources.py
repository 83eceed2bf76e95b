"""What the compiler gave the kernels of layer norm, gated product, embedding and clipping; no GPU needed."""
from test_kernel_resources import kernels  # noqa: F401  (the fixture)


def of(kernels, *names):  # noqa: F811
    return {n: v for n, v in kernels.items() if "rocprim" not in n and any(f"{len(k)}{k}" in n for k in names)}


def test_gated_products_keep_their_sums_in_registers(kernels):  # noqa: F811
    found = of(kernels, "gated_wide_kernel", "gated_direct_kernel", "gated_product_kernel", "few_rows_kernel", "gated_join_kernel", "gate_grad_kernel")
    # 16 and 8 bits large tiles, four forms of small ones; two tiles of all five types; few rows with 8 and 16 wavefronts, gated and not; joins; three types by width
    assert [len(of(kernels, n)) for n in ("gated_wide_kernel", "gated_direct_kernel", "gated_product_kernel", "few_rows_kernel", "gated_join_kernel", "gate_grad_kernel")] == [4, 16, 10, 20, 6, 9]
    assert {n: v for n, v in found.items() if v[1]} == {}


def test_layer_norm_keeps_its_rows_in_registers(kernels):  # noqa: F811
    found = of(kernels, "layer_norm_kernel", "layer_norm_long_kernel", "layer_norm_grad_kernel", "layer_norm_grad_long_kernel", "layer_norm_sums_kernel")
    assert len(found) == 9 * 9 + 9 + 9 * 9 + 9 + 1
    # (a workgroup of 1024 threads leaves a thread 128 registers: up to 11 words of a gradient's row with a stream of 16 bits go to memory)
    tight = {n: v for n, v in found.items() if "layer_norm_grad_kernel" in n and "Li1024E" in n and "fLi1024E" not in n}
    assert len(tight) == 6 and {n: v for n, v in tight.items() if v[1] > 44} == {}
    assert {n: v for n, v in found.items() if n not in tight and v[1]} == {}


def test_embedding_and_clipping_keep_to_registers(kernels):  # noqa: F811
    found = of(kernels, "embedding_kernel", "embedding_sums_kernel", "embedding_join_kernel", "sort_count_kernel", "sort_offsets_kernel", "sort_move_kernel", "sort_small_kernel", "squares_kernel",
               "clip_kernel")
    assert len(found) == 12 + 12 + 8 + 1 + 1 + 2 + 4 + 1 + 1
    assert {n: v for n, v in found.items() if v[1]} == {}
