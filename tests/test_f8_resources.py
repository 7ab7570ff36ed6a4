"""Register and scratch use of the 8-bit floating tier's kernels and of the gradient's, read from the built library (no GPU
needed)."""
from test_kernel_resources import records  # noqa: F401 (the fixture)


def test_the_tiles_keep_nothing_in_scratch(records):  # noqa: F811
    # a value kept in private memory is waited for together with the loads into LDS, which are meant to stay in flight
    mine = [k for k in records if any(n in k[".name"] for n in ("f8_gemm_kernel", "f8_group_kernel", "f8_stream_kernel",
                                                              "4kxw411grad_kernel"))]
    assert len(mine) >= 6 + 4 + 24 + 2
    bad = {k[".name"]: k[".private_segment_fixed_size"] for k in mine if k[".private_segment_fixed_size"]}
    assert not bad


def test_two_work_groups_of_the_smaller_tiles_fit_a_cu(records):  # noqa: F811
    # 512 registers a SIMD lane: kernels meant for two waves a SIMD hold up to 256
    for k in records:
        if any(n in k[".name"] for n in ("f8_gemm_kernel", "f8_group_kernel", "4kxw411grad_kernel")):
            assert k[".vgpr_count"] + k.get(".agpr_count", 0) <= 256, k[".name"]
