"""The expert-layer entry points without a GPU: nothing runs before gpuq_init, and sizes are pure functions."""
import pytest


@pytest.fixture(scope="module")
def lib():
    import gpuq
    return gpuq.open_lib()


def test_sizes(lib):
    assert [lib.gpuq_mxfp4_bytes(f, 2, 3, 512) for f in (0, 1, 2)] == [6 * 272, 6 * 272, 32 * 272]
    assert [lib.gpuq_mxfp4_bytes(f, 1, 5, 32) for f in (0, 1, 2)] == [5 * 17, 5 * 272, 16 * 272]
    assert lib.gpuq_mxfp4_bytes(2, 256, 2048, 7168) == 256 * 2048 * 7168 * 17 // 32
    assert [lib.gpuq_mxfp4_bytes(*a) for a in ((0, 1, 0, 32), (1, 0, 1, 32), (2, 1, 1, 33), (1, 1, -1, 32), (3, 1, 1, 32),
                                               (-1, 1, 1, 32), (0, 1, 1, 1 << 25), (2, 1 << 20, 1 << 20, 32))] == [0] * 8
    # many F32 and F16 rows as 3 and 2 BF16 rows of whole 128s; partial sums only where there are few tiles
    assert [lib.gpuq_mxfp4_matmul_work(t, 0, 8192, 1, 8192, 3200, 0, 8192) for t in (0, 1, 30, 39)] == [8192 * 19200,
                                                                                                   8192 * 12800, 0, 0]
    assert [lib.gpuq_mxfp4_matmul_work(t, 0, 16, 1, 64, 32, 0, 16) for t in (0, 1, 30, 39)] == [0] * 4
    part = lib.gpuq_mxfp4_matmul_work(30, 0, 100, 1, 64, 4096, 0, 100)
    assert part > 0 and part % (100 * 64 * 4) == 0 and lib.gpuq_mxfp4_matmul_work(30, 1, 100, 1, 64, 4096, 0, 100) % part == 0
    assert lib.gpuq_mxfp4_matmul_work(30, 0, 8192, 1, 8192, 4096, 0, 8192) == 0
    assert [lib.gpuq_mxfp4_matmul_work(*a) for a in ((8, 0, 1, 1, 1, 32, 0, 1), (30, 0, 0, 1, 1, 32, 0, 1),
                                                     (0, 0, 1, 1, 1, 33, 0, 1), (0, 0, 1, 0, 1, 32, 0, 1))] == [0] * 4
    assert lib.gpuq_route_group_work(4096, 64) == 0 and lib.gpuq_route_group_work(4097, 64) == 2 * 64 * 4
    assert lib.gpuq_route_group_work(1 << 21, 64) == 128 * 64 * 4


def test_nothing_runs_before_init(lib):
    if lib.gpuq_can_dequantize_type(23) == 1:
        pytest.skip("the library was initialized earlier in this process (GPU tests ran first)")
    assert lib.gpuq_mxfp4_quantize_dev(0, 4096, 1, 1, 32, 32, 0, 4096, None, None) == 0
    assert lib.gpuq_mxfp4_matmul_dev(30, 4096, 1, 32, 4096, None, 1, 1, 32, None, None, 1, 0, 4096, None, None) == 0
    assert lib.gpuq_route_dev(0, 4096, 1, 8, 8, 2, 0, None, 1, 1, 1, 1.0, 4096, 4096, None) == 1
    assert lib.gpuq_route_group_dev(4096, 1, 2, 8, 4096, 4096, 4096, None, None) == 1
