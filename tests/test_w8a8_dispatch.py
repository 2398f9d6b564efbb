"""CPU: the launches that the entry points of the 8-bit layers make (tests/w8a8_launches.py), held against what a launch may be."""
import shutil

import pytest

torch = pytest.importorskip("torch")
import w8a8_launches  # noqa: E402

pytestmark = pytest.mark.skipif(shutil.which("gcc") is None, reason="builds the stand-in for the HIP calls")


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return w8a8_launches.build(tmp_path_factory.mktemp("fake"))


def within_limits(launched):
    for kernel, grid, block, lds, most in launched:
        assert grid[1] <= 65535 and grid[2] <= 65535, (kernel, grid)
        assert all(g * b < 1 << 32 for g, b in zip(grid, block)), (kernel, grid, block)
        n = 1
        for v in grid + block:
            n *= v
        assert n <= 1 << 32 and min(grid) >= 1, (kernel, grid, block)
        assert lds <= most, (kernel, lds, most)


# up to 64 * 65535 tokens, past them, and past what one launch of the few-token kernel holds
MANY = [64 * 65535, 64 * 65535 + 1, 5_000_000, 8_000_000, 534_773_760, 534_773_761, 1_000_000_000]


@pytest.mark.parametrize("K,N", [(31, 16), (33, 1), (63, 16), (127, 16), (31, 40)])
def test_rows_of_any_alignment_in_their_millions(fake, K, N):
    for M, (rc, launched) in zip(MANY, w8a8_launches.launches(fake, [dict(op="matmul", M=M, K=K, N=N) for M in MANY])):
        assert rc == 0 and launched, M
        within_limits(launched)
        kernel, grid = launched[-1][:2]
        blocks = grid[1] * grid[2] * 64 if "w8_few" in kernel else grid[0] * 256   # (256 tokens a block at the most)
        assert blocks >= M, (M, kernel, grid)


def test_every_launch_is_within_limits(fake):
    sizes = [(M, K, N) for M in (1, 17, 64, 65, 3772, 8193, 120704, 1 << 20, 1 << 24) for K in (1, 8, 31, 384, 513, 4096, 131071)
             for N in (1, 52, 513, 4097, 1 << 20)]
    calls = [dict(op=op, M=M, K=K, N=N, H=H, gap=gap) for M, K, N in sizes for op, H, gap in
             (("matmul", 0, -K % 16), ("matmul", 0, 1), ("linear", 0, 0), ("feed_forward", 33, 0), ("quantize", 0, 0))]
    for c, (rc, launched) in zip(calls, w8a8_launches.launches(fake, calls)):
        assert rc in (0, -1), c
        assert rc or launched, c
        within_limits(launched)


@pytest.mark.parametrize("large,small", [(dict(op="feed_forward", M=30000, K=64, H=512, N=64), dict(op="feed_forward", M=30000, K=64, H=512, N=48)),
                                         (dict(op="linear", M=64, K=512, N=64), dict(op="linear", M=60, K=512, N=64))])
@pytest.mark.parametrize("t", [0, 1, 2])
def test_two_first_calls_of_a_kernel_at_once(fake, large, small, t):
    """Calls of one kernel that need different amounts of LDS, the smaller one's on another thread while the larger one's is
    being granted: what is granted never gets less again."""
    large, small = dict(large, t=t), dict(small, t=t)
    for rc, launched in w8a8_launches.launches(fake, [dict(large, beside=small), large, small, large]):
        assert rc == 0 and launched
        within_limits(launched)
    (_, a), (_, b) = w8a8_launches.launches(fake, [large, small])
    assert a[0][0] == b[0][0] and a[0][3] > b[0][3]


def test_the_products_tested_on_the_gpu_take_every_kernel(fake):
    import itertools
    from test_gpu_w8a8_kernels import PRODUCTS
    calls = [dict(op="matmul", M=M, K=K, N=N, gap=-K % 16) for _, _, M, K, N in PRODUCTS]
    taken = set()
    for (kernel, split, M, K, N), (rc, launched) in zip(PRODUCTS, w8a8_launches.launches(fake, calls)):
        assert rc == 0 and kernel in launched[0][0] and len(launched) == 1 + split, (M, K, N, launched)
        within_limits(launched)
        taken.add((kernel, split))
    # no size of a grid over the range takes another one
    sizes = [2 ** i for i in range(0, 18, 2)], [16, 96, 384, 1536, 6144, 24576, 98304], [1, 16, 64, 130, 520, 2080, 8320, 33280]
    calls = [dict(op="matmul", M=M, K=K, N=N) for M, K, N in itertools.product(*sizes)]
    for c, (rc, launched) in zip(calls, w8a8_launches.launches(fake, calls)):
        assert rc == 0 and any(k in launched[0][0] and split == (len(launched) == 2) for k, split in taken), (c, launched)


def test_the_layers_tested_on_the_gpu_take_every_kernel(fake):
    from test_gpu_w8a8_kernels import FEED_FORWARD, LINEAR, QUANTIZE
    want = [(f"quantize_rows_kernelI{c}Li{lanes}E", dict(op="quantize", M=M, K=K, t=t)) for lanes, M, K in QUANTIZE
            for t, c in ((0, "f"), (1, "DF16_"), (2, "DF16b"))]
    want += [(k, dict(op="linear", M=M, K=K, N=N)) for k, M, K, N in LINEAR]
    want += [(k, dict(op="feed_forward", M=M, K=K, H=H, N=N)) for k, M, K, H, N in FEED_FORWARD]
    for (kernel, c), (rc, launched) in zip(want, w8a8_launches.launches(fake, [c for _, c in want])):
        assert rc == 0 and kernel in launched[0][0], (c, launched)
        within_limits(launched)
