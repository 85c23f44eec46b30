"""An output of the 8-bit projection depends on its own row and channel alone, to the bit: not on how many
rows there are (which decides between the kernels), nor on what stands in the other rows and channels."""
import pytest
import torch

from spiral_amd import ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def problem(m, k, n, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    return x, w, torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4, torch.randn(n, generator=g, device="cuda")


# rows that are held in one launch, few rows with a launch of their own, the rows kernel (up to 256 values), tiles
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k,n", [(40, 33), (128, 256), (256, 100), (300, 70), (640, 129), (2049, 40)])
def test_any_number_of_rows(dev, k, n, dtype):
    x, w, s, b = problem(600, k, n, dtype)
    for act in (None, "relu", "leaky_relu"):
        want = ops.linear_int8(x, w, s, b, act, out_dtype=F32)
        for m in (1, 2, 8, 16, 17, 40, 64, 65, 300):
            assert torch.equal(ops.linear_int8(x[:m], w, s, b, act, out_dtype=F32), want[:m]), m


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_rows_in_one_pass_and_in_tiles(dev, dtype):
    x, w, s, b = problem(65_536, 512, 72, dtype)
    want = ops.linear_int8(x, w, s, b, out_dtype=F32)
    for m in (5, 100, 3000):
        assert torch.equal(ops.linear_int8(x[:m], w, s, b, out_dtype=F32), want[:m])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k", [(9, 128), (50, 700), (300, 31), (300, 128), (300, 256), (300, 330), (300, 900), (1000, 520)])
def test_neighbours_of_rows_out_of_the_ordinary(dev, m, k, dtype):
    x, w, s, b = problem(m, k, 200, dtype)
    want = ops.linear_int8(x, w, s, b, out_dtype=F32)
    odd = torch.zeros(m, dtype=torch.bool, device=dev)
    odd[2::7] = True
    levels = [0.0, float("nan"), float("inf"), 1e38, 1e-38]
    changed = x.clone()
    rows = odd.nonzero()[:, 0]
    for i, level in enumerate(levels):
        changed[rows[i::len(levels)]] = level
    got = ops.linear_int8(changed, w, s, b, out_dtype=F32)
    assert torch.equal(got[~odd], want[~odd])
    lost = ~changed.isfinite().all(1)
    # (a row of 1e38 may pass float32's range: 1e38 * 127 * 700 * 0.01 = 9e40; what is lost is not a number)
    assert bool(got[lost].isnan().all()) and not bool(got[~lost].isnan().any())
    zero = (changed == 0).all(1)
    assert torch.equal(got[zero], b.expand(int(zero.sum()), -1))


@pytest.mark.parametrize("m,k", [(9, 128), (50, 700), (300, 128), (300, 900)])
def test_neighbours_of_channels_out_of_the_ordinary(dev, m, k):
    x, w, s, b = problem(m, k, 200, F32)
    want = ops.linear_int8(x, w, s, b)
    odd = torch.zeros(200, dtype=torch.bool, device=dev)
    odd[5::11] = True
    t = s.clone()
    t[5::33], t[16::33], t[27::33] = 0.0, 1e-30, 1e25
    assert torch.equal(ops.linear_int8(x, w, t, b)[:, ~odd], want[:, ~odd])


@pytest.mark.parametrize("m", [0, 1, 2])
def test_rows_far_apart(dev, m):
    """Rows 2^24 values and more apart: copied where there are several, and a single one has no distance."""
    x, w, s, b = problem(2, 128, 40, BF16)
    wide = torch.zeros(2, 1 << 24, dtype=BF16, device=dev)
    wide[:, 5:133] = x
    assert torch.equal(ops.linear_int8(wide[:m, 5:133], w, s, b), ops.linear_int8(x[:m], w, s, b))
    q, scale = ops.quantize_rows_int8(wide[:m, 5:133])
    want = ops.quantize_rows_int8(x[:m])
    assert torch.equal(q, want[0]) and torch.equal(scale, want[1])
