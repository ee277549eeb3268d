"""Layer norm on the GPU: rows whose sums are exact in 32 bits, so that their
means are to be right to the last bit."""

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from veles.znicz_amd import ops  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E32 = 2.0 ** -24
#: with the values below, of at most 10 bits, sums of so many are exact
WIDTHS = [1, 3, 7, 13, 15, 28, 63, 95, 250, 500, 1000, 1021, 2049, 3000, 4097,
          8191, 9999, 16384, 16385, 20001, 33000]
VALUES = [3.0, 100.0, 1000.0, -10000.0, 0.625]


def values_of(dtype):
    return torch.tensor(VALUES, dtype=dtype, device="cuda")


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("name", sorted(TYPES))
def test_rows_of_equal_values_give_the_shift(C, name):
    """Nothing of a row is left without its mean: y is the shift, and the
    deviation is that of eps, however large the values are."""
    dtype, R, eps = TYPES[name], 11, 1e-5
    v = values_of(dtype).repeat(3)[:R]
    x = v[:, None].expand(R, C).contiguous()
    rng = numpy.random.RandomState(C)
    w = torch.from_numpy(rng.normal(1, 0.3, C).astype("f4")).cuda()
    b = torch.from_numpy(rng.normal(0, 0.3, C).astype("f4")).cuda()
    y = torch.empty_like(x)
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    ops.layer_norm_fwd(x, y, w, b, mean, rstd, eps)
    # (33000 values of 10 bits: 26 bits, in steps that even numbers have)
    assert torch.equal(mean, v.float())
    assert torch.equal(y, b.to(dtype).expand(R, C))
    want = 1 / numpy.sqrt(numpy.float64(numpy.float32(eps)))
    # the square root and the division are off by half a step each, or the
    # reciprocal square root by one
    assert (numpy.abs(rstd.double().cpu().numpy() - want) <=
            want * 3 * E32).all()


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("name", sorted(TYPES))
def test_equal_gradients_of_equal_values_are_none(C, name):
    """err_output of one value has no part that moves a row."""
    dtype, R = TYPES[name], 11
    dy = values_of(dtype).repeat(3)[:R, None].expand(R, C).contiguous()
    x = torch.full_like(dy, 3.0)
    mean = torch.full((R,), 3.0, device="cuda")
    rstd = torch.full((R,), 316.25, device="cuda")
    dx = torch.full_like(dy, 55.0)
    dw, db = torch.empty(C).cuda(), torch.empty(C).cuda()
    ops.layer_norm_bwd(dy, x, None, mean, rstd, dx, dw, db)
    assert (dx == 0).all()
    assert (dw == 0).all()
    only = torch.full_like(dy, 55.0)
    ops.layer_norm_bwd(dy, x, None, mean, rstd, only)
    assert (only == 0).all()


@pytest.mark.parametrize("C", [7, 96, 1000, 4097, 20001, 33000])
def test_means_beyond_all_numbers(C):
    """A sum that is infinite leaves the mean that, as before."""
    x = torch.zeros(3, C, device="cuda")
    x[0, C - 1] = float("inf")
    x[1, 0] = -float("inf")
    x[2, 0] = float("nan")
    mean, rstd = torch.empty(3).cuda(), torch.empty(3).cuda()
    ops.layer_norm_fwd(x, torch.empty_like(x), None, None, mean, rstd)
    assert mean[0] == float("inf") and mean[1] == -float("inf")
    assert torch.isnan(mean[2]) and torch.isnan(rstd).all()
