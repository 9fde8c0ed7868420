"""What the documentation of the panel operators says beyond their formulas, on the GPU."""
import pytest
import torch

from spla_amd import kernels

pytestmark = pytest.mark.gpu


def test_a_norm_beyond_fp32():
    """1000 values of 3e38: the norm, 9.5e39, reads as infinity in 32 bits.  Computed inside, it scales (by 64 bits); given as the 32-bit infinity, it does not, in place or into `out`."""
    values = torch.full((1000,), 3e38, device="cuda")
    norm = kernels.global_norm([values])
    assert float(norm) == float("inf")
    kept, out = values.clone(), [torch.zeros_like(values)]
    assert kernels.clip_global_norm([values], 1.0, out=out, norm=norm) is norm
    assert torch.equal(values, kept) and torch.equal(out[0], kept)
    kernels.clip_global_norm([values], 1.0, norm=norm)
    assert torch.equal(values, kept)
    assert float(kernels.clip_global_norm([values], 1.0, out=out)) == float("inf")
    # every value is 1000 ** -0.5 now: off by the factor's rounding, the product's and that of 3e38 to the input's type (which the factor takes out again)
    want = 1000 ** -0.5
    assert ((out[0].double() - want).abs() <= want * 3 * 2.0 ** -24).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_given_norm_that_is_not_finite_scales_nothing(dtype, bad):
    t = [torch.arange(3001, device="cuda").to(dtype), torch.ones(5, device="cuda")]
    kept = [x.clone() for x in t]
    kernels.clip_global_norm(t, 0.25, norm=torch.tensor(bad, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(t, kept))
