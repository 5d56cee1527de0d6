"""4-bit codes, bit by bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def values(law, rows, d, dtype):
    g = torch.Generator().manual_seed(rows * 7 + d)
    x = torch.randn(rows, d, generator=g)
    if law == "borders":       # multiples of a quarter, many of them half way between levels
        x = torch.randint(-28, 29, (rows, d), generator=g) / 4.0
    if law == "small":         # next to large ones: most become zeros of either sign
        x[torch.rand(rows, d, generator=g) < 0.7] *= 0.01
    if law == "wide":
        x = x * torch.exp2(torch.randint(-14, 15, (rows, d), generator=g).float())
    if law == "zeros":
        x[:, : d // 2] = 0.0
        x[::2] = -0.0
    return x.to(dtype)


@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("law", ["normal", "borders", "small", "wide", "zeros"])
@pytest.mark.parametrize("rows,d", [(1, 1), (7, 31), (5, 33), (64, 96), (33, 200), (16, 768),
                                    (3, 4099)])
def test_codes_do_not_depend_on_the_type(method, dtype, law, rows, d):
    """Values of 16 bits and the same ones in 32 have the same codes, signs of zeros included, and
    the same scales."""
    from pilotann_b200 import extension as e
    x = values(law, rows, d, dtype).cuda()
    a, b = e.quantize_fp4(x, method), e.quantize_fp4(x.float(), method)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert method == "mxfp4" or torch.equal(a.row_scale, b.row_scale)
