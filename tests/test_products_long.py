"""Long sums of the grouped products.

Tolerances.  A result held in type t is at most half a step off, eps(t) / 2 of its value.  A step of the
tensor cores adds 16 products to a sum in fp32 and may cut off what is below 2^-23 of that sum in
each of the 17 terms; a sum is added up in parts of 8192 terms, 512 steps, and the parts are
rounded to the nearest.  Positive terms of one distribution add up evenly, so the sum is on
average half of the part's: at most 17 * 513 * 2^-24 of the result is cut off."""
import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CUT = 17 * 513 * 2.0 ** -24


def ext():
    from pilotann_b200 import extension
    return extension


def positive(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (0.1 + 0.1 * torch.rand(shape, generator=g, device="cuda")).to(dtype)


def blocks_product(a, b):
    """a @ b.T in 64 bits, some of the summed axis at a time."""
    return sum(a[:, i:i + 65536].double() @ b[:, i:i + 65536].double().T
               for i in range(0, a.size(1), 65536))


def check(got, want):
    far = (got.double() - want) / want
    assert far.abs().max() <= torch.finfo(got.dtype).eps / 2 * (1 + CUT) + CUT


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,d,d_out", [(1 << 20, 64, 64), ((1 << 18) + 77, 64, 128),
                                          (1 << 18, 72, 200), ((1 << 18) + 1, 136, 264)])
def test_gradient_of_the_matrix_of_a_long_group(dtype, rows, d, d_out):
    x, dy = positive((rows, d), dtype, rows), positive((rows, d_out), dtype, d)
    if dtype == F16:
        x = x / 4           # sums within fp16's range
    # a few rows of a second group, so that the long one ends inside a slice's reach
    offsets = torch.tensor([0, rows - 37, rows], device="cuda")
    w = torch.zeros(2, d_out, d, device="cuda", dtype=dtype)
    _, dw = ext().project_grouped_backward(dy, x, w, offsets, want_query=False)
    for g, (lo, hi) in enumerate(((0, rows - 37), (rows - 37, rows))):
        check(dw[g], blocks_product(dy[lo:hi].T, x[lo:hi].T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,d,d_out", [([5], 65536, 136), ([40, 24], 40008, 264),
                                            ([100], 65536, 1000), ([2100], 20480, 2560),
                                            ([38000], 8256, 72)])
def test_products_over_a_long_axis(dtype, counts, d, d_out):
    """Forward, and the gradient of the rows with the axes in each other's place."""
    rows, n = sum(counts), len(counts)
    edges = [sum(counts[:i]) for i in range(n + 1)]
    offsets = torch.tensor(edges, device="cuda")
    x, w = positive((rows, d), dtype, rows), positive((n, d_out, d), dtype, d)
    y = ext().project_grouped(x, w, offsets)
    # w as [n, d, d_out]: the summed axis of the gradient of the rows is the long one
    dx, _ = ext().project_grouped_backward(x, torch.zeros(rows, d_out, device="cuda", dtype=dtype),
                                           w.transpose(1, 2).contiguous(), offsets, want_VT=False)
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        want = blocks_product(x[lo:hi], w[g])
        check(y[lo:hi], want)
        check(dx[lo:hi], want)
