"""Products whose bounded wait runs out: they wait for what they have started, return, and leave the
GPU as it was.  Nothing faults, traps or hangs: the warps that store do not wait for the first sum,
and take the rest of their CTA along."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def forward(e, x, w, dy, offsets):
    return e.project_grouped(x, w, offsets)


def gradient_of_rows(e, x, w, dy, offsets):
    return e.project_grouped_backward(dy, x, w, offsets, want_VT=False)[0]


def gradient_of_matrices(e, x, w, dy, offsets):
    return e.project_grouped_backward(dy, x, w, offsets, want_query=False)[1]


# rows per group, d, d_out: tiles of 16 to 256 columns by one CTA, then pairs; the gradients of the
# matrices with last slices of 64, 16 and 1 rows
GROUPED = [([2] * 100, 264, 136), ([100, 28], 128, 264), ([300, 340], 136, 2504),
           ([20000, 20000], 72, 72), ([1041, 1040, 1039], 520, 776), ([64, 0, 2001], 264, 300)]


@pytest.fixture
def library():
    from pilotann_b200 import _C
    lib = _C.lib()
    lib.pa_device_status(1)
    yield lib
    lib.pa_selftest_sum_polls(-1)
    lib.pa_device_status(1)


@pytest.mark.parametrize("call", [forward, gradient_of_rows, gradient_of_matrices])
@pytest.mark.parametrize("counts,d,d_out", GROUPED)
def test_a_grouped_product_gives_up(library, call, counts, d, d_out):
    from pilotann_b200 import extension as e
    g = torch.Generator(device="cuda").manual_seed(d)
    rows, n = sum(counts), len(counts)
    x = torch.randn(rows, d, generator=g, device="cuda").to(BF16)
    w = torch.randn(n, d_out, d, generator=g, device="cuda").to(BF16)
    dy = torch.randn(rows, d_out, generator=g, device="cuda").to(BF16)
    offsets = torch.tensor([sum(counts[:i]) for i in range(n + 1)], device="cuda")
    want = call(e, x, w, dy, offsets)
    assert library.pa_device_status(0) == 0
    library.pa_selftest_sum_polls(0)
    call(e, x, w, dy, offsets)
    assert library.pa_device_status(1) == 1
    library.pa_selftest_sum_polls(-1)
    assert torch.equal(call(e, x, w, dy, offsets), want)
    assert library.pa_device_status(0) == 0


@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,d,d_out", [(1, 768, 40000), (20, 200, 5000), (50, 96, 20000),
                                          (100, 4096, 3000), (700, 520, 2000)])
def test_a_product_of_4_bit_rows_gives_up(library, method, rows, d, d_out):
    from pilotann_b200 import extension as e
    g = torch.Generator(device="cuda").manual_seed(d)
    q = e.quantize_fp4(torch.randn(rows, d, generator=g, device="cuda"), method)
    t = e.quantize_fp4(torch.randn(d_out, d, generator=g, device="cuda"), method)
    want = e.project_fp4(q, t)
    library.pa_selftest_sum_polls(0)
    e.project_fp4(q, t)
    assert library.pa_device_status(1) == 1
    library.pa_selftest_sum_polls(-1)
    assert torch.equal(e.project_fp4(q, t), want)
    assert library.pa_device_status(0) == 0
