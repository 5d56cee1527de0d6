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


@pytest.mark.parametrize("call", [forward, gradient_of_rows, gradient_of_matrices])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,d,d_out", [c for c in GROUPED if 0 not in c[0]])
def test_a_product_that_gave_up_is_nan_and_the_next_one_raises(library, call, dtype, counts, d, d_out):
    """No warp has waited for a sum, so no tile was stored.  The kernel is over without a second
    launch, and what was not started never is."""
    from pilotann_b200 import extension as e
    g = torch.Generator(device="cuda").manual_seed(d)
    rows, n = sum(counts), len(counts)
    x = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    w = torch.randn(n, d_out, d, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, d_out, generator=g, device="cuda").to(dtype)
    offsets = torch.tensor([sum(counts[:i]) for i in range(n + 1)], device="cuda")
    library.pa_selftest_sum_polls(0)
    got = call(e, x, w, dy, offsets)
    library.pa_selftest_sum_polls(-1)
    torch.cuda.synchronize()
    assert got.isnan().all()
    for again in (lambda: call(e, x, w, dy, offsets),
                  lambda: e.project_grouped_backward(dy, x, w, offsets),
                  lambda: e.project_fp4(x, e.quantize_fp4(w), offsets)):
        with pytest.raises(RuntimeError, match="gave up"):
            again()
    # the router's scores are another kernel's: nothing distrusts them
    assert library.pa_device_status(1) == 1 and library.pa_device_status(0) == 0
    assert not call(e, x, w, dy, offsets).isnan().any()


@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("out", [F32, BF16, F16])
def test_scores_that_gave_up_are_nan(library, method, out):
    from pilotann_b200 import extension as e
    q = e.quantize_fp4(torch.randn(300, 200, device="cuda"), method)
    t = e.quantize_fp4(torch.randn(30001, 200, device="cuda"), method)
    library.pa_selftest_sum_polls(0)
    got = e.project_fp4(q, t, dtype=out)
    library.pa_selftest_sum_polls(-1)
    torch.cuda.synchronize()
    assert got.isnan().all()
    with pytest.raises(RuntimeError, match="gave up"):
        e.project_fp4(q, t)
    assert library.pa_device_status(1) == 1
    assert not e.project_fp4(q, t, dtype=out).isnan().any()


def test_a_replayed_product_that_gave_up_is_nan(library):
    """A graph keeps the limit that it was captured with."""
    from pilotann_b200 import extension as e
    x = torch.randn(700, 264, device="cuda", dtype=BF16)
    w = torch.randn(2, 136, 264, device="cuda", dtype=BF16)
    offsets = torch.tensor([0, 300, 700], device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    library.pa_selftest_sum_polls(0)
    with torch.cuda.graph(graph):
        y = e.project_grouped(x, w, offsets)
    library.pa_selftest_sum_polls(-1)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert y.isnan().all()
    assert library.pa_device_status(1) == 1
