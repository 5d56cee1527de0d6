"""Products of grouped rows and 4-bit tables against plain 64-bit computations.

Tolerances.  A result held in type t is at most half a step off, eps(t) / 2 of its value (plus
half the smallest subnormal).  A sum of n products in fp32 whose every addition may be cut off
instead of rounded is off by at most (n + 1) 2^-23 sum |a||b|; both are added, nothing else is
allowed for.  Quantised values have no tolerance."""
import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ext():
    from pilotann_b200 import extension
    return extension


def off_by(got, want, magnitude, n):
    """Largest excess of |got - want| over what the rounding of a sum of n products allows."""
    t = torch.finfo(got.dtype)
    slip = (n + 1) * 2.0 ** -23 * magnitude
    allowed = t.eps / 2 * (want.abs() + slip) + slip + t.smallest_normal * t.eps / 2
    far = (got.double() - want).abs()
    assert not torch.isnan(far).any()
    return (far - allowed).max().item() if far.numel() else 0.0


def offsets_of(counts, before=0):
    return torch.tensor([before] + [before + sum(counts[:i + 1]) for i in range(len(counts))])


# ---- refusals, on the CPU ---------------------------------------------------------------
def test_c_entry_points_refuse_bad_arguments():
    from pilotann_b200 import _C
    L = _C.lib()

    def refused(rc, text):
        assert rc == _C.PA_ERR_ARG and text in L.pa_last_error(), L.pa_last_error()

    refused(L.pa_group_rows(0, 0, 0, 4, 0, 0, 0), b"n_groups")
    refused(L.pa_group_rows(0, 0, 0, 4, 1025, 0, 0), b"n_groups")
    refused(L.pa_group_rows(0, 0, 0, 1 << 31, 4, 0, 0), b"rows")
    refused(L.pa_group_rows(0, 0, 0, 4, 4, 0, 0), b"null")
    refused(L.pa_group_rows(16, 16, 16, 100000, 4, 0, 0), b"workspace")
    refused(L.pa_project_grouped(0, 0, 0, 0, 4, 2, 0, 8, 8, 8, 0, 0, 0), b"d_out")
    refused(L.pa_project_grouped(0, 0, 0, 0, 4, 2, 8, 65537, 8, 65537, 0, 0, 0), b"d_out")
    refused(L.pa_project_grouped(0, 0, 0, 0, 4, 2, 8, 8, 7, 8, 0, 0, 0), b"strides")
    refused(L.pa_project_grouped(0, 0, 0, 0, 4, 2, 8, 8, 8, 8, 3, 0, 0), b"dtype")
    refused(L.pa_project_grouped(0, 0, 0, 0, 4, 2, 8, 8, 8, 8, 0, 0, 0), b"null")
    refused(L.pa_project_grouped_backward(16, 0, 0, 0, 0, 0, 4, 2, 8, 8, 8, 8, 7, 0, 0, 0), b"strides")
    refused(L.pa_project_grouped_backward(0, 16, 0, 0, 0, 0, 4, 2, 8, 8, 8, 8, 8, 0, 0, 0), b"null")
    refused(L.pa_quantize_fp4(0, 0, 0, 0, 4, 0, 8, 0, 0, 0), b"d must")
    refused(L.pa_quantize_fp4(0, 0, 0, 0, 4, 8, 4, 0, 0, 0), b"stride")
    refused(L.pa_quantize_fp4(0, 0, 0, 0, 4, 8, 8, 0, 2, 0), b"method")
    refused(L.pa_quantize_fp4(8, 16, 16, 16, 4, 8, 8, 0, 1, 0), b"aligned")
    refused(L.pa_dequantize_fp4(0, 0, 0, 0, 4, 8, 1, 0), b"null")
    refused(L.pa_project_fp4(0, 0, 0, 0, 0, 0, 0, 0, 4, 2, 8, 8, 0, 0, 0), b"offsets")
    refused(L.pa_project_fp4(0, 0, 0, 0, 0, 0, 0, 0, 4, 1, 8, 1 << 31, 0, 0, 0), b"table rows")
    refused(L.pa_project_fp4(0, 0, 0, 0, 0, 0, 0, 0, 4, 1, 8, 8, 7, 0, 0), b"dtype")
    refused(L.pa_project_fp4(16, 16, 16, 0, 16, 16, 0, 0, 4, 1, 8, 8, 0, 1, 0), b"row scales")
    refused(L.pa_project_grouped(16, 16, 16, 16, 4, 2, 9, 8, 9, 8, 1, 0, 0), b"workspace")
    refused(L.pa_project_grouped(16, 17, 16, 16, 4, 2, 8, 8, 8, 8, 1, 0, 0), b"aligned")
    refused(L.pa_project_grouped(18, 16, 16, 16, 4, 2, 8, 8, 8, 8, 0, 0, 0), b"aligned")
    refused(L.pa_quantize_fp4(16, 16, 16, 18, 4, 8, 8, 0, 0, 0), b"aligned")
    refused(L.pa_project_fp4(17, 16, 16, 0, 16, 16, 0, 0, 4, 1, 8, 8, 1, 0, 0), b"aligned")
    refused(L.pa_project_grouped_backward(16, 0, 16, 0, 16, 16, 4, 2, 8, 9, 9, 8, 8, 1, 0, 0),
            b"workspace")
    assert L.pa_project_grouped_workspace_bytes(16, 16, 4, 2, 8, 8, 8, 1) == 0
    assert L.pa_project_grouped_workspace_bytes(18, 16, 4, 2, 8, 8, 8, 1) == 4 * 8 * 2
    assert L.pa_project_grouped_workspace_bytes(16, 16, 4, 2, 9, 8, 9, 1) == (4 + 2 * 8) * 16 * 2
    assert L.pa_group_rows_workspace_bytes(8192, 64) == 0
    assert L.pa_group_rows_workspace_bytes(8193, 64) >= 3 * 65 * 4


def test_cpu_tensors_are_refused():
    e = ext()
    x, w, o = torch.zeros(4, 32), torch.zeros(2, 8, 32), torch.tensor([0, 2, 4])
    for call in (lambda: e.group_rows(o, 2), lambda: e.project_grouped(x, w, o),
                 lambda: e.project_grouped_backward(x, x, w, o), lambda: e.quantize_fp4(x),
                 lambda: e.Fp4Table(torch.zeros(4, 16, dtype=torch.uint8),
                                    torch.zeros(4, 1, dtype=torch.uint8), None, 32, "mxfp4")):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="Fp4Table"):
        e.project_fp4(x, x)
    with pytest.raises(RuntimeError, match="Fp4Table"):
        e.dequantize_fp4(x)
    with pytest.raises(RuntimeError, match="unknown 4-bit method"):
        e.quantize_fp4(x, "fp4")


@pytest.mark.gpu
def test_wrong_tensors_are_refused():
    e = ext()
    x, w = torch.zeros(4, 32, device="cuda"), torch.zeros(2, 8, 32, device="cuda")
    o = torch.tensor([0, 2, 4], device="cuda")

    def refused(call, text):
        with pytest.raises(RuntimeError, match=text):
            call()

    refused(lambda: e.group_rows(o.int(), 2), "int64")
    refused(lambda: e.group_rows(o, 0), "n_groups")
    refused(lambda: e.group_rows(o, 1025), "n_groups")
    refused(lambda: e.group_rows(torch.zeros(4, 2, dtype=torch.int64, device="cuda")[:, 0], 2),
            "contiguous")
    refused(lambda: e.project_grouped(x.double(), w, o), "query must be type")
    refused(lambda: e.project_grouped(x.half(), w, o), "VT must be type")
    refused(lambda: e.project_grouped(x, w, o[:2]), "offsets.size")
    refused(lambda: e.project_grouped(x, w, o.int()), "int64")
    refused(lambda: e.project_grouped(x, w, o.cpu()), "CUDA tensor")
    refused(lambda: e.project_grouped(x[:, :16], w, o), "VT.size")
    refused(lambda: e.project_grouped(x, w.transpose(1, 2), o), "contiguous")
    refused(lambda: e.project_grouped(x.t().contiguous().t(), w, o), "contiguous rows")
    refused(lambda: e.project_grouped(x[:1].expand(4, 32), w, o), "contiguous rows")
    refused(lambda: e.project_grouped(x, torch.zeros(0, 8, 32, device="cuda"), o[:1]), "VT.size")
    refused(lambda: e.project_grouped_backward(x, x, w, o), "grad.shape")
    refused(lambda: e.quantize_fp4(x.double()), "must be type")
    refused(lambda: e.quantize_fp4(x[0]), "dim")
    refused(lambda: e.quantize_fp4(torch.zeros(2, 0, device="cuda")), "d <=")
    t = e.quantize_fp4(x, "nvfp4")
    refused(lambda: e.project_fp4(x, t, dtype=torch.float64), "dtype")
    refused(lambda: e.project_fp4(x[:, :16], t), "table.d")
    refused(lambda: e.project_fp4(x, t, o), "offsets")
    refused(lambda: e.project_fp4(x, e.quantize_fp4(w)), "offsets")
    refused(lambda: e.project_fp4(e.quantize_fp4(x), t), "method")
    refused(lambda: e.Fp4Table(t.codes, t.scales, None, 32, "nvfp4"), "row_scale")
    refused(lambda: e.Fp4Table(t.codes, t.scales, t.row_scale, 33, "nvfp4"), "codes")
    refused(lambda: e.Fp4Table(t.codes, t.scales, None, 32, "mxfp4"), "scales")


# ---- rows by group -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n_groups", [(0, 3), (1, 1), (31, 2), (33, 64), (1024, 64),
                                           (1000, 1024), (8192, 5), (8193, 5), (20000, 33),
                                           (100003, 1024), (300000, 1)])
@pytest.mark.parametrize("law", ["even", "one", "outside"])
def test_group_rows_is_a_stable_sort(rows, n_groups, law):
    g = torch.Generator().manual_seed(rows + n_groups)
    ids = torch.randint(n_groups, (rows,), generator=g)
    if law == "one":
        ids[:] = n_groups - 1
    if law == "outside":
        at = torch.rand(rows, generator=g)
        ids[at < 0.2] = -1
        ids[(at > 0.2) & (at < 0.3)] = n_groups
        ids[(at > 0.3) & (at < 0.4)] = (1 << 40) + 1
        ids[(at > 0.4) & (at < 0.5)] = -(1 << 62)
    order, offsets = ext().group_rows(ids.cuda(), n_groups)
    key = torch.where((ids >= 0) & (ids < n_groups), ids, torch.full_like(ids, n_groups))
    assert torch.equal(order.cpu(), torch.sort(key, stable=True)[1])
    count = torch.bincount(key, minlength=n_groups + 1)
    assert torch.equal(offsets.cpu(), torch.cumsum(count, 0) - count)


# ---- a matrix per group ----------------------------------------------------------------------
def grouped_plain(x, w, dy, offsets):
    """y, dx, dw in 64 bits, and the sums of magnitudes beside them."""
    x, w, dy = x.double(), w.double(), dy.double()
    y, dx, dw = x.new_zeros(dy.shape), torch.zeros_like(x), torch.zeros_like(w)
    ay, ax, aw = torch.zeros_like(y), torch.zeros_like(dx), torch.zeros_like(dw)
    edges = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        a, b = x[lo:hi], dy[lo:hi]
        y[lo:hi], ay[lo:hi] = a @ w[g].T, a.abs() @ w[g].abs().T
        dx[lo:hi], ax[lo:hi] = b @ w[g], b.abs() @ w[g].abs()
        dw[g], aw[g] = b.T @ a, b.abs().T @ a.abs()
    return (y, dx, dw), (ay, ax, aw)


GROUPS = {                     # rows per group, rows before the first, behind the last
    "one": ([1], 0, 0),
    "single row of many": ([0, 0, 1, 0], 0, 0),
    "ragged": ([3, 0, 64, 65, 1, 0, 130], 0, 0),
    "outside": ([17, 0, 70], 5, 9),
    "tiles": ([128, 256, 64], 0, 64),
    "long": ([777], 0, 0),
    "many": ([i % 5 for i in range(200)], 0, 3),
    "empty": ([0, 0], 0, 7),
}
WIDTHS = [(1, 1), (17, 33), (64, 128), (96, 64), (200, 333), (136, 264), (768, 40), (520, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("d,d_out", WIDTHS)
def test_grouped_products_and_gradients(dtype, groups, d, d_out):
    counts, before, behind = GROUPS[groups]
    offsets = offsets_of(counts, before)
    rows, n = before + sum(counts) + behind, len(counts)
    g = torch.Generator().manual_seed(d * 1000 + d_out)
    x = torch.randn(rows, d, generator=g).to(dtype).cuda()
    w = torch.randn(n, d_out, d, generator=g).to(dtype).cuda()
    dy = torch.randn(rows, d_out, generator=g).to(dtype).cuda()
    want, size = grouped_plain(x, w, dy, offsets)
    x.requires_grad_(True), w.requires_grad_(True)
    y = ext().project_grouped(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for name, got, n_sum, i in (("y", y, d, 0), ("dx", dx, d_out, 1), ("dw", dw, max(counts), 2)):
        assert got.dtype == dtype and got.shape == want[i].shape
        assert off_by(got, want[i], size[i], n_sum) <= 0, name
    outside = torch.ones(rows, dtype=torch.bool)
    outside[before:before + sum(counts)] = False
    assert not y[outside].any() and not dx[outside].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,d,d_out", [
    ([1000, 0, 1, 3000, 257, 742], 512, 640),       # tiles of 256 x 256, many a CTA
    ([2500, 77, 2423], 320, 1100),                  # both sides ragged
    ([i % 3 for i in range(1024)], 72, 136),        # the most groups
    ([0] * 1023 + [40], 264, 72),
    ([20000], 24, 72),                              # a long sum, few tiles
    ([5], 4096, 24),
])
def test_large_grouped_products(dtype, counts, d, d_out):
    """Kernels for large groups, the largest number of groups and long sums; twice, with the same
    bits."""
    e, offsets = ext(), offsets_of(counts)
    rows, n = sum(counts), len(counts)
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    w = torch.randn(n, d_out, d, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, d_out, generator=g, device="cuda").to(dtype)
    want, size = grouped_plain(x, w, dy, offsets)
    offsets = offsets.cuda()
    y = e.project_grouped(x, w, offsets)
    dx, dw = e.project_grouped_backward(dy, x, w, offsets)
    for got, n_sum, i in ((y, d, 0), (dx, d_out, 1), (dw, max(counts), 2)):
        assert off_by(got, want[i], size[i], n_sum) <= 0
    again = e.project_grouped_backward(dy, x, w, offsets)
    assert torch.equal(e.project_grouped(x, w, offsets), y)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.gpu
def test_fp32_sums_stay_exact_over_long_axes():
    """65536 rows in one sum: the error of a sum kept in levels of 256 terms is that of about
    2 * 16 roundings of random sign, 2^-24 each, of the size of the result (a single running sum
    has 256 of them)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(65536, 40, generator=g, device="cuda")
    dy = torch.randn(65536, 48, generator=g, device="cuda")
    w = torch.zeros(1, 48, 40, device="cuda")
    _, dw = ext().project_grouped_backward(dy, x, w, torch.tensor([0, 65536], device="cuda"),
                                           want_query=False)
    want = dy.double().T @ x.double()
    assert (dw[0].double() - want).norm() / want.norm() < 32 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("want", [(True, False), (False, True)])
def test_gradient_of_one_side(want):
    x = torch.randn(40, 64, device="cuda", dtype=BF16, requires_grad=want[0])
    w = torch.randn(2, 32, 64, device="cuda", dtype=BF16, requires_grad=want[1])
    offsets = torch.tensor([0, 20, 40], device="cuda")
    dy = torch.randn(40, 32, device="cuda", dtype=BF16)
    ext().project_grouped(x, w, offsets).backward(dy)
    both = ext().project_grouped_backward(dy, x.detach(), w.detach(), offsets)
    assert (x.grad is None) != want[0] and (w.grad is None) != want[1]
    assert torch.equal(x.grad if want[0] else w.grad, both[0 if want[0] else 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_rows_of_wider_tensors(dtype, shift):
    """Rows start anywhere in wider ones: row strides and alignments other than the row's own."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(150, 211, generator=g).to(dtype).cuda()
    wide_dy = torch.randn(150, 163, generator=g).to(dtype).cuda()
    x, dy = wide[:, shift:shift + 136], wide_dy[:, shift:shift + 72]
    w = torch.randn(3, 72, 136, generator=g).to(dtype).cuda()
    offsets = offsets_of([70, 0, 80])
    want, size = grouped_plain(x, w, dy, offsets)
    y = ext().project_grouped(x, w, offsets.cuda())
    dx, dw = ext().project_grouped_backward(dy, x, w, offsets.cuda())
    for got, n_sum, i in ((y, 136, 0), (dx, 72, 1), (dw, 80, 2)):
        assert off_by(got, want[i], size[i], n_sum) <= 0
    only_x, none = ext().project_grouped_backward(dy, x, w, offsets.cuda(), want_VT=False)
    none_x, only_w = ext().project_grouped_backward(dy, x, w, offsets.cuda(), want_query=False)
    assert none is None and none_x is None
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    # weights that start off a 16-byte boundary
    flat = torch.randn(3 * 72 * 136 + 1, generator=g).to(dtype).cuda()
    w = flat[1:].view(3, 72, 136)
    want, size = grouped_plain(x, w, dy, offsets)
    assert off_by(ext().project_grouped(x, w, offsets.cuda()), want[0], size[0], 136) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("counts", [[40, 3, 90], [130, 70, 129], [1, 1, 1]])
def test_a_group_does_not_see_its_neighbours(dtype, poison, counts):
    """NaN and infinity in one group's rows, gradients and matrix stay there."""
    g = torch.Generator().manual_seed(6)
    rows, d, d_out = sum(counts), 72, 136
    x, dy = torch.randn(rows, d, generator=g), torch.randn(rows, d_out, generator=g)
    w = torch.randn(3, d_out, d, generator=g)
    offsets = offsets_of(counts)
    lo, hi = offsets[1].item(), offsets[2].item()
    clean = [t.clone() for t in (x, w, dy)]
    x[lo:hi], dy[lo:hi], w[1] = poison, poison, poison
    x, w, dy = (t.to(dtype).cuda() for t in (x, w, dy))
    y = ext().project_grouped(x, w, offsets.cuda())
    dx, dw = ext().project_grouped_backward(dy, x, w, offsets.cuda())
    (wy, wx, ww), (ay, ax, aw) = grouped_plain(*(t.to(dtype).cuda() for t in clean), offsets)
    keep = torch.ones(rows, dtype=torch.bool)
    keep[lo:hi] = False
    assert off_by(y[keep], wy[keep], ay[keep], d) <= 0
    assert off_by(dx[keep], wx[keep], ax[keep], d_out) <= 0
    assert off_by(dw[::2], ww[::2], aw[::2], max(counts)) <= 0
    assert not torch.isfinite(y[lo:hi]).any() and not torch.isfinite(dx[lo:hi]).any()
    assert not torch.isfinite(dw[1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_against_differences(dtype):
    """The product is linear in the rows and in the matrices: a step h of either changes
    <dy, y> by exactly h times the gradient along it, whatever h is."""
    g = torch.Generator().manual_seed(7)
    offsets = offsets_of([30, 0, 41]).cuda()
    x = torch.randn(71, 48, generator=g).to(dtype).cuda()
    w = torch.randn(3, 40, 48, generator=g).to(dtype).cuda()
    dy = torch.randn(71, 40, generator=g).to(dtype).cuda()
    dx, dw = ext().project_grouped_backward(dy, x, w, offsets)
    eps = torch.finfo(dtype).eps
    for grad, at in ((dx, 0), (dw, 1)):
        step = torch.zeros_like(grad)
        where = torch.randperm(step.numel(), generator=g)[:50]
        step.view(-1)[where.cuda()] = 1.0
        there = [x, w]
        there[at] = step            # f(v + step) - f(v) = f(step)
        y = ext().project_grouped(there[0], there[1], offsets).double()
        change = (y * dy.double()).sum()
        along = (grad.double() * step.double()).sum()
        # every y and every gradient is rounded once, and is a sum cut off at most n times
        a = [there[0].double().abs(), there[1].double().abs(), dy.double().abs()]
        slack = grouped_plain(*a, offsets.cpu())[0]
        size = (slack[0] * a[2]).sum()
        assert (change - along).abs() <= (eps + 2 * 72 * 2.0 ** -23) * size


@pytest.mark.gpu
def test_gradient_of_a_sum_is_expanded():
    x = torch.randn(20, 24, device="cuda", requires_grad=True)
    w = torch.randn(2, 8, 24, device="cuda", requires_grad=True)
    offsets = torch.tensor([0, 5, 20], device="cuda")
    ext().project_grouped(x, w, offsets).sum().backward()
    want, size = grouped_plain(x.detach(), w.detach(), torch.ones(20, 8, device="cuda"),
                               offsets.cpu())
    assert off_by(x.grad, want[1], size[1], 8) <= 0 and off_by(w.grad, want[2], size[2], 15) <= 0


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(20, 24, device="cuda", requires_grad=True)
    w = torch.randn(2, 8, 24, device="cuda", requires_grad=True)
    y = ext().project_grouped(x, w, torch.tensor([0, 5, 20], device="cuda"))
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 40, 20, 64], [-5, 10, 20, 1000], [64, 32, 16, 0],
                                 [1 << 62, -(1 << 62), 7, 1 << 40]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_that_do_not_ascend_stay_inside(bad, dtype):
    """Unspecified results, but nothing outside the tensors: guard rows stay as they were.
    (Every offset is clamped to [0, rows] before it is used.)"""
    from pilotann_b200 import _C
    rows, d, d_out = 64, 64, 64
    x, w = torch.ones(rows, d, device="cuda", dtype=dtype), torch.ones(3, d_out, d, device="cuda",
                                                                      dtype=dtype)
    out = torch.full((rows + 256, d_out), 7.0, device="cuda", dtype=dtype)
    offsets = torch.tensor(bad, device="cuda")
    _C.check(_C.lib().pa_project_grouped(out.data_ptr() + 128 * d_out * out.element_size(),
                                         x.data_ptr(), w.data_ptr(), offsets.data_ptr(), rows, 3,
                                         d, d_out, d, d_out, 0 if dtype == F32 else 1, 0,
                                         torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (out[:128] == 7).all() and (out[128 + rows:] == 7).all()
    ext().project_grouped_backward(x, x, w, offsets)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows(dtype):
    e = ext()
    x, w = torch.zeros(0, 72, device="cuda", dtype=dtype), torch.ones(3, 40, 72, device="cuda", dtype=dtype)
    offsets = torch.zeros(4, dtype=torch.int64, device="cuda")
    dy = torch.zeros(0, 40, device="cuda", dtype=dtype)
    assert e.project_grouped(x, w, offsets).shape == (0, 40)
    dx, dw = e.project_grouped_backward(dy, x, w, offsets)
    assert dx.shape == (0, 72) and dw.shape == w.shape and not dw.any()
    for method in ("mxfp4", "nvfp4"):
        table = e.quantize_fp4(w, method)
        assert e.project_fp4(x, table, offsets).shape == (0, 40)
        none = e.quantize_fp4(x, method)
        assert e.dequantize_fp4(none).shape == (0, 72)
        assert e.project_fp4(w[0], none).shape == (40, 0)


@pytest.mark.gpu
def test_fp4_scores_past_2_31_elements():
    """40000 queries against 65536 vectors: offsets into the scores need more than 32 bits."""
    e = ext()
    q = torch.randn(40_000, 32, device="cuda", dtype=BF16)
    table = e.quantize_fp4(torch.randn(65_536, 32, device="cuda"), "nvfp4")
    codes = e.quantize_fp4(q, "nvfp4")
    got = e.project_fp4(codes, table, dtype=BF16)
    a, b = e.dequantize_fp4(codes).double(), e.dequantize_fp4(table).double()
    for lo in (0, 32_700, 39_900):
        part = a[lo:lo + 100]
        assert off_by(got[lo:lo + 100], part @ b.T, part.abs() @ b.abs().T, 32) <= 0


@pytest.mark.gpu
def test_outputs_past_2_31_elements():
    """600 000 rows of 4096 values: offsets into the result need more than 32 bits."""
    rows, d, d_out = 600_000, 16, 4096
    x = torch.randn(rows, d, device="cuda", dtype=BF16)
    w = torch.randn(2, d_out, d, device="cuda", dtype=BF16)
    offsets = torch.tensor([0, 300_001, rows], device="cuda")
    y = ext().project_grouped(x, w, offsets)
    for lo, g in ((0, 0), (300_000, 0), (300_001, 1), (599_900, 1)):
        hi = min(lo + 100, 300_001 if g == 0 else rows)
        a, b = x[lo:hi].double(), w[g].double()
        assert off_by(y[lo:hi], a @ b.T, a.abs() @ b.abs().T, d) <= 0


# ---- 4-bit blocks ---------------------------------------------------------------------------
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def nearest_level(v):
    """Index of the nearest level of |v|, of two at the same distance the even one."""
    far = (v.abs().clamp(max=6.0).unsqueeze(-1) - LEVELS).abs()
    least = far.min(-1, keepdim=True)[0]
    hit = far == least
    even = torch.tensor([1, 0] * 4, dtype=torch.bool)
    score = hit.int() * (1 + even.int())
    return score.argmax(-1)


def fp4_plain(x, method):
    """(values, scales) of rows x by the definition, in 64 bits on the CPU; quotients are
    rounded to fp32, as the definition has them."""
    x = x.double()
    rows, d = x.shape
    size = 32 if method == "mxfp4" else 16
    blocks = torch.nn.functional.pad(x, (0, -d % 32)).view(rows, -1, size)
    top = blocks.abs().amax(-1)
    if method == "mxfp4":
        power = torch.where(top > 0, torch.frexp(top)[1] - 1, -127) - 2
        step = torch.ldexp(torch.ones_like(top), power.clamp(min=-127))
        bad = ~top.isfinite()
    else:
        most = top.amax(-1, keepdim=True)
        part, power = torch.frexp(most / 2688.0)
        power = torch.where(part == 0.5, power - 1, power).clamp(min=-126)
        row = torch.ldexp(torch.ones_like(most), power)
        quotient = (top / row / 6.0).nan_to_num(0.0, 0.0).float()
        step = quotient.clamp(max=448.0).to(torch.float8_e4m3fn).double() * row
        bad = ~most.isfinite().expand_as(top)
    value = torch.where(step.unsqueeze(-1) > 0, (blocks / step.unsqueeze(-1)).float().double(),
                        0.0).nan_to_num(0.0, 0.0, 0.0)
    out = LEVELS[nearest_level(value)].copysign(value) * step.unsqueeze(-1)
    out[bad] = float("nan")
    return out.view(rows, -1)[:, :d], step


def fp4_inputs(law, rows, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + d)
    x = torch.randn(rows, d, generator=g)
    if law == "borders":       # multiples of a quarter, many of them half way between levels
        x = torch.randint(-28, 29, (rows, d), generator=g) / 4.0
    if law == "wide":          # from subnormal to the largest values of the type
        x = x * torch.exp2(torch.randint(-14, 15, (rows, d), generator=g).float())
        if dtype == F32:
            x = x * torch.exp2(torch.randint(-115, 105, (rows, 1), generator=g).float())
    if law == "zeros":
        x[:, : d // 2] = 0.0
        x[::2] = -0.0
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("law", ["normal", "borders", "wide", "zeros"])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 16), (7, 31), (9, 32), (5, 33), (64, 96), (33, 200),
                                    (16, 768), (3, 4099), (2, 8192)])
def test_fp4_codes_follow_the_definition(method, dtype, law, rows, d):
    x = fp4_inputs(law, rows, d, dtype)
    table = ext().quantize_fp4(x.cuda(), method)
    got = ext().dequantize_fp4(table).cpu().double()
    want, _ = fp4_plain(x, method)
    assert torch.equal(got, want.float().double())
    padded = -(-d // 32) * 32
    assert table.shape == (rows, d) and table.codes.shape == (rows, padded // 2)
    behind = table.codes.cpu().view(rows, -1)[:, (d + 1) // 2:]
    assert not (behind & 0x77).any()           # zero codes behind the row
    if method == "mxfp4":
        assert table.row_scale is None
    else:
        power = torch.frexp(table.row_scale.cpu())[0]
        assert (power == 0.5).all()            # powers of two


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_fp4_of_nan_and_infinity(dtype, poison):
    x = torch.randn(6, 96).to(dtype)
    x[2, 40] = poison
    mx = ext().dequantize_fp4(ext().quantize_fp4(x.cuda(), "mxfp4")).cpu()
    nv = ext().dequantize_fp4(ext().quantize_fp4(x.cuda(), "nvfp4")).cpu()
    assert mx[2, 32:64].isnan().all() and nv[2].isnan().all()
    clean = x.clone()
    clean[2, 40] = 0.0
    keep = torch.ones(6, 96, dtype=torch.bool)
    keep[2, 32:64] = False
    assert torch.equal(mx[keep], fp4_plain(clean, "mxfp4")[0].float()[keep])
    keep[2] = False
    assert torch.equal(nv[keep], fp4_plain(clean, "nvfp4")[0].float()[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
def test_fp4_rows_of_wider_tensors_and_tables_per_group(method):
    e = ext()
    wide = torch.randn(40, 301, device="cuda")
    for shift in (0, 1, 4):
        part = wide[:, shift:shift + 200]
        a, b = e.quantize_fp4(part, method), e.quantize_fp4(part.contiguous(), method)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    t = e.quantize_fp4(part.contiguous().view(4, 10, 200), method)
    assert t.shape == (4, 10, 200) and torch.equal(t.codes.view(40, -1), b.codes)
    assert torch.equal(e.dequantize_fp4(t).view(40, 200), e.dequantize_fp4(b))
    assert e.quantize_fp4(wide[:0], method).shape == (0, 301)
    assert t.nbytes() == 40 * (112 + (7 if method == "mxfp4" else 14 + 4))


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("rows,d,d_out", [(1, 1, 1), (1, 768, 1000), (3, 33, 130), (17, 200, 333),
                                          (64, 96, 64), (129, 776, 257), (300, 4100, 520),
                                          (700, 64, 1000)])
def test_fp4_scores(method, out, rows, d, d_out):
    e = ext()
    g = torch.Generator().manual_seed(rows + d)
    q = torch.randn(rows, d, generator=g).cuda()
    table = e.quantize_fp4(torch.randn(d_out, d, generator=g).cuda(), method)
    codes = e.quantize_fp4(q, method)
    a, b = e.dequantize_fp4(codes).double(), e.dequantize_fp4(table).double()
    got = e.project_fp4(q, table, dtype=out)
    assert got.dtype == out
    # row scales are powers of two and block scales products of few bits: no rounding but the sum
    assert off_by(got, a @ b.T, a.abs() @ b.abs().T, -(-d // 32) * 32) <= 0
    assert torch.equal(e.project_fp4(codes, table, dtype=out), got)
    # a query's scores do not depend on the batch it comes in, up to the order of its sum
    one = e.project_fp4(q[:1], table, dtype=out)
    assert off_by(one, (a @ b.T)[:1], (a.abs() @ b.abs().T)[:1], -(-d // 32) * 32) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("d,d_out", [(17, 33), (200, 333), (776, 260)])
def test_fp4_scores_by_group(method, groups, d, d_out):
    e = ext()
    counts, before, behind = GROUPS[groups]
    offsets = offsets_of(counts, before)
    rows = before + sum(counts) + behind
    g = torch.Generator().manual_seed(d)
    q = torch.randn(rows, d, generator=g).to(BF16).cuda()
    table = e.quantize_fp4(torch.randn(len(counts), d_out, d, generator=g).cuda(), method)
    a, b = e.dequantize_fp4(e.quantize_fp4(q, method)), e.dequantize_fp4(table)
    dy = torch.zeros(rows, d_out, device="cuda")
    want, size = grouped_plain(a, b, dy, offsets)
    got = e.project_fp4(q, table, offsets.cuda(), dtype=F32)
    assert off_by(got, want[0], size[0], -(-d // 32) * 32) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("up_q,up_t", [(40, 40), (-40, -40), (90, -90), (-100, 100), (0, -110)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_fp4_scores_of_large_and_small_values(method, up_q, up_t, out):
    """Scales far from one, on both sides: what one side's scale takes away the other gives back."""
    e = ext()
    g = torch.Generator().manual_seed(12)
    q = (torch.randn(33, 160, generator=g) * 2.0 ** up_q).cuda()
    t = (torch.randn(200, 160, generator=g) * 2.0 ** up_t).cuda()
    q[3], t[5] = 0.0, 0.0
    codes, table = e.quantize_fp4(q, method), e.quantize_fp4(t, method)
    a, b = e.dequantize_fp4(codes).double(), e.dequantize_fp4(table).double()
    got = e.project_fp4(codes, table, dtype=out)
    assert off_by(got, a @ b.T, a.abs() @ b.abs().T, 160) <= 0


@pytest.mark.gpu
def test_fp4_scores_of_extreme_row_scales():
    """Row scales whose product leaves fp32's range: zeros stay zeros, the rest is what it is."""
    e = ext()
    q = torch.full((3, 32), 2.0 ** 120, device="cuda")
    q[1] = 0.0
    q[2] = 2.0 ** -120
    t = torch.full((2, 32), 2.0 ** 120, device="cuda")
    t[1] = 2.0 ** -120
    got = e.project_fp4(e.quantize_fp4(q, "nvfp4"), e.quantize_fp4(t, "nvfp4"))
    want = torch.tensor([[float("inf"), 32.0], [0.0, 0.0], [32.0, 0.0]])
    # 2^120 and 2^-120 are not 6 times an E4M3 number: half a step of each side's scale and code
    assert torch.equal(got.isinf().cpu(), want.isinf())
    assert torch.allclose(got.cpu()[1:], want[1:], rtol=0.25) and torch.allclose(got[0, 1].cpu(), want[0, 1], rtol=0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,d,d_out", [(5000, 544, 3000), (2, 2080, 40000), (1, 65536, 40),
                                          (700, 512, 17)])
def test_large_fp4_scores(method, rows, d, d_out):
    """Many tiles a CTA, in units of several, and the longest rows."""
    e = ext()
    g = torch.Generator(device="cuda").manual_seed(d)
    codes = e.quantize_fp4(torch.randn(rows, d, generator=g, device="cuda").to(BF16), method)
    table = e.quantize_fp4(torch.randn(d_out, d, generator=g, device="cuda"), method)
    a, b = e.dequantize_fp4(codes).double(), e.dequantize_fp4(table).double()
    got = e.project_fp4(codes, table, dtype=BF16)
    assert off_by(got, a @ b.T, a.abs() @ b.abs().T, d) <= 0
    assert torch.equal(e.project_fp4(codes, table, dtype=BF16), got)


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
def test_fp4_scores_of_the_most_groups(method):
    e = ext()
    counts = [i % 3 for i in range(1024)]
    offsets, rows = offsets_of(counts), sum(counts)
    q = torch.randn(rows, 96, device="cuda")
    table = e.quantize_fp4(torch.randn(1024, 40, 96, device="cuda"), method)
    a, b = e.dequantize_fp4(e.quantize_fp4(q, method)), e.dequantize_fp4(table)
    want, size = grouped_plain(a, b, torch.zeros(rows, 40, device="cuda"), offsets)
    assert off_by(e.project_fp4(q, table, offsets.cuda()), want[0], size[0], 96) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
def test_fp4_scores_of_nan_rows(method):
    """A NaN in a query or a table row makes its own scores NaN and no others."""
    e = ext()
    g = torch.Generator().manual_seed(8)
    q, t = torch.randn(40, 96, generator=g), torch.randn(150, 96, generator=g)
    q[7, 50], t[130, 3] = float("nan"), float("inf")
    got = e.project_fp4(q.cuda(), e.quantize_fp4(t.cuda(), method)).cpu()
    nan = torch.zeros(40, 150, dtype=torch.bool)
    nan[7], nan[:, 130] = True, True
    assert torch.equal(got.isnan(), nan)


# ---- as they are used -----------------------------------------------------------------------
@pytest.mark.gpu
def test_routed_queries_against_the_leaves_of_their_router():
    """Router, rows by group, product with the group's leaves: ||q||^2 - 2 q.l + ||l||^2 are
    the distances that routing_cuda itself returns; then the same over 4-bit leaves."""
    e = ext()
    g = torch.Generator().manual_seed(9)
    n_r, n_l, d, batch = 32, 64, 96, 500
    rv = torch.randn(n_r, d, generator=g).cuda()
    ev = torch.randn(n_r, n_l, d, generator=g).cuda()
    en = torch.randint(1000, (n_r, n_l), generator=g).cuda()
    q = torch.randn(batch, d, generator=g).cuda()
    router, distances = e.routing_cuda(q, rv, en, ev)
    order, offsets = e.group_rows(router, n_r)
    rows = q[order]
    dots = torch.empty(batch, n_l, device="cuda")
    dots.index_copy_(0, order, e.project_grouped(rows, ev, offsets))
    norm = (q * q).sum(1, keepdim=True) + (ev * ev).sum(2)[router]
    a, b = q.double().abs(), ev.double().abs()[router]
    size = (a * a).sum(1, keepdim=True) + (b * b).sum(2) + 2 * (b @ a.unsqueeze(2)).squeeze(2)
    assert ((norm - 2 * dots - distances).abs() <= (2 * d + 4) * 2.0 ** -23 * size).all()
    table = e.quantize_fp4(ev, "nvfp4")
    scores = e.project_fp4(rows, table, offsets)
    x4, t4 = e.dequantize_fp4(e.quantize_fp4(rows, "nvfp4")).double(), e.dequantize_fp4(table).double()
    mine = t4[router[order]]
    want = (mine @ x4.unsqueeze(2)).squeeze(2)
    assert off_by(scores, want, (mine.abs() @ x4.abs().unsqueeze(2)).squeeze(2), d) <= 0


@pytest.mark.gpu
def test_a_step_in_a_graph_and_on_two_streams():
    """Forward and gradients captured once and replayed on new values, then the same calls on
    two streams at once: results are those of plain calls, bit by bit."""
    e = ext()
    g = torch.Generator().manual_seed(10)
    ids = torch.randint(6, (300,), generator=g).cuda()
    x = torch.randn(300, 136, generator=g).to(BF16).cuda()
    w = torch.randn(6, 72, 136, generator=g).to(BF16).cuda()
    dy = torch.randn(300, 72, generator=g).to(BF16).cuda()

    def step(ids, x, w, dy):
        order, offsets = e.group_rows(ids, 6)
        rows = x[order]
        y = e.project_grouped(rows, w, offsets)
        dx, dw = e.project_grouped_backward(dy, rows, w, offsets)
        s = e.project_fp4(rows, e.quantize_fp4(w, "mxfp4"), offsets)
        return y, dx, dw, s

    plain = step(ids, x, w, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, x, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(ids, x, w, dy)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, plain))
    ids.copy_(torch.randint(6, (300,), generator=g))
    x.copy_(torch.randn(300, 136, generator=g))
    want = step(ids, x, w, dy)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    other = [t.clone() for t in (ids.flip(0), x.flip(0), w.flip(0), dy)]
    want_other = step(*other)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for s, args in zip(streams, ((ids, x, w, dy), other)):
            with torch.cuda.stream(s):
                got.append(step(*args))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[0], want))
        assert all(torch.equal(a, b) for a, b in zip(got[1], want_other))


@pytest.mark.gpu
def test_a_captured_step_while_an_eager_graph_lives():
    """Autograd is refused in a capture; the explicit gradients are captured beside a live
    eager graph of the same leaves, which still gives its own."""
    e = ext()
    x = torch.randn(50, 64, device="cuda", dtype=BF16, requires_grad=True)
    w = torch.randn(2, 32, 64, device="cuda", dtype=BF16, requires_grad=True)
    offsets = torch.tensor([0, 20, 50], device="cuda")
    ones = torch.ones(50, 32, device="cuda", dtype=BF16)
    eager = e.project_grouped(x, w, offsets)
    want = torch.autograd.grad(eager, (x, w), ones, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="project_grouped_backward"):
            e.project_grouped(x, w, offsets)
        with torch.no_grad():
            y = e.project_grouped(x, w, offsets)
            held = e.project_grouped_backward(ones, x, w, offsets)
    graph.replay()
    assert torch.equal(y, eager) and all(torch.equal(a, b) for a, b in zip(held, want))
    again = torch.autograd.grad(eager, (x, w), ones)
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.gpu
def test_first_call_of_a_thread():
    """A thread that has made no GPU call yet has no context bound: a child process, so that
    the library itself is fresh too."""
    import subprocess
    import sys
    code = """
import threading, torch
from pilotann_b200 import extension as e
x = torch.randn(40, 64, device="cuda").bfloat16()
w = torch.randn(2, 32, 64, device="cuda").bfloat16()
o = torch.tensor([0, 10, 40], device="cuda")
dy = torch.randn(40, 32, device="cuda").bfloat16()
t = e.quantize_fp4(w)
torch.cuda.synchronize()
got = []
for call in (lambda: e.project_grouped_backward(dy, x, w, o), lambda: e.project_fp4(x, t, o)):
    thread = threading.Thread(target=lambda: got.append(call()))
    thread.start(); thread.join()
assert len(got) == 2, got
want = e.project_grouped_backward(dy, x, w, o)
assert torch.equal(got[0][0], want[0]) and torch.equal(got[0][1], want[1])
assert torch.equal(got[1], e.project_fp4(x, t, o))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_first_calls_in_a_capture():
    """Nothing has to have run before a stream capture: a fresh process captures its first calls."""
    import subprocess
    import sys
    code = """
import torch
from pilotann_b200 import extension as e
ids = torch.randint(4, (20000,), device="cuda")
x = torch.randn(1500, 320, device="cuda").bfloat16()
w = torch.randn(3, 304, 320, device="cuda").bfloat16()
xf, wf = x.float(), w.float()
xo, wo = x[:, :319].contiguous(), w[:, :, :319].contiguous()
o = torch.tensor([0, 700, 700, 1500], device="cuda")
dy = torch.randn(1500, 304, device="cuda").bfloat16()
torch.cuda.synchronize()
def step():
    t = e.quantize_fp4(w, "nvfp4")
    return [*e.group_rows(ids, 4), e.project_grouped(x, w, o), e.project_grouped(xf, wf, o),
            e.project_grouped(xo, wo, o), *e.project_grouped_backward(dy, x, w, o),
            e.project_fp4(x, t, o, dtype=torch.bfloat16), e.dequantize_fp4(t)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    held = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(held, step()))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    e = ext()
    x, w = torch.randn(10, 64, device="cuda:1"), torch.randn(2, 8, 64, device="cuda:1")
    offsets = torch.tensor([0, 4, 10], device="cuda:1")
    want, size = grouped_plain(x, w, torch.zeros(10, 8, device="cuda:1"), offsets.cpu())
    assert off_by(e.project_grouped(x, w, offsets), want[0], size[0], 64) <= 0
    assert e.project_fp4(x, e.quantize_fp4(w), offsets).device == x.device
