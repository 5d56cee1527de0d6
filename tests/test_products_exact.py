"""Products whose sums are exact: small whole numbers, every partial sum of which fp32 holds as it
is, in whatever order and however a step cuts off.  Results are compared bit by bit with the exact
sum rounded once, so that a slice that is lost, doubled or cleared too far shows."""
import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ext():
    from pilotann_b200 import extension
    return extension


def whole(shape, seed, most=3, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device=device).float()


def edges_of(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def product(a, b):
    """a @ b.T, exact: magnitudes are at most 9 for a term, 2^53 / 9 terms."""
    return a.double() @ b.double().T


@pytest.mark.parametrize("rows,step", [(20000, 16), (65536, 16)])
def test_a_lost_step_shows(rows, step):
    """Without the 16 rows of one step, wherever it lies, hardly a sum is what it was: a sum stays only
    if 16 products of numbers from -3 to 3 add up to 0."""
    x, dy = whole((rows, 24), 1), whole((rows, 72), 2)
    for at in (0, rows // 2, rows - step):
        lost = product(dy[at:at + step].T, x[at:at + step].T)
        assert (lost != 0).double().mean() > 0.9
    assert product(dy.abs().T, x.abs().T).max() < 2 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,d,d_out", [
    ([20000], 24, 72), ([65536], 64, 40), ([1 << 20], 64, 64),
    ([8191, 8192, 8193, 16385], 72, 136),           # about the length of a part of a sum
    ([8191, 0, 8192, 8193, 16385, 1], 136, 264),
    ([70001, 15, 20000], 200, 333), ([33000, 3], 128, 128), ([1000, 0, 1, 3000, 257, 742], 512, 640)])
def test_gradients_of_matrices(dtype, counts, d, d_out):
    rows, edges = sum(counts), edges_of(counts)
    x = whole((rows, d), rows, device="cuda").to(dtype)
    dy = whole((rows, d_out), d, device="cuda").to(dtype)
    w = torch.zeros(len(counts), d_out, d, device="cuda", dtype=dtype)
    _, dw = ext().project_grouped_backward(dy, x, w, torch.tensor(edges, device="cuda"),
                                           want_query=False)
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        assert torch.equal(dw[g], product(dy[lo:hi].T, x[lo:hi].T).to(dtype)), g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,d,d_out", [
    ([1], 65536, 40), ([5, 0, 9], 40008, 264), ([40], 16384, 1000), ([100, 90], 24576, 264),
    ([300, 1], 8200, 2560), ([2100], 20480, 2560), ([38000], 8256, 72), ([700, 33], 8191, 136)])
def test_products_and_gradients_of_rows(dtype, counts, d, d_out):
    """The long axis is summed in both: w lies the other way round for the gradient."""
    rows, edges = sum(counts), edges_of(counts)
    x = whole((rows, d), rows, device="cuda").to(dtype)
    w = whole((len(counts), d_out, d), d, device="cuda").to(dtype)
    offsets = torch.tensor(edges, device="cuda")
    y = ext().project_grouped(x, w, offsets)
    dx, _ = ext().project_grouped_backward(x, torch.zeros(rows, d_out, device="cuda", dtype=dtype),
                                           w.transpose(1, 2).contiguous(), offsets, want_VT=False)
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        want = product(x[lo:hi], w[g]).to(dtype)
        assert torch.equal(y[lo:hi], want) and torch.equal(dx[lo:hi], want), g


def levels(shape, seed):
    """Numbers that 4 bits hold, a 6 in every block: every scale is a power of two."""
    g = torch.Generator().manual_seed(seed)
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    x = level[torch.randint(8, shape, generator=g)]
    x[..., ::16] = 6.0
    return x * (1.0 - 2.0 * torch.randint(2, shape, generator=g))


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("rows,d,d_out", [(1, 65536, 40), (3, 40000, 300), (1, 768, 5000),
                                          (20, 33, 130), (50, 8200, 1000), (100, 4100, 257),
                                          (700, 2080, 1000), (260, 65504, 200)])
def test_scores(method, out, rows, d, d_out):
    e = ext()
    q, t = levels((rows, d), rows), levels((d_out, d), d)
    # a product is a multiple of 1/4 of at most 36: sums of 65536 stay below 2^24 quarters
    want = product(q.cuda(), t.cuda())
    assert want.abs().max() < 2 ** 22
    table = e.quantize_fp4(t.cuda(), method)
    assert torch.equal(e.dequantize_fp4(table).cpu(), t)
    assert torch.equal(e.project_fp4(q.cuda(), table, dtype=out), want.to(out))


@pytest.mark.gpu
def test_scores_of_extreme_row_scales():
    """Values of 2^120 and 2^-120, whose row scales multiply past fp32's range, and what they are held
    as: a block's scale is max / 6 in E4M3, to the nearest of 8 steps an octave, and a value the nearest
    level of that scale.  max = 2^k: with s = 2^(k - 11) (the least with 2^k <= 2688 s), 2048 / 6 =
    341.33 is held as 352, and 2048 / 352 = 5.82 as 6: 2112 s = 1.03125 2^k."""
    e = ext()
    big, small, held = 2.0 ** 120, 2.0 ** -115, 1.03125
    q = torch.full((3, 32), big, device="cuda")
    q[1], q[2] = 0.0, small
    t = torch.full((2, 32), big, device="cuda")
    t[1] = small
    a, b = e.quantize_fp4(q, "nvfp4"), e.quantize_fp4(t, "nvfp4")
    assert torch.equal(e.dequantize_fp4(a), held * q) and torch.equal(e.dequantize_fp4(b), held * t)
    inf, both = float("inf"), 32 * held * held
    want = torch.tensor([[inf, both * 32], [0.0, 0.0], [both * 32, 0.0]])
    assert torch.equal(e.project_fp4(a, b).cpu(), want)
