"""What the products do with tensors that carry derivatives."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def ext():
    from pilotann_b200 import extension
    return extension


def case(dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(20, 64, generator=g), torch.randn(20, 32, generator=g)
    w = torch.randn(2, 32, 64, generator=g)
    return *(t.to(dtype).cuda() for t in (x, w, dy)), torch.tensor([0, 5, 20], device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_mode_tangents_are_refused(dtype):
    """A dual tensor requires no gradient: its tangent would be lost without a word."""
    e = ext()
    x, w, dy, offsets = case(dtype)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, dy)]
        for call in (lambda: e.project_grouped(dual[0], w, offsets),
                     lambda: e.project_grouped(x, dual[1], offsets),
                     lambda: e.project_grouped_backward(dual[2], x, w, offsets),
                     lambda: e.project_grouped_backward(dy, dual[0], w, offsets),
                     lambda: e.project_grouped_backward(dy, x, dual[1], offsets)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        inside = e.project_grouped(x, w, offsets)       # without a tangent as ever
    assert torch.equal(inside, e.project_grouped(x, w, offsets))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda v: e.project_grouped(v, w, offsets), (x,), (x,))


def test_codes_and_scores_have_no_gradient():
    e = ext()
    x, w, _, offsets = case()
    x.requires_grad_(True), w.requires_grad_(True)
    table = e.quantize_fp4(w, "nvfp4")
    scores = e.project_fp4(x, table, offsets)
    assert not scores.requires_grad and not e.dequantize_fp4(table).requires_grad
    with torch.no_grad():
        assert torch.equal(scores, e.project_fp4(x, table, offsets))
