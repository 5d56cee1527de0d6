"""Arguments of the products' C entries that would make a kernel fault are errors before anything is
enqueued."""
import pytest


@pytest.mark.parametrize("call,args", [
    ("pa_group_rows", (12, 16, 16, 4, 4, 0, 0)),
    ("pa_group_rows", (16, 20, 16, 4, 4, 0, 0)),
    ("pa_group_rows", (16, 16, 4, 4, 4, 0, 0)),
    ("pa_group_rows", (16, 16, 16, 100000, 4, 18, 0)),
    ("pa_project_grouped", (16, 16, 16, 20, 4, 2, 8, 8, 8, 8, 0, 0, 0)),
    ("pa_project_grouped", (16, 16, 16, 17, 4, 2, 8, 8, 8, 8, 1, 0, 0)),
    ("pa_project_grouped_backward", (16, 16, 16, 16, 16, 12, 4, 2, 8, 8, 8, 8, 8, 0, 0, 0)),
    ("pa_project_grouped_backward", (16, 0, 16, 16, 16, 9, 4, 2, 8, 8, 8, 8, 8, 2, 0, 0)),
    ("pa_project_fp4", (16, 16, 16, 0, 16, 16, 0, 4, 4, 2, 8, 8, 0, 0, 0)),
])
def test_pointers_off_their_alignment_are_refused(call, args):
    """64-bit numbers off 8 bytes are a misaligned address on the GPU."""
    from pilotann_b200 import _C
    lib = _C.lib()
    assert getattr(lib, call)(*args) == _C.PA_ERR_ARG
    assert b"aligned" in lib.pa_last_error()
