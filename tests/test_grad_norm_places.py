"""Where the gradient norm's results may lie: refusals that need no GPU."""
import pytest

from pcp_amd import _lib
from test_score_abi import CLIP, call_list


@pytest.mark.parametrize("change,fine", [
    (dict(norm=0x1000, coef=0x1000), False),                 # one place for both
    (dict(norm=0x10000), False), (dict(norm=0x1018c), False),          # a gradient's first and last element
    (dict(coef=0x20000), False), (dict(coef=0x20060), False),
    (dict(norm=0x10190), True), (dict(norm=0xfffc), True), (dict(coef=0x20064), True), (dict(coef=0x1fffc), True),
    (dict(coef=0x20000, counts=[100, 0]), True),             # a tensor without elements has no place
    (dict(norm=0x1000, coef=0x1004, grads=[0x10000, 0x10000]), True),
    (dict(norm=0x1000, coef=0x1000, counts=[0, 0]), False),
])
def test_norm_without_outputs(change, fine):
    """100 f32 elements at 0x10000 and 50 bf16 ones at 0x20000; the results behind one another at 0x1000 unless changed."""
    got, said = call_list(_lib.GradClipArgs, "pcp_grad_clip_args_init", "pcp_grad_clip", CLIP,
                          dict(norm=0x1000, coef=0x1004, max_norm=1.0), dict(out=None, out_dtypes=None, **change))
    assert got == -1 and ("context is NULL" if fine else "overlap") in said, said
