"""GPU: results of the two-launch layer that pass their type's range."""
import pytest
import torch

import moe_small_reference as R
from test_gpu_moe_small import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["dense", "w8"])
@pytest.mark.parametrize("T", [1, 9])
def test_fp16_results_past_the_largest_number_are_infinite(kind, T):
    """Where the value in 64 bits is twice fp16's largest number or more the result is the infinity of its sign; elsewhere it is
    finite and as close as ever.  (bf16 ends where the fp32 sums end: there it is the sums that overflow, in either direction.)"""
    lay = Layer(kind, T, 256, 128, 8, 2, torch.float16)
    top = torch.finfo(torch.float16).max
    if kind == "dense":                                   # every other channel
        lay.w2[:, ::2] = torch.where(lay.w2[:, ::2] < 0, -1.0, 1.0).half() * (top / 2)
    else:
        lay.w2[1][:, ::2] *= 1e7
    out = lay()
    ref, bound = R.layer(lay.x, lay.router, lay.experts, 2, int8=kind == "w8")
    past = ref.abs() - bound > 2 * top
    assert past.any() and not past[:, 1::2].any()
    assert torch.equal(out[past].double(), torch.sign(ref[past]) * float("inf"))
    inside = ref.abs() + bound < top / 2
    assert inside[:, 1::2].all()
    R.assert_close(torch.where(inside, out, 0), torch.where(inside, ref, 0.0), torch.where(inside, bound, 0.0))
