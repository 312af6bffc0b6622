"""CPU: what the classifier-head entry points refuse before anything reaches a GPU: buffers asked for rows that no call takes."""
import pytest
import torch

from wfd_gan_amd import heads

LIKE = {"norm": heads.norm_output_like, "norm gradients": heads.norm_gradients_like, "scores": heads.scores_like,
        "distill": heads.distill_output_like}


@pytest.mark.parametrize("name", LIKE)
def test_buffers_for_rows_that_no_call_takes(name):
    """The calls' own refusals: no division by zero, no wrapped sizes."""
    like = LIKE[name]
    for bad in (torch.zeros(4, 0), torch.zeros(())):
        with pytest.raises(ValueError, match="at least one element"):
            like(bad)
    for bad in (torch.zeros(4, 10, dtype=torch.float64), torch.zeros(4, 10, dtype=torch.int32)):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            like(bad)
    with pytest.raises(ValueError, match="more than 2"):
        like(torch.zeros(1, 1).expand((1 << 31) + 3, 1))
    assert like(torch.zeros(0, 10))[0].shape[0] == 0


def test_buffers_for_alternatives_that_no_call_gives():
    for k in (-1, 11, 65, (1 << 32) + 3):
        with pytest.raises(ValueError, match="not supported"):
            heads.scores_like(torch.zeros(4, 10), k)
