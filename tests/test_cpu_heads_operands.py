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


def test_per_row_operands_in_another_order_of_the_rows_dimensions():
    """As many elements as rows, but laid out over the leading dimensions in another order: refused, not read in the wrong order.  One
    dimension, the rows' own, or either with dimensions of 1 go on to the next check (there is no GPU here)."""
    x = torch.zeros(3, 4, 10)
    y, f, stat = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3), torch.zeros(4, 3, 2)
    good, gf = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)
    ti, tv = torch.zeros(3, 4, 2, dtype=torch.int32), torch.zeros(3, 4, 2)
    s = heads.LabelScores(None, gf, torch.zeros(3, 4, 2), None, None, None)
    for call in (lambda: heads.label_logprobs(x, y), lambda: heads.layer_norm_backward(x, x, None, f, gf),
                 lambda: heads.layer_norm_backward(x, x, None, gf, f), lambda: heads.label_logprobs_backward(x, y, s, gf),
                 lambda: heads.label_logprobs_backward(x, good, s._replace(stat=stat), gf),
                 lambda: heads.label_logprobs_backward(x, good, s._replace(entropy=f), gf, gf),
                 lambda: heads.label_logprobs_backward(x, good, s, f), lambda: heads.label_logprobs_backward(x, good, s, gf, f),
                 lambda: heads.distill_loss(x, ti, tv, y, label_weight=0.5), lambda: heads.distill_loss(x, ti, tv, row_scale=f)):
        with pytest.raises(ValueError, match="the rows' is .3, 4."):
            call()
    for shape in ((3, 4), (12,), (12, 1), (3, 4, 1), (1, 12), (1, 3, 1, 4)):
        v, g = torch.zeros(shape, dtype=torch.int32), torch.zeros(shape)
        t = s._replace(entropy=g, stat=torch.zeros(*shape, 2))
        for call in (lambda: heads.label_logprobs(x, v), lambda: heads.layer_norm_backward(x, x, None, g, g),
                     lambda: heads.label_logprobs_backward(x, v, t, g, g), lambda: heads.distill_loss(x, ti, tv, v, row_scale=g)):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call()
    # with one leading dimension there is only one order
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        heads.label_logprobs(torch.zeros(12, 10), torch.zeros(3, 4, dtype=torch.int32))
