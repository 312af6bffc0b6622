"""GPU: corners of the classifier-head operators' documented range: rows of one and two columns."""
import pytest
import torch

from tests import heads_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
INF = float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- layer norm of one and two columns ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [1, 7, 2500])
@pytest.mark.parametrize("n", [1, 2])
def test_norm_backward_of_one_and_two_columns(n, m, t):
    """dx of one column is 0; of two it is what eps leaves of a difference, so every operation is rounded on its own: the bits of the
    formula's operations one by one in fp32."""
    from wfd_gan_amd import heads
    g = gen(10 * m + n)
    for wt in {t, F32, None}:
        x, dy = (torch.randn(m, n, generator=g) * 1.5 + 2).to(t), torch.randn(m, n, generator=g).to(t)
        w = torch.ones(n) if wt is None else (1 + 0.2 * torch.randn(n, generator=g)).to(wt)
        wd = None if wt is None else w.to(DEV)
        r = heads.layer_norm(x.to(DEV), wd)
        dx = heads.layer_norm_backward(dy.to(DEV), x.to(DEV), wd, r.mean, r.rstd).dx.cpu()
        mean, rstd = r.mean.cpu()[:, None], r.rstd.cpu()[:, None]
        v, xh = dy.float() * w.float(), (x.float() - mean) * rstd
        total = lambda a: a[:, :1] if n == 1 else a[:, :1] + a[:, 1:]
        want = (rstd * (v - total(v) / n - xh * (total(v * xh) / n))).to(t)
        assert n == 2 or float(dx.abs().max()) == 0
        assert torch.equal(dx, want)
