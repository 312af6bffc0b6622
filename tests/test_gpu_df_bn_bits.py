"""GPU: the bits of the tall BatchNorm statistics.  The combine of the chunks' means and squared deviations is restated in fp32 with
every rounding where the kernel has it (16 groups of chunks whose folds round product and sum once, then the groups' folds, of
which the 4th and the 10th do), so that an observer trained again gives the checkpoint of the builds before."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
f32 = np.float32
GROUPS, FUSED = 16, (4, 10)


def fold(a, b, fused):
    """(mean, sum of squared deviations, count) of a and b together, per column, counts the same for all columns"""
    if b[2] <= 0:
        return a
    tot, delta = f32(a[2] + b[2]), b[0] - a[0]
    w, d2 = f32(f32(a[2] * b[2]) / tot), delta * delta
    if fused:                                              # one rounding: product and sum fit 80 bits but for ties
        t = (d2.astype(np.longdouble) * np.longdouble(w) + b[1].astype(np.longdouble)).astype(f32)
    else:
        t = b[1] + d2 * w
    return a[0] + delta * f32(b[2] / tot), a[1] + t, tot


def combine(part, M, rpc, fused=FUSED):
    nchunk, _, N = part.shape
    zero = np.zeros(N, f32), np.zeros(N, f32), f32(0)
    groups = [zero] * GROUPS
    for c in range(nchunk):
        groups[c % GROUPS] = fold(groups[c % GROUPS], (part[c, 0], part[c, 1], f32(min(rpc, M - c * rpc))), True)
    a = groups[0]
    for k in range(1, GROUPS):
        a = fold(a, groups[k], k in fused)
    return a


@pytest.mark.parametrize("M,N,rpc,apart", [(700, 32, 64, 0), (5000, 33, 64, 0), (20011, 64, 64, 0), (179200, 32, 175, 0),
                                           (37, 5, 64, 0), (5000, 33, 64, 3), (20011, 64, 64, 3)])
def test_tall_batchnorm_statistics_bit_for_bit(M, N, rpc, apart):
    """``apart``: how far the groups of chunks lie from each other."""
    from wfd_gan_amd._lib import lib
    g = torch.Generator().manual_seed(M)
    z = ((torch.randn(M, N, generator=g) * 2 + 3 * torch.randn(N, generator=g)) * (1 + torch.arange(M)[:, None] / M)).to(DEV)
    z += apart * (torch.arange(M, device=DEV) // rpc % GROUPS * 7 % 5)[:, None]
    nchunk = -(-M // rpc)
    part = torch.zeros(nchunk, 2, N, device=DEV)
    mean, istd = torch.zeros(N, device=DEV), torch.zeros(N, device=DEV)
    rm, rv = torch.randn(N, generator=g), torch.rand(N, generator=g) + 0.5
    rmd, rvd = rm.to(DEV), rv.to(DEV)
    lib().bn_tall_stats(z.data_ptr(), N, M, N, rpc, part.data_ptr(), 1e-5, 0.1, mean.data_ptr(), istd.data_ptr(), rmd.data_ptr(),
                        rvd.data_ptr(), torch.cuda.current_stream().cuda_stream)
    p = part.cpu().numpy()
    mu, m2, cnt = combine(p, M, rpc)
    assert cnt == M and np.array_equal(mean.cpu().numpy(), mu)
    assert np.array_equal(istd.cpu().numpy(), f32(1) / np.sqrt(m2 / f32(M) + f32(1e-5)))
    keep = f32(1) - f32(0.1)
    assert np.array_equal(rmd.cpu().numpy(), keep * rm.numpy() + f32(0.1) * mu)
    assert np.array_equal(rvd.cpu().numpy(), keep * rv.numpy() + f32(0.1) * (m2 / (f32(M) - f32(1))))
    # the statistics themselves: sums of rpc elements in fp32 (rpc U), then 16 + chunks / 16 folds of a few U each
    zd = z.double().cpu()
    assert np.allclose(mean.cpu(), zd.mean(0), rtol=0, atol=float(zd.abs().mean(0).max()) * (rpc + 4 * (16 + nchunk / 16)) * 2.0 ** -24)
    if apart:                                              # another rule for the groups' folds shows in the bits
        assert not np.array_equal(m2, combine(p, M, rpc, fused=())[1])
        assert not np.array_equal(m2, combine(p, M, rpc, fused=tuple(range(GROUPS)))[1])
