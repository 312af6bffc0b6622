"""GPU: corners of the classifier-head operators' documented range: rows of one and two columns, masks of the type's
lowest value at low temperatures, NaN at the first class, rows whose only entry of the teacher is wrong, rows
without a term, results passed in again for a call that writes less, gradients
that are not wanted, shares of a masked class."""
import itertools

import numpy as np
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
    formula's operations one by one in fp32.  The last product, rstd times the difference, may be rounded to fp16 at once (gfx950 has
    an instruction for it) instead of to fp32 first: where the fp32 product lies midway between two fp16 values, or next to it, the two
    differ by a step, and the one that is rounded once is the nearer.  The weight's types come in every order, each order from the
    same seed."""
    from wfd_gan_amd import heads
    for order in itertools.permutations(dict.fromkeys((t, F32, None))):
        g = gen(10 * m + n)
        for wt in order:
            x, dy = (torch.randn(m, n, generator=g) * 1.5 + 2).to(t), torch.randn(m, n, generator=g).to(t)
            w = torch.ones(n) if wt is None else (1 + 0.2 * torch.randn(n, generator=g)).to(wt)
            wd = None if wt is None else w.to(DEV)
            r = heads.layer_norm(x.to(DEV), wd)
            dx = heads.layer_norm_backward(dy.to(DEV), x.to(DEV), wd, r.mean, r.rstd).dx.cpu()
            mean, rstd = r.mean.cpu()[:, None], r.rstd.cpu()[:, None]
            v, xh = dy.float() * w.float(), (x.float() - mean) * rstd
            total = lambda a: a[:, :1] if n == 1 else a[:, :1] + a[:, 1:]
            d = v - total(v) / n - xh * (total(v * xh) / n)
            fits = dx == (rstd * d).to(t)
            if t == F16:                                   # 24 x 24 bits are exact in 64; numpy rounds those to fp16 at once
                fits |= dx == torch.from_numpy((rstd.double() * d.double()).numpy().astype(np.float16))
            assert n == 2 or float(dx.abs().max()) == 0
            assert bool(fits.all())


# ---- entropy under masks of the type's lowest value -------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("temp", [1e-6, 1e-5, 1e-4, 1e-3])
@pytest.mark.parametrize("m,v", [(1, 100), (3, 1401), (3, 5003), (2050, 5003), (1, 50257), (3, 50257), (600, 50257), (1, 128000),
                                 (3, 128000), (600, 128000)])
def test_entropy_of_one_class_left_among_the_lowest_values(m, v, temp, t):
    """Whole lanes, waves and parts hold masked classes only.  Everything but one class has share 0, so log probability and entropy
    are 0 to the bit, and so is the gradient of both."""
    from wfd_gan_amd import heads
    at = torch.randint(0, v, (m,), generator=gen(v + m)).to(DEV)
    x = torch.full((m, v), torch.finfo(t).min, dtype=t, device=DEV)
    x[torch.arange(m, device=DEV), at] = 1.5
    y = at.to(torch.int32)
    for k in (0, 1):
        r = heads.label_logprobs(x, y, k, temperature=temp)
        assert float(r.entropy.abs().max()) == 0 and float(r.logprob.abs().max()) == 0
        if k:
            assert torch.equal(r.top_index[:, 0], y) and float(r.top_logprob.abs().max()) == 0
    one = torch.ones(m, device=DEV)
    d = heads.label_logprobs_backward(x, y, r, one, one, temperature=temp)
    assert float(d.abs().max()) == 0


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("temp", [1e-5, 1e-3, 1.0])
@pytest.mark.parametrize("m,v", [(4, 1000), (4, 20011), (2050, 4000), (4, 131072)])
def test_entropy_of_a_short_run_left_among_the_lowest_values(m, v, temp, t):
    """Seven classes in a row are left: against the definition, with the gradient of log probability and entropy."""
    from wfd_gan_amd import heads
    g = gen(v)
    x = torch.full((m, v), torch.finfo(t).min, dtype=t)
    lo = v // 3
    x[:, lo:lo + 7] = (torch.randn(m, 7, generator=g) * temp).to(t)
    y = (lo + torch.randint(0, 7, (m,), generator=g)).to(torch.int32)
    r = heads.label_logprobs(x.to(DEV), y.to(DEV), 5, temperature=temp)
    rows = [0, 1, 2, m - 1]
    want = R.scores(x[rows], y[rows], 5, temp)
    R.check(r.entropy[rows], want["entropy"], want["b_entropy"], F32, "entropy")
    R.check(r.logprob[rows], want["logprob"], want["b_logprob"], F32, "logprob")
    assert torch.equal(r.top_index[rows].cpu().long(), want["top_index"])
    dl, dh = torch.randn(m, generator=g), torch.randn(m, generator=g)
    d = heads.label_logprobs_backward(x.to(DEV), y.to(DEV), r, dl.to(DEV), dh.to(DEV), temperature=temp)
    want, bound = R.scores_backward(x[rows], y[rows], r.stat[rows], r.entropy[rows], dl[rows], dh[rows], temp)
    R.check(d[rows], want, bound, t, "dlogits")


# ---- NaN at the first class -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v", [(3, 5), (3, 64), (3, 100), (3, 1401), (3, 2049), (3, 9001), (2050, 3001), (600, 33000), (3, 131075)])
def test_nan_at_the_first_class_is_the_first_alternative(m, v, t):
    """NaN stand before all numbers and by index among themselves, in every form: rows in a wave, in a workgroup, in parts."""
    from wfd_gan_amd import heads
    x = torch.randn(m, v, generator=gen(v)).to(t)
    x[:, 0] = float("nan")
    x[1, 2] = float("nan")
    x[2, v // 2] = INF
    if m > 600:
        x[600] = float("nan")                             # nothing else in the row
    rows = [0, 1, 2, min(m - 1, 600)]
    for k in (1, min(v, 20)):
        r = heads.label_logprobs(x.to(DEV), None, k)
        want = R.scores(x[rows], None, k, 1.0)
        assert torch.equal(r.top_index[rows].cpu().long(), want["top_index"])
        assert int(r.top_index[:, 0].abs().max()) == 0 and bool(r.top_logprob.isnan().all())


# ---- a teacher whose only entry is wrong --------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [5, 100, 1401, 40003, 140001])
@pytest.mark.parametrize("temp", [1.0, 2.0])
def test_a_wrong_index_alone_in_its_row_shows_in_loss_and_gradient(v, temp, t):
    """Index V with no other entry, with absent ones and with ones at -inf; without labels, and with label -1."""
    from wfd_gan_amd import heads
    x = torch.randn(4, v, generator=gen(v)).to(t).to(DEV)
    y = torch.full((4,), -1, dtype=torch.int32, device=DEV)
    good = [0, 1, 2]
    for ti, tv in (([[v], [0], [v + 5], [v]], [[0.5]] * 4),
                   ([[v, -1, -1], good, [-1, v, -1], [1, v, 2]], [[0.5] * 3, [0.1, 0.2, 0.3], [0.5] * 3, [-INF, 1.0, -INF]])):
        ti, tv = torch.tensor(ti, dtype=torch.int32, device=DEV), torch.tensor(tv, device=DEV)
        for kw in (dict(), dict(labels=y, weight=0.6, label_weight=0.4)):
            r = heads.distill_loss(x, ti, tv, temperature=temp, **kw)
            assert r.loss.isnan().tolist() == [True, False, True, True]
            assert r.dlogits.isnan().all(1).tolist() == [True, False, True, True]
            assert bool(r.dlogits[1].isfinite().all())
            assert heads.distill_loss(x, ti, tv, temperature=temp, grad=False, **kw).loss.isnan().tolist() == [True, False, True, True]


# ---- rows without a term ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [5, 100, 1401, 40003, 140001])
def test_distill_rows_without_a_term_have_gradient_zero_whatever_they_hold(v, t):
    """Padding rows: no entry (or none above -inf) and no label.  Their loss is 0, so their gradient is, also where the logits are NaN
    or infinite; the rows beside them keep theirs, and a NaN row with a term is NaN."""
    from wfd_gan_amd import heads
    m = 9
    x = torch.randn(m, v, generator=gen(v)).to(t)
    x[0] = float("nan")
    x[1, v // 2] = INF
    x[2] = -INF
    x[3, 0] = float("nan")
    x[4, v - 1] = float("nan")
    x[7, 1] = float("nan")
    ti = torch.tensor([[-1, -1]] * 6 + [[0, 1]] * 3, dtype=torch.int32)
    ti[4] = torch.tensor([0, 1])
    tv = torch.zeros(m, 2)
    tv[4] = -INF
    y = torch.tensor([-1] * 6 + [2, 2, -1], dtype=torch.int32)
    none, bad, fine = slice(0, 6), 7, [6, 8]
    for kw in (dict(), dict(labels=y.to(DEV), weight=0.5, label_weight=0.5),
               dict(labels=y.to(DEV), temperature=2.0, weight=0.5, label_weight=0.5), dict(temperature=0.5)):
        r = heads.distill_loss(x.to(DEV), ti.to(DEV), tv.to(DEV), **kw)
        assert float(r.loss[none].abs().max()) == 0 and float(r.dlogits[none].abs().max()) == 0
        assert bool(r.loss[bad].isnan()) and bool(r.dlogits[bad].isnan().all())
        w, u = kw.get("weight", 1.0), kw.get("label_weight", 0.0)
        loss, bl, d, bd = R.distill(x[fine], ti[fine], tv[fine], y[fine] if u else None, kw.get("temperature", 1.0), w, u,
                                    torch.ones(2))
        R.check(r.loss[fine], loss, bl, F32, "loss")
        R.check(r.dlogits[fine], d, bd, t, "dlogits")
    # the label's term alone
    r = heads.distill_loss(x.to(DEV), ti.to(DEV), tv.to(DEV), y.to(DEV), weight=0.0, label_weight=1.0)
    rows = [0, 1, 2, 3, 4, 5, 8]
    assert float(r.loss[rows].abs().max()) == 0 and float(r.dlogits[rows].abs().max()) == 0
    assert bool(r.dlogits[bad].isnan().all()) and bool(r.dlogits[6].isfinite().all()) and float(r.dlogits[6].abs().max()) > 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [5, 100, 1401, 40003])
def test_scores_rows_without_a_label_have_gradient_zero_whatever_they_hold(v, t):
    """Without a label the log probability is 0 and without d_entropy nothing else is left to differentiate."""
    from wfd_gan_amd import heads
    x = torch.randn(5, v, generator=gen(v)).to(t)
    x[0] = float("nan")
    x[1, v // 2] = INF
    x[3, 1] = float("nan")
    y = torch.tensor([-1, -3, -1, 2, 2], dtype=torch.int32, device=DEV)
    one = torch.ones(5, device=DEV)
    r = heads.label_logprobs(x.to(DEV), y)
    assert float(r.logprob[:3].abs().max()) == 0
    d = heads.label_logprobs_backward(x.to(DEV), y, r, one)
    assert float(d[:3].abs().max()) == 0 and bool(d[3].isnan().all()) and bool(d[4].isfinite().all()) and float(d[4].abs().max()) > 0
    d = heads.label_logprobs_backward(x.to(DEV), y, r, one, one)
    assert d.isnan().all(1).tolist() == [True, True, False, True, False]


# ---- a result passed in again for a call that writes less ---------------------------------------------------------------------
def test_a_result_passed_in_again_holds_what_the_call_wrote():
    """What a call does not write is None in what it returns, not the numbers of the call before; the tensors that it does write are
    those passed in."""
    from wfd_gan_amd import heads
    x = torch.randn(4, 300, generator=gen(1)).to(DEV)
    z = torch.randn(4, 300, generator=gen(2)).to(DEV)
    y = torch.tensor([3, 1, -1, 299], dtype=torch.int32, device=DEV)
    full = heads.layer_norm(x)
    bare = heads.layer_norm(z, stats=False, out=full)
    assert bare.y is full.y and bare.mean is None and bare.rstd is None
    full = heads.label_logprobs(x, y, 5)
    r = heads.label_logprobs(z, y, 0, out=full)
    assert r.top_logprob is None and r.top_index is None and r.logprob is full.logprob and r.entropy is full.entropy
    r = heads.label_logprobs(z, None, 5, out=full)
    assert r.logprob is None and r.top_index is full.top_index and r.stat is full.stat
    ti, tv = torch.zeros(4, 1, dtype=torch.int32, device=DEV), torch.zeros(4, 1, device=DEV)
    full = heads.distill_loss(x, ti, tv)
    alone = heads.distill_loss(z, ti, tv, grad=False, out=full)
    assert alone.loss is full.loss and alone.dlogits is None
    # nothing left out: the very result
    for again, out in ((heads.layer_norm(z, out=(o := heads.norm_output_like(z))), o),
                       (heads.label_logprobs(z, y, 5, out=(o := heads.scores_like(z, 5))), o),
                       (heads.distill_loss(z, ti, tv, out=(o := heads.distill_output_like(z))), o)):
        assert again is out


# ---- gradients that are not wanted ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [16385, 40001])
def test_norm_backward_of_long_rows_without_some_of_the_weights_gradients(n, t):
    """dx alone needs no walk down the columns: the partial sums stay as they were.  One of the two gradients alone, and dx, have the
    bits of the full call; in place as well."""
    from wfd_gan_amd import heads
    g = gen(n)
    x, dy = (torch.randn(5, n, generator=g).to(t).to(DEV) for _ in range(2))
    w = torch.randn(n, generator=g).to(DEV)
    r = heads.layer_norm(x, w, w)
    full = heads.layer_norm_backward(dy, x, w, r.mean, r.rstd)
    for dw, db in ((None, None), (full.dweight, None), (None, full.dbias)):
        work = torch.full_like(full.work, 77.0)
        o = heads.NormGradients(torch.empty_like(x), None if dw is None else torch.empty_like(dw),
                                None if db is None else torch.empty_like(db), work)
        got = heads.layer_norm_backward(dy, x, w, r.mean, r.rstd, out=o)
        assert torch.equal(got.dx, full.dx)
        assert all(a is None if b is None else torch.equal(a, b) for a, b in ((got.dweight, dw), (got.dbias, db)))
        if dw is None and db is None:
            assert bool((work == 77.0).all())
    for where in (dy.clone(), x.clone()):
        args = (where, x) if torch.equal(where, dy) else (dy, where)
        o = heads.NormGradients(where, None, None, full.work)
        assert torch.equal(heads.layer_norm_backward(*args, w, r.mean, r.rstd, out=o).dx, full.dx)


# ---- a teacher's share of a class that the student has masked -----------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [9, 1401, 140001])
def test_a_teachers_share_of_a_masked_class(v, t):
    """Any share within fp32's range makes the loss infinite; one beyond it (e^-200) is none, and the rest of the row keeps its
    digits."""
    from wfd_gan_amd import heads
    x = torch.randn(3, v, generator=gen(v)).to(t)
    x[:, 1] = -INF
    ti = torch.tensor([[0, 1, 2]] * 3, dtype=torch.int32)
    tv = torch.tensor([[0.5, -60.0, 0.2], [0.5, -200.0, 0.2], [0.5, -INF, 0.2]])
    r = heads.distill_loss(x.to(DEV), ti.to(DEV), tv.to(DEV))
    assert float(r.loss[0]) == INF and float(r.loss[1]) != INF
    one = torch.ones(2)
    loss, bl, d, bd = R.distill(x[1:], torch.tensor([[0, -1, 2]] * 2), tv[1:], None, 1.0, 1.0, 0.0, one)
    R.check(r.loss[1:], loss, bl, F32, "loss")
    R.check(r.dlogits[1:], d, bd, t, "dlogits")
    assert bool(r.dlogits[0].isfinite().all())
