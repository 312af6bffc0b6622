"""GPU: the classifier-head operators (wfd_gan_amd.heads) against their definitions in 64 bits (tests/heads_ref.py, which also
derives the tolerances): sizes around every border of the kernels, strides and alignments, masked rows, ties, non-finite
values, broadcast and repeated operands, streams, captured graphs, and the run of them as a student's training step."""
import math

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


def randn(g, *shape, t=F32):
    return torch.randn(*shape, generator=g).to(t)


def strided(t, pad, off):
    """The same values as rows of a wider device tensor that begin ``off`` elements in."""
    m, n = t.shape
    wide = torch.full((m, n + pad + off), float("nan"), dtype=t.dtype, device=DEV)
    view = wide[:, off:off + n]
    view.copy_(t)
    return view


# ---- layer norm ------------------------------------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (5, 2), (33, 7), (3, 8), (130, 64), (17, 127), (9, 128), (4, 129), (70, 257), (21, 511), (64, 512),
              (3, 513), (10, 1000), (5, 1024), (13, 1401), (3, 2047), (6, 2048), (2, 2049), (3, 4096), (2, 4099), (2, 8192),
              (1, 8200), (2, 16384), (2, 16385), (1, 32768), (2, 40001), (1, 70000)]


def norm_inputs(m, n, t, wt, seed, w=True, b=True):
    g = gen(seed)
    x = (randn(g, m, n) * 1.5 + 3 * randn(g, n)).to(t)
    return x, (1 + 0.3 * randn(g, n)).to(wt) if w else None, (0.5 * randn(g, n)).to(wt) if b else None, randn(g, m, n).to(t)


def dev(t):
    return None if t is None else t.to(DEV)


def check_norm(x, w, b, dy, eps, xd, dyd):
    from wfd_gan_amd import heads
    t, wt = x.dtype, (w if w is not None else b if b is not None else torch.empty(0)).dtype
    y, mean, rstd, by, bm, br = R.layer_norm(x, w, b, eps)
    got = heads.layer_norm(xd, dev(w), dev(b), eps)
    R.check(got.y, y, by, t, "y")
    R.check(got.mean, mean, bm, F32, "mean")
    R.check(got.rstd, rstd, br * rstd, F32, "rstd")
    back = heads.layer_norm_backward(dyd, xd, dev(w), got.mean, got.rstd, bias=True)
    dx, dw, db, bdx, bdw, bdb = R.layer_norm_backward(dy, x, w, got.mean, got.rstd)
    R.check(back.dx, dx, bdx, t, "dx")
    if w is not None:
        R.check(back.dweight, dw, bdw, wt, "dweight")
    else:
        assert back.dweight is None
    R.check(back.dbias, db, bdb, wt if w is not None else F32, "dbias")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", NORM_SIZES)
def test_norm_sizes(size, t):
    m, n = size
    for wt in {t, F32}:
        x, w, b, dy = norm_inputs(m, n, t, wt, seed=m * 131 + n)
        check_norm(x, w, b, dy, 1e-5, x.to(DEV), dy.to(DEV))


@pytest.mark.parametrize("t", TYPES)
def test_norm_many_rows(t):
    for m, n in ((9001, 100), (4097, 520), (2050, 1401), (1030, 4100)):
        x, w, b, dy = norm_inputs(m, n, t, F32, seed=m)
        check_norm(x, w, b, dy, 1e-5, x.to(DEV), dy.to(DEV))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [3, 5, 64, 127, 129, 513, 1000, 1401, 2047, 2049, 4096, 4099, 6001, 8192, 8200, 16384])
def test_norm_backward_on_both_sides_of_few_rows(n, t):
    """Few rows are done in one launch, more with partial sums: every team's form on both sides of the borders, with strides, in
    place, and without some of the weights' gradients."""
    from wfd_gan_amd import heads
    few = 1024 if t != F32 or n <= 2048 else 512
    for m in (few, few + 1):
        x, w, b, dy = norm_inputs(m, n, t, F32, seed=n + m)
        xd, dyd, wd = strided(x, 3, 1), strided(dy, 2, 1), dev(w)
        check_norm(x, w, b, dy, 1e-5, xd, dyd)
        r = heads.layer_norm(xd, wd, dev(b))
        full = heads.layer_norm_backward(dyd, xd, wd, r.mean, r.rstd)
        for where in ("dy", "x"):
            dd, xx = dyd.clone(memory_format=torch.contiguous_format), xd.clone(memory_format=torch.contiguous_format)
            o = full._replace(dx=dd if where == "dy" else xx, dweight=torch.empty_like(wd), dbias=torch.empty_like(wd))
            g = heads.layer_norm_backward(dd, xx, wd, r.mean, r.rstd, out=o)
            assert torch.equal(g.dx, full.dx) and torch.equal(g.dweight, full.dweight) and torch.equal(g.dbias, full.dbias)
        for dw, db in ((None, full.dbias), (full.dweight, None), (None, None)):
            o = full._replace(dx=torch.empty_like(full.dx), dweight=None if dw is None else torch.empty_like(dw),
                              dbias=None if db is None else torch.empty_like(db))
            g = heads.layer_norm_backward(dyd, xd, wd, r.mean, r.rstd, out=o)
            assert torch.equal(g.dx, full.dx)
            assert all(a is None if c is None else torch.equal(a, c) for a, c in ((g.dweight, dw), (g.dbias, db)))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [3, 64, 1401, 2048, 9000, 33001])
def test_norm_strides_and_missing_weights(n, t):
    for k, (w, b) in enumerate(((True, False), (False, True), (False, False))):
        x, w, b, dy = norm_inputs(6, n, t, t, seed=n + k, w=w, b=b)
        check_norm(x, w, b, dy, 1e-5, strided(x, 5, k), strided(dy, 3, k + 1))
    # operands on odd places of a larger buffer, a transposed input (copied), a broadcast gradient (stride 0, copied)
    x, w, b, dy = norm_inputs(6, n, t, t, seed=n)
    buf = torch.zeros(2 * n + 3, dtype=t, device=DEV)
    wd, bd = buf[1:n + 1], buf[n + 2:2 * n + 2]
    wd.copy_(w), bd.copy_(b)
    from wfd_gan_amd import heads
    got = heads.layer_norm(x.t().contiguous().to(DEV).t(), wd, bd, 1e-5)
    assert torch.equal(got.y, heads.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5).y)
    one = dy[:1].to(DEV).expand(6, n)
    a = heads.layer_norm_backward(one, x.to(DEV), wd, got.mean, got.rstd)
    c = heads.layer_norm_backward(one.contiguous(), x.to(DEV), wd, got.mean, got.rstd)
    assert all(torch.equal(p, q) for p, q in zip(a[:3], c[:3]))


def test_norm_leading_dimensions_empty_and_constant_rows():
    from wfd_gan_amd import heads
    x, w, b, dy = (dev(v) for v in norm_inputs(12, 96, BF16, F32, seed=1))
    flat = heads.layer_norm(x, w, b)
    cube = heads.layer_norm(x.view(2, 3, 2, 96), w, b)
    assert cube.y.shape == (2, 3, 2, 96) and cube.mean.shape == (2, 3, 2)
    assert torch.equal(cube.y.view(12, 96), flat.y) and torch.equal(cube.rstd.view(12), flat.rstd)
    bare = heads.layer_norm(x, w, b, stats=False)
    assert bare.mean is None and torch.equal(bare.y, flat.y)
    row = heads.layer_norm(x[0], w, b)
    assert row.y.shape == (96,) and torch.equal(row.y, flat.y[0])
    none = torch.empty(0, 96, dtype=BF16, device=DEV)
    r = heads.layer_norm(none, w, b)
    g = heads.layer_norm_backward(none, none, w, r.mean, r.rstd)
    assert r.y.shape == (0, 96) and float(g.dweight.abs().max()) == 0 and float(g.dbias.abs().max()) == 0
    half = w.to(BF16)
    g = heads.layer_norm_backward(none, none, half, r.mean, r.rstd)
    assert float(g.dweight.abs().max()) == 0 and g.dweight.dtype == BF16
    # a constant row has variance 0: y = bias exactly
    same = torch.full((3, 1401), 7.25, dtype=F16, device=DEV)
    r = heads.layer_norm(same, None, None, 1e-5)
    assert float(r.y.abs().max()) == 0 and torch.allclose(r.rstd, torch.full_like(r.rstd, 1e-5 ** -0.5), rtol=1e-6)


def test_norm_large_offset_and_non_finite_rows():
    """The variance is taken about the mean: an offset of 10^4 leaves the digits that fp32 inputs have."""
    from wfd_gan_amd import heads
    x, w, b, dy = norm_inputs(4, 2048, F32, F32, seed=3)
    x = x + 1e4
    check_norm(x, w, b, dy, 1e-5, x.to(DEV), dy.to(DEV))
    x[1, 5], x[2, 7] = float("nan"), INF
    got = heads.layer_norm(x.to(DEV), dev(w), dev(b))
    assert bool(got.y[1:3].isnan().all()) and bool(got.y[0].isfinite().all()) and bool(got.y[3].isfinite().all())


def test_norm_in_place_and_reused_results():
    from wfd_gan_amd import heads
    for n in (128, 1401, 5000, 36000):
        x, w, b, dy = (dev(v) for v in norm_inputs(7, n, BF16, F32, seed=n))
        want = heads.layer_norm(x, w, b)
        back = heads.layer_norm_backward(dy, x, w, want.mean, want.rstd)
        out = heads.norm_output_like(x)
        again = heads.layer_norm(x, w, b, out=out)
        assert again.y is out.y and torch.equal(again.y, want.y)
        for where in ("dy", "x"):
            dd, xx = dy.clone(), x.clone()
            o = heads.norm_gradients_like(x, w, b)._replace(dx=dd if where == "dy" else xx)
            g = heads.layer_norm_backward(dd, xx, w, want.mean, want.rstd, out=o)
            assert torch.equal(g.dx, back.dx) and torch.equal(g.dweight, back.dweight) and torch.equal(g.dbias, back.dbias)
        xx = x.clone()
        heads.layer_norm(xx, w, b, out=out._replace(y=xx))
        assert torch.equal(xx, want.y)


def test_norm_gradient_against_differences():
    """Directional derivative of <y, dy> by central differences in 64 bits along random directions, from the kernels' dx, dw, db."""
    from wfd_gan_amd import heads
    x, w, b, dy = norm_inputs(5, 37, F32, F32, seed=9)
    r = heads.layer_norm(dev(x), dev(w), dev(b))
    g = heads.layer_norm_backward(dev(dy), dev(x), dev(w), r.mean, r.rstd)
    f = lambda xx, ww, bb: float((R.layer_norm(xx, ww, bb, 1e-5)[0] * dy.double()).sum())
    X, W, B = x.double(), w.double(), b.double()
    for k in range(4):
        gg = gen(50 + k)
        vx, vw, vb = (torch.randn(v.shape, generator=gg).double() for v in (X, W, B))
        h = 1e-5
        num = (f(X + h * vx, W + h * vw, B + h * vb) - f(X - h * vx, W - h * vw, B - h * vb)) / (2 * h)
        ana = float((g.dx.cpu().double() * vx).sum() + (g.dweight.cpu().double() * vw).sum() + (g.dbias.cpu().double() * vb).sum())
        # fp32 sums of ~260 terms of size ~1 (1e-5), differences: h^2 f''' + rounding / h (1e-8)
        assert abs(num - ana) < 1e-4


# ---- scores ------------------------------------------------------------------------------------------------------------
CLASSES = [1, 2, 3, 7, 16, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 500, 511, 513, 1000, 1024, 1025, 1401, 2047, 2048,
           2049, 3001, 4096, 4097, 8191, 8193, 10007, 16385, 32000, 40003, 50257, 65537, 131075, 262147]


def logits_of(m, v, t, seed, spread=3.0):
    return (torch.randn(m, v, generator=gen(seed)) * spread).to(t)


def check_scores(x, y, k, temp, xd):
    from wfd_gan_amd import heads
    got = heads.label_logprobs(xd, dev(y), k, temperature=temp)
    want = R.scores(x, y, k, temp)
    R.check(got.entropy, want["entropy"], want["b_entropy"], F32, "entropy")
    if y is not None:
        R.check(got.logprob, want["logprob"], want["b_logprob"], F32, "logprob")
    if k:
        assert torch.equal(got.top_index.cpu().long(), want["top_index"]), "top_index"
        R.check(got.top_logprob, want["top_logprob"], want["b_top"], F32, "top_logprob")
    return got


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", CLASSES)
def test_scores_sizes(v, t):
    for m, k, temp in ((1, min(v, 20), 1.0), (3, min(v, 64), 0.7), (5, 0, 2.0), (70 if v < 5000 else 9, min(v, 5), 1.0)):
        x = logits_of(m, v, t, seed=v + m)
        y = torch.randint(0, v, (m,), generator=gen(v), dtype=torch.int32)
        check_scores(x, y, k, temp, x.to(DEV))


@pytest.mark.parametrize("t", TYPES)
def test_scores_many_rows(t):
    for m, v, k in ((5000, 100, 5), (3000, 37, 37), (1500, 1401, 10), (700, 9001, 20), (600, 33000, 1)):
        x = logits_of(m, v, t, seed=m)
        y = torch.randint(-1, v, (m,), generator=gen(v), dtype=torch.int32)
        check_scores(x, y, k, 1.0, x.to(DEV))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [5, 100, 1401, 5000, 40003])
def test_scores_masks_ties_and_order(v, t):
    """Rows: all -inf; all the type's lowest value; one class left; fewer classes left than alternatives; all equal; ascending;
    descending; few distinct values; zeros of both signs; half of the classes at the lowest value; one huge value."""
    low = torch.finfo(t).min
    x = logits_of(12, v, t, seed=v)
    g = gen(v + 1)
    x[0] = -INF
    x[1] = low
    x[2] = -INF
    x[2, v // 2] = 1.5
    x[3, 3:] = -INF
    x[4] = 0.25
    x[5] = torch.linspace(-20, 20, v)
    x[6] = torch.linspace(20, -20, v)
    x[7] = torch.randint(0, 3, (v,), generator=g).to(t)
    x[8] = torch.where(torch.rand(v, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0)).to(t)
    x[9, ::2] = low
    x[10, v - 1] = 1000.0
    y = torch.tensor([0, v - 1, v // 2, 2, -1, 0, v - 1, 1, 0, 0, v - 1, -100], dtype=torch.int32)
    k = min(v, 20)
    for pad, off in ((0, 0), (3, 1)):
        check_scores(x, y, k, 1.0, strided(x, pad, off) if pad else x.to(DEV))
    check_scores(x[:, : v], y, min(v, 64), 0.5, x.to(DEV))
    for r in range(12):                                  # the same rows one at a time: the form that splits a row
        check_scores(x[r:r + 1], y[r:r + 1], k, 1.0, x[r:r + 1].to(DEV))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [3, 2050])
def test_scores_where_large_values_stand_together(m, t):
    """Rows that rise, fall, drift, or have one high run: the lists run over and the k-th value itself is looked for."""
    g = gen(m)
    for v in (100, 300, 600, 1024, 1401, 2048, 2100, 4000, 16000, 20000) + ((131072,) if m == 3 else ()):
        rows = min(m, 2050 if v <= 4000 else 3)
        x = randn(g, rows, v) * 3
        kind = torch.arange(rows) % 5
        rise = x.sort(1).values
        x = torch.where((kind == 0)[:, None], rise, x)
        x = torch.where((kind == 1)[:, None], rise.flip(1), x)
        x = torch.where((kind == 2)[:, None], x - torch.arange(v) * (20.0 / v), x)
        high = torch.zeros(v)
        high[v // 3: v // 3 + 250] = 30.0
        x = torch.where((kind == 3)[:, None], x + high, x)
        x = torch.where((kind == 4)[:, None], (rise * 2).round() / 2, x).to(t)
        y = torch.randint(0, v, (rows,), generator=g).to(torch.int32)
        for k in (7, 64):
            check_scores(x, y, k, 1.0, strided(x, 1, 1) if v == 4000 else x.to(DEV))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [1, 48, 49, 64])
def test_scores_of_many_rows_pick_what_few_rows_pick(k, t):
    """Around the sizes where a wave takes a row of its own if there are many: the same alternatives as for 40 of the rows."""
    from wfd_gan_amd import heads
    g = torch.Generator(device=DEV).manual_seed(k)
    for v in (1025, 1060, 1151, 1153, 1400, 2049, 2100, 2303, 2305, 4100) + ((8191, 8193) if t == F32 else (16384, 16391)):
        x = torch.randn(2048, v, generator=g, device=DEV).to(t)
        x[:, ::7] = -INF
        y = torch.randint(0, v, (2048,), generator=g, device=DEV, dtype=torch.int32)
        a = heads.label_logprobs(x, y, k)
        for lo in (0, 1000, 2008):
            s = slice(lo, lo + 40)
            b = heads.label_logprobs(x[s], y[s], k)
            assert torch.equal(a.top_index[s], b.top_index)
            want = R.scores(x[s].cpu(), y[s].cpu(), k, 1.0)
            assert torch.equal(a.top_index[s].cpu().long(), want["top_index"])
            R.check(a.logprob[s], want["logprob"], want["b_logprob"], F32, "logprob")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [1, 2, 100, 1401, 5000, 40003])
def test_scores_of_a_class_alone_in_its_row(v, t):
    """Everything else masked: probability 1 and entropy 0, to the bit, at any value and temperature."""
    from wfd_gan_amd import heads
    m = 40
    g = gen(v)
    x = torch.full((m, v), -INF, dtype=t)
    at = torch.randint(0, v, (m,), generator=g)
    x[torch.arange(m), at] = (randn(g, m) * 20).to(t)
    for rows in (1, m):
        for temp in (0.3, 1.0, 7.0):
            r = heads.label_logprobs(x[:rows].to(DEV), at[:rows].to(torch.int32).to(DEV), 1, temperature=temp)
            assert float(r.logprob.abs().max()) == 0 and float(r.entropy.abs().max()) == 0
            assert float(r.top_logprob.abs().max()) == 0 and torch.equal(r.top_index[:, 0].cpu().long(), at[:rows])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [6, 1401, 40003])
def test_scores_non_finite_and_wrong_labels(v, t):
    from wfd_gan_amd import heads
    x = logits_of(5, v, t, seed=v)
    x[0, 3] = float("nan")
    x[1] = -INF
    x[1, 4] = float("nan")
    x[2, 2] = INF
    x[3, 5], x[3, 1] = float("nan"), float("nan")
    y = torch.tensor([0, 4, 2, 1, v], dtype=torch.int32)
    for rows in (slice(0, 5), slice(0, 1), slice(1, 2), slice(2, 3), slice(3, 4)):
        got = heads.label_logprobs(x[rows].to(DEV), y[rows].to(DEV), 5)
        want = R.scores(x[rows], y[rows], 5, 1.0)
        assert torch.equal(got.top_index.cpu().long(), want["top_index"])
        for r, name in ((got.entropy, "entropy"), (got.logprob, "logprob"), (got.top_logprob, "top")):
            bad = r.cpu().isnan().reshape(r.shape[0], -1)
            assert bool(bad[: 4 if rows.stop == 5 else 1].all()), name
    got = heads.label_logprobs(x.to(DEV), y.to(DEV), 5)
    assert bool(got.logprob[4].isnan()) and bool(got.entropy[4].isfinite())
    d = heads.label_logprobs_backward(x.to(DEV), y.to(DEV), got, torch.ones(5, device=DEV), torch.ones(5, device=DEV))
    assert bool(d.isnan().all())


def test_scores_many_equal_maxima_beyond_any_buffer():
    """Thousands of classes share the largest values, so that the alternatives are decided by index alone."""
    for t in TYPES:
        for v in (3000, 20011, 150001):
            x = torch.full((3, v), -1.0).to(t)
            x[0, ::3] = 2.0
            x[1, v // 2:] = 2.0
            x[2, v - 40:] = 2.0
            x[2, v - 30] = 3.0
            check_scores(x, None, 64, 1.0, x.to(DEV))
            for r in range(3):
                check_scores(x[r:r + 1], None, 64, 1.0, x[r:r + 1].to(DEV))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [1, 2, 5, 64, 100, 129, 1000, 1401, 4097, 33001])
def test_scores_backward(v, t):
    from wfd_gan_amd import heads
    low = torch.finfo(t).min
    m = 9
    x = logits_of(m, v, t, seed=3 * v)
    x[1] = -INF
    if v > 3:
        x[2, 1:] = -INF
        x[3, ::2] = low
        x[4] = low
        x[5] = 0.5
    y = torch.randint(0, v, (m,), generator=gen(v), dtype=torch.int32)
    y[6] = -1
    dl, dh = randn(gen(1), m), randn(gen(2), m)
    for k, (xd, temp) in enumerate(((x.to(DEV), 1.0), (strided(x, 4, 1), 0.7), (strided(x, 8, 0), 3.0))):
        got = heads.label_logprobs(xd, y.to(DEV), temperature=temp)
        for a, b in ((dl, dh), (dl, None), (None, dh)):
            d = heads.label_logprobs_backward(xd, y.to(DEV) if a is not None else None, got, dev(a), dev(b), temperature=temp)
            want, bound = R.scores_backward(x, y if a is not None else None, got.stat, got.entropy, a, b, temp)
            R.check(d, want, bound, t, f"dlogits {k}")
    # over the logits themselves
    xd = x.to(DEV)
    got = heads.label_logprobs(xd, y.to(DEV))
    want = heads.label_logprobs_backward(xd, y.to(DEV), got, dev(dl), dev(dh))
    heads.label_logprobs_backward(xd, y.to(DEV), got, dev(dl), dev(dh), out=xd)
    assert torch.equal(xd, want)


def test_scores_of_split_rows_are_the_same_every_time():
    """Which thread writes an alternative depends on the order of arrival; every thread holds the same statistics."""
    from wfd_gan_amd import heads
    for seed in (21, 22, 23):
        x = logits_of(20, 70001, BF16, seed=seed, spread=2.5).to(DEV)
        first = heads.label_logprobs(x, None, 9)
        for _ in range(20):
            again = heads.label_logprobs(x, None, 9)
            assert torch.equal(again.top_logprob, first.top_logprob) and torch.equal(again.top_index, first.top_index)
        # the first alternative is the maximum: its log probability is the one in stat
        assert torch.equal(first.top_logprob[:, 0], -first.stat[:, 1])


def test_scores_gradient_against_differences():
    from wfd_gan_amd import heads
    x = logits_of(4, 23, F32, seed=5)
    y = torch.tensor([0, 22, 7, -1], dtype=torch.int32)
    dl, dh = randn(gen(3), 4), randn(gen(4), 4)
    got = heads.label_logprobs(x.to(DEV), y.to(DEV), temperature=0.8)
    d = heads.label_logprobs_backward(x.to(DEV), y.to(DEV), got, dev(dl), dev(dh), temperature=0.8).cpu().double()

    def f(xx):
        r = R.scores(xx, y, 0, 0.8)
        return float((r["logprob"] * dl.double() + r["entropy"] * dh.double()).sum())
    for k in range(4):
        v = torch.randn(x.shape, generator=gen(60 + k)).double()
        num = (f(x.double() + 1e-5 * v) - f(x.double() - 1e-5 * v)) / 2e-5
        assert abs(num - float((d * v).sum())) < 5e-5          # fp32 gradients: 92 terms below 3, 4 U each


def test_scores_leading_dimensions_reuse_and_no_labels():
    from wfd_gan_amd import heads
    x = logits_of(12, 300, BF16, seed=2).to(DEV)
    y = torch.arange(12, dtype=torch.int32, device=DEV)
    a = heads.label_logprobs(x, y, 3)
    b = heads.label_logprobs(x.view(3, 4, 300), y.view(3, 4), 3)
    assert b.logprob.shape == (3, 4) and b.top_index.shape == (3, 4, 3) and b.stat.shape == (3, 4, 2)
    assert all(torch.equal(p.reshape(-1), q.reshape(-1)) for p, q in zip(a[:5], b[:5]))
    out = heads.scores_like(x, 3)
    c = heads.label_logprobs(x, y, 3, out=out)
    assert c is out and all(torch.equal(p, q) for p, q in zip(a[:5], c[:5]))
    n = heads.label_logprobs(x, None, 3)
    assert n.logprob is None and torch.equal(n.entropy, a.entropy) and torch.equal(n.top_index, a.top_index)
    e = heads.label_logprobs(x[:0], y[:0], 3)
    assert e.logprob.shape == (0,) and e.top_index.shape == (0, 3)
    one = heads.label_logprobs(x[0], y[0], 3)
    assert one.logprob.shape == () and torch.equal(one.top_index, a.top_index[0])


# ---- distillation --------------------------------------------------------------------------------------------------------
def distill_inputs(m, v, k, t, seed):
    g = gen(seed)
    x = (torch.randn(m, v, generator=g) * 2.5).to(t)
    ti = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(m)]).to(torch.int32) if k else \
        torch.empty(m, 0, dtype=torch.int32)
    tv = torch.randn(m, k, generator=g) * 3
    y = torch.randint(0, v, (m,), generator=g, dtype=torch.int32)
    rs = torch.rand(m, generator=g) + 0.25
    return x, ti, tv, y, rs


def check_distill(x, ti, tv, y, temp, w, u, rs, gs, xd, grad=True):
    from wfd_gan_amd import heads
    got = heads.distill_loss(xd, dev(ti), dev(tv), dev(y), temperature=temp, weight=w, label_weight=u, row_scale=dev(rs),
                             grad_scale=gs, grad=grad)
    scale = (rs if rs is not None else torch.ones(x.shape[0])).double() * gs
    loss, bl, d, bd = R.distill(x, ti, tv, y, temp, w, u, scale)
    R.check(got.loss, loss, bl, F32, "loss")
    if grad:
        R.check(got.dlogits, d, bd, x.dtype, "dlogits")
    else:
        assert got.dlogits is None
    return got


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [1, 2, 5, 64, 100, 127, 129, 257, 512, 1000, 1401, 2048, 2049, 4097, 8200, 16385, 32000, 50257, 65537,
                               70001, 131075])
def test_distill_sizes(v, t):
    for m, k, temp, w, u in ((1, min(v, 8), 1.0, 1.0, 0.0), (7, min(v, 64), 2.0, 0.7, 0.3), (3, 1, 0.5, 1.0, 0.0),
                             (40 if v < 5000 else 5, min(v, 16), 1.0, 0.5, 0.5), (4, 0, 1.0, 0.0, 1.0)):
        x, ti, tv, y, rs = distill_inputs(m, v, k, t, seed=v + m)
        check_distill(x, ti, tv, y, temp, w, u, rs, 1.0, x.to(DEV))


@pytest.mark.parametrize("t", TYPES)
def test_distill_many_rows_and_loss_alone(t):
    for m, v, k in ((4000, 100, 8), (2500, 33, 33), (900, 1401, 256), (300, 200, 200), (600, 9001, 20)):
        x, ti, tv, y, rs = distill_inputs(m, v, k, t, seed=m)
        for temp, w, u in ((2.0, 0.5, 0.5), (1.0, 1.0, 0.0)):
            a = check_distill(x, ti, tv, y, temp, w, u, rs, 0.5, x.to(DEV))
            b = check_distill(x, ti, tv, y, temp, w, u, rs, 0.5, x.to(DEV), grad=False)
            assert torch.equal(a.loss, b.loss)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [9, 100, 1401, 20011, 140001])
def test_distill_masks_repeats_and_missing_entries(v, t):
    """Rows: a repeated index; the label among the entries; no entry; all entries -inf; entries -inf among others; student all -inf;
    student -inf where the teacher is not, and where it is; no label; student at the type's lowest value; row_scale 0."""
    m, k = 12, min(v, 9)
    x, ti, tv, y, rs = distill_inputs(m, v, k, t, seed=v)
    ti[0, :4] = ti[0, 5]
    y[1] = ti[1, 2]
    ti[2] = -1
    tv[3] = -INF
    tv[4, ::2] = -INF
    x[5] = -INF
    free = [i for i in range(v) if i not in set(ti[6].tolist())]
    x[6, free[0] if free else 0] = -INF
    x[7, ti[7, 1].long()] = -INF
    y[7] = ti[7, 0]
    y[8] = -7
    x[9] = torch.finfo(t).min
    rs[10] = 0.0
    ti[11, 1::2] = -5
    for pad, off in ((0, 0), (2, 1), (8, 0)):
        xd = strided(x, pad, off) if pad else x.to(DEV)
        for temp, w, u in ((1.0, 1.0, 0.0), (2.0, 0.6, 0.4), (1.0, 0.5, 0.5), (1.0, 0.0, 1.0)):
            check_distill(x, ti, tv, y, temp, w, u, rs, 1.0, xd)
    for r in range(m):
        check_distill(x[r:r + 1], ti[r:r + 1], tv[r:r + 1], y[r:r + 1], 1.5, 0.6, 0.4, rs[r:r + 1], 2.0, x[r:r + 1].to(DEV))


@pytest.mark.parametrize("v", [7, 1401, 40003, 140001])
def test_distill_wrong_index_and_label_show(v):
    from wfd_gan_amd import heads
    x, ti, tv, y, rs = distill_inputs(4, v, 5, BF16, seed=v)
    ti[1, 3] = v
    y[2] = v + 3
    got = check_distill(x, ti, tv, y, 1.0, 0.5, 0.5, rs, 1.0, x.to(DEV))
    assert got.loss.isnan().tolist() == [False, True, True, False]
    only = heads.distill_loss(x.to(DEV), dev(ti), dev(tv), dev(y), weight=0.0, label_weight=1.0)
    assert only.loss.isnan().tolist() == [False, False, True, False]            # entries without weight are not read


def test_distill_in_place_equals_out_of_place():
    from wfd_gan_amd import heads
    for v in (100, 1401, 33000, 70000, 140001):
        for m in (2, 6):
            x, ti, tv, y, rs = (dev(a) for a in distill_inputs(m, v, 16, BF16, seed=v))
            want = heads.distill_loss(x, ti, tv, y, temperature=2.0, weight=0.5, label_weight=0.5, row_scale=rs)
            out = heads.distill_output_like(x)._replace(dlogits=x)
            got = heads.distill_loss(x, ti, tv, y, temperature=2.0, weight=0.5, label_weight=0.5, row_scale=rs, out=out)
            assert torch.equal(got.loss, want.loss) and torch.equal(x, want.dlogits)


def test_distill_teacher_sure_beyond_the_range_of_exponentials():
    """Entries 60 to 130 below the best one: shares that are tiny, subnormal or zero in fp32 add nothing worth a digit."""
    for t in TYPES:
        x, ti, tv, y, rs = distill_inputs(8, 300, 60, t, seed=4)
        tv = -torch.linspace(0, 130, 60).repeat(8, 1)
        tv[:, 1:] -= 2.0
        check_distill(x, ti, tv, y, 1.0, 1.0, 0.0, rs, 1.0, x.to(DEV))
        check_distill(x, ti, tv, y, 0.9, 0.5, 0.5, rs, 1.0, x.to(DEV))


def test_distill_gradient_against_differences():
    x, ti, tv, y, rs = distill_inputs(4, 19, 6, F32, seed=8)
    ti[0, 1] = ti[0, 0]
    got = check_distill(x, ti, tv, y, 1.7, 0.6, 0.4, rs, 1.0, x.to(DEV))
    d = got.dlogits.cpu().double()
    f = lambda xx: float((R.distill(xx, ti, tv, y, 1.7, 0.6, 0.4, rs)[0] * rs.double()).sum())
    for k in range(4):
        v = torch.randn(x.shape, generator=gen(70 + k)).double()
        num = (f(x.double() + 1e-5 * v) - f(x.double() - 1e-5 * v)) / 2e-5
        assert abs(num - float((d * v).sum())) < 2e-5


# ---- streams, graphs, the whole run ----------------------------------------------------------------------------------------
def _all_ops(heads, s, out):
    n = heads.layer_norm(s["x"], s["w"], s["b"], out=out["norm"])
    g = heads.layer_norm_backward(s["dy"], s["x"], s["w"], n.mean, n.rstd, out=out["normb"])
    a = heads.label_logprobs(s["logits"], s["y"], 7, out=out["scores"])
    d = heads.label_logprobs_backward(s["logits"], s["y"], a, s["dl"], s["dh"], out=out["scoresb"])
    e = heads.distill_loss(s["logits"], s["ti"], s["tv"], s["y"], temperature=2.0, weight=0.5, label_weight=0.5, out=out["distill"])
    return [n.y, n.mean, n.rstd, g.dx, g.dweight, g.dbias, a.logprob, a.entropy, a.stat, a.top_logprob, a.top_index, d, e.loss,
            e.dlogits]


def _state(seed, rows, n, v, t):
    from wfd_gan_amd import heads
    x, w, b, dy = (dev(a) for a in norm_inputs(rows, n, t, F32, seed))
    lg, ti, tv, y, rs = (dev(a) for a in distill_inputs(rows, v, 7, t, seed))
    s = dict(x=x, w=w, b=b, dy=dy, logits=lg, ti=ti, tv=tv, y=y, dl=rs, dh=-rs)
    out = dict(norm=heads.norm_output_like(x), normb=heads.norm_gradients_like(x, w, b), scores=heads.scores_like(lg, 7),
               scoresb=torch.empty_like(lg), distill=heads.distill_output_like(lg))
    return s, out


SHAPES = [(3, 700, 60001, BF16), (300, 1401, 5001, F16), (64, 512, 100, F32)]


@pytest.mark.parametrize("shape", SHAPES)
def test_two_streams_at_once_and_repeats_are_bit_identical(shape):
    from wfd_gan_amd import heads
    states = [_state(k, *shape) for k in (1, 2)]
    want = [[t.clone() for t in _all_ops(heads, s, o)] for s, o in states]
    torch.cuda.synchronize()
    for _, o in states:
        for r in o.values():
            for t in (r if isinstance(r, tuple) else (r,)):
                if t is not None:
                    t.zero_()
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for rep in range(3):
        for (s, o), st in zip(states, streams):
            with torch.cuda.stream(st):
                _all_ops(heads, s, o)
    torch.cuda.synchronize()
    for (s, o), w in zip(states, want):
        got = [o["norm"].y, o["norm"].mean, o["norm"].rstd, *o["normb"][:3], *o["scores"][:5], o["scoresb"], *o["distill"][:2]]
        assert all(torch.equal(p, q) for p, q in zip(got, w))


@pytest.mark.parametrize("shape", SHAPES)
def test_captured_and_replayed(shape):
    """Two graphs of all five calls, replayed several times with eager work of the same operators in between and new inputs in
    the captured buffers: every replay gives the eager result of the inputs it finds."""
    from wfd_gan_amd import heads
    states = [_state(k, *shape) for k in (3, 4)]
    graphs = []
    side = torch.cuda.Stream()
    for s, o in states:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _all_ops(heads, s, o)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = _all_ops(heads, s, o)
        graphs.append((gr, res))
    for rep in range(4):
        for (s, o), (gr, res) in zip(states, graphs):
            fresh, fo = _state(10 + rep, *shape)
            for key in s:
                s[key].copy_(fresh[key])
            for t in res:
                t.zero_()
            gr.replay()
            eager = _all_ops(heads, fresh, fo)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(res, eager)), rep


def test_results_do_not_touch_their_neighbours():
    """Results inside a larger buffer: what lies before and behind them stays."""
    from wfd_gan_amd import heads
    for t in TYPES:
        for m, n in ((3, 7), (5, 1401), (2, 5003), (1, 40001)):
            x, w, b, dy = (dev(a) for a in norm_inputs(m, n, t, F32, seed=n))
            lg, ti, tv, y, rs = (dev(a) for a in distill_inputs(m, n, 3, t, seed=n))

            def guarded(numel, dt):
                buf = torch.full((numel + 64,), 77, dtype=dt, device=DEV)
                return buf, buf[32:32 + numel]
            bufs = []

            def place(shape, dt):
                buf, view = guarded(math.prod(shape), dt)
                bufs.append((buf, view.numel()))
                return view.view(shape)
            no = heads.NormOutput(place((m, n), t), place((m,), F32), place((m,), F32))
            heads.layer_norm(x, w, b, out=no)
            like = heads.norm_gradients_like(x, w, b)
            heads.layer_norm_backward(dy, x, w, no.mean, no.rstd, out=heads.NormGradients(
                place((m, n), t), place((n,), F32), place((n,), F32), place((like.work.numel(),), F32)))
            so = heads.scores_like(lg, 3)
            so = heads.LabelScores(place((m,), F32), place((m,), F32), place((m, 2), F32), place((m, 3), F32),
                                   place((m, 3), torch.int32), None if so.work is None else place((so.work.numel(),), F32))
            heads.label_logprobs(lg, y, 3, out=so)
            heads.label_logprobs_backward(lg, y, so, rs, rs, out=place((m, n), t))
            do = heads.distill_output_like(lg)
            heads.distill_loss(lg, ti, tv, y, label_weight=0.5, out=heads.DistillOutput(
                place((m,), F32), place((m, n), t), None if do.work is None else place((do.work.numel(),), F32)))
            torch.cuda.synchronize()
            for buf, numel in bufs:
                assert bool((buf[:32] == 77).all()) and bool((buf[32 + numel:] == 77).all())


def test_student_step_norm_product_scores_distill():
    """The operators as they are used together: a teacher's head (norm, product, its top alternatives) feeds a student's loss, whose
    gradient goes back through the product (wfd_gemm_f32) and the norm; against the same step in 64 bits with autograd."""
    from wfd_gan_amd import heads
    from wfd_gan_amd._lib import lib
    L = lib()
    st = torch.cuda.current_stream().cuda_stream
    B, F, C, k, T = 64, 512, 100, 8, 2.0
    g = gen(21)
    feat, tfeat = randn(g, B, F), randn(g, B, F)
    W, TW = randn(g, C, F) * 0.06, randn(g, C, F) * 0.15
    nw, nb = 1 + 0.1 * randn(g, F), 0.1 * randn(g, F)
    y = torch.randint(0, C, (B,), generator=g, dtype=torch.int32)

    def product(layout, a, b, m, n, kk):
        out = torch.empty(m, n, device=DEV)
        L.gemm_f32(layout, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), out.data_ptr(), n, 0, m, n, kk, 1, st)
        return out
    fd, Wd = feat.to(DEV), W.to(DEV)
    teacher = heads.label_logprobs(product(0, heads.layer_norm(tfeat.to(DEV), dev(nw), dev(nb)).y, TW.to(DEV), B, C, F), None, k)
    norm = heads.layer_norm(fd, dev(nw), dev(nb))
    logits = product(0, norm.y, Wd, B, C, F)
    loss = heads.distill_loss(logits, teacher.top_index, teacher.top_logprob, dev(y), temperature=T, weight=0.7, label_weight=0.3,
                              grad_scale=1.0 / B)
    dh = product(1, loss.dlogits, Wd, B, F, C)
    dW = product(2, loss.dlogits, norm.y, C, F, B)
    back = heads.layer_norm_backward(dh, fd, dev(nw), norm.mean, norm.rstd)

    D = torch.float64
    f64, W64, nw64, nb64 = (v.to(D).requires_grad_() for v in (feat, W, nw, nb))
    tl = torch.nn.functional.layer_norm(tfeat.to(D), (F,), nw.to(D), nb.to(D), 1e-5) @ TW.to(D).T
    top = tl.log_softmax(1).topk(k, dim=1)
    assert torch.equal(top.indices, teacher.top_index.cpu().long())
    s = torch.nn.functional.layer_norm(f64, (F,), nw64, nb64, 1e-5) @ W64.T
    q = (top.values / T).softmax(1)
    kl = (q * (q.log() - (s / T).log_softmax(1).gather(1, top.indices))).sum(1)
    ce = -s.log_softmax(1).gather(1, y.long()[:, None])[:, 0]
    rows = 0.7 * T * T * kl + 0.3 * ce
    rows.mean().backward()
    # products of 512 terms in fp32: 512 U of the sum of magnitudes, far below 1e-4 of the largest entry of each result
    for got, want in ((loss.loss, rows), (dW, W64.grad), (back.dx, f64.grad), (back.dweight, nw64.grad), (back.dbias, nb64.grad)):
        want = want.detach()
        assert float((got.cpu().double() - want).abs().max()) <= 1e-4 * float(want.abs().max())


def test_rows_beyond_32_bit_offsets():
    """Buffers of more than 2^31 elements: the last rows against the definition, in place where a call allows it."""
    from wfd_gan_amd import heads
    m, v = 33001, 66001                                       # 2.18e9 elements
    x = torch.empty(m, v, dtype=BF16, device=DEV)
    x.fill_(-3.0)
    last = logits_of(3, v, BF16, seed=1)
    x[-3:].copy_(last)
    y = torch.zeros(m, dtype=torch.int32, device=DEV)
    y[-3:] = torch.tensor([5, v - 1, -1], dtype=torch.int32, device=DEV)
    got = heads.label_logprobs(x, y, 5)
    want = R.scores(last, y[-3:].cpu(), 5, 1.0)
    R.check(got.logprob[-3:], want["logprob"], want["b_logprob"], F32, "logprob")
    assert torch.equal(got.top_index[-3:].cpu().long(), want["top_index"])
    assert got.top_index[1000].tolist() == [0, 1, 2, 3, 4]
    ti = torch.zeros(m, 2, dtype=torch.int32, device=DEV)
    tv = torch.zeros(m, 2, device=DEV)
    ti[:, 1] = v - 1
    one = torch.ones(3, dtype=torch.float64)
    loss, bl, d, bd = R.distill(last, ti[-3:].cpu(), tv[-3:].cpu(), None, 1.0, 1.0, 0.0, one)
    out = heads.distill_loss(x, ti, tv, out=heads.DistillOutput(torch.empty(m, device=DEV), x, None))
    R.check(out.loss[-3:], loss, bl, F32, "loss")
    R.check(x[-3:], d, bd, BF16, "dlogits")
    x[-3:].copy_(last)
    dl = torch.ones(m, device=DEV)
    d, bd = R.scores_backward(last, y[-3:].cpu(), got.stat[-3:], got.entropy[-3:], torch.ones(3), None, 1.0)
    heads.label_logprobs_backward(x, y, got, dl, out=x)
    R.check(x[-3:], d, bd, BF16, "scores gradient")
    n = 8000                                                  # the same buffer as 272262 rows of 8000
    rows = x.view(-1)[: (x.numel() // n) * n].view(-1, n)
    r = rows.shape[0]
    a, w, b, dy = norm_inputs(3, n, BF16, F32, seed=2)
    rows.zero_()
    rows[-3:].copy_(a)
    wd, bd_ = w.to(DEV), b.to(DEV)
    g = torch.zeros_like(rows)
    g[-3:].copy_(dy)
    got = heads.layer_norm(rows, wd, bd_)
    yy, mean, rstd, by, bm, br = R.layer_norm(a, w, b, 1e-5)
    R.check(got.y[-3:], yy, by, BF16, "y")
    back = heads.layer_norm_backward(g, rows, wd, got.mean, got.rstd)
    dx, dw, db, bdx, bdw, bdb = R.layer_norm_backward(dy, a, w, got.mean[-3:], got.rstd[-3:])
    R.check(back.dx[-3:], dx, bdx, BF16, "dx")
    R.check(back.dweight, dw, bdw, F32, "dweight")            # every other row has a zero gradient
    assert float(back.dx[:1000].abs().max()) == 0 and r > 2 ** 31 // n
    torch.cuda.synchronize()
    del x, rows, g, got, back
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t", TYPES)
def test_results_beyond_the_caches_have_the_bits_of_smaller_calls(t):
    """A gradient of 250 MB and more is stored another way, and a workgroup then has many rows: bit for bit the same as the calls on
    100 of the rows, on rows that begin on both sides of a 4-byte border."""
    from wfd_gan_amd import heads
    m, v, k = 2001, 63001, 7
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(m, v, generator=g, device=DEV).to(t)
    ti = torch.randint(0, v, (m, k), generator=g, device=DEV, dtype=torch.int32)
    tv = torch.randn(m, k, generator=g, device=DEV)
    y = torch.randint(0, v, (m,), generator=g, device=DEV, dtype=torch.int32)
    a = heads.distill_loss(x, ti, tv, y, temperature=2.0, weight=0.7, label_weight=0.3)
    alone = heads.distill_loss(x, ti, tv, y, temperature=2.0, weight=0.7, label_weight=0.3, grad=False)
    assert torch.equal(a.loss, alone.loss)
    got = heads.label_logprobs(x, y)
    b = heads.label_logprobs_backward(x, y, got, torch.ones(m, device=DEV))
    for lo in (0, 101, 1901):
        s = slice(lo, lo + 100)
        part = heads.distill_loss(x[s], ti[s], tv[s], y[s], temperature=2.0, weight=0.7, label_weight=0.3)
        assert torch.equal(part.loss, a.loss[s]) and torch.equal(part.dlogits, a.dlogits[s])
        mine = heads.LabelScores(*[f[s] if f is not None and f.shape[:1] == (m,) else f for f in got])
        assert torch.equal(heads.label_logprobs_backward(x[s], y[s], mine, torch.ones(100, device=DEV)), b[s])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,v", [(1100, 20001), (600, 40001), (300, 63000), (300, 100001)])
def test_distill_of_many_long_rows_has_the_bits_of_fewer(m, v, t):
    """Workgroups that walk several rows each against calls on 100 of the rows, loss alone against loss with gradient."""
    from wfd_gan_amd import heads
    if t == F32 and v > 65536:
        v = 65535                                             # the longest fp32 row that is not split
    g = torch.Generator(device=DEV).manual_seed(v)
    x = torch.randn(m, v, generator=g, device=DEV).to(t)
    ti = torch.randint(-1, v, (m, 9), generator=g, device=DEV, dtype=torch.int32)
    tv = torch.randn(m, 9, generator=g, device=DEV)
    y = torch.randint(-1, v, (m,), generator=g, device=DEV, dtype=torch.int32)
    for kw in (dict(temperature=2.0, weight=0.7, label_weight=0.3), dict(temperature=1.0)):
        a = heads.distill_loss(x, ti, tv, y, **kw)
        assert torch.equal(heads.distill_loss(x, ti, tv, y, grad=False, **kw).loss, a.loss)
        for lo in (0, m // 2 - 7, m - 100):
            s = slice(lo, lo + 100)
            part = heads.distill_loss(x[s], ti[s], tv[s], y[s], **kw)
            assert torch.equal(part.loss, a.loss[s]) and torch.equal(part.dlogits, a.dlogits[s])
    rows = [0, 1, m // 2, m - 1]
    one = torch.ones(len(rows), dtype=torch.float64)
    loss, bl, d, bd = R.distill(x[rows].cpu(), ti[rows].cpu(), tv[rows].cpu(), None, 1.0, 1.0, 0.0, one)
    R.check(a.loss[rows], loss, bl, F32, "loss")
    R.check(a.dlogits[rows], d, bd, t, "dlogits")


def test_captured_with_results_of_its_own():
    """Calls that make their results inside the capture: fresh memory of the graph's own pool, alive as long as the results."""
    from wfd_gan_amd import heads
    s, _ = _state(7, 20, 300, 70001, BF16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            heads.label_logprobs(s["logits"], s["y"], 9)
            heads.distill_loss(s["logits"], s["ti"], s["tv"])
            heads.layer_norm(s["x"], s["w"], s["b"])
    torch.cuda.current_stream().wait_stream(st)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        a = heads.label_logprobs(s["logits"], s["y"], 9)
        b = heads.distill_loss(s["logits"], s["ti"], s["tv"])
        c = heads.layer_norm(s["x"], s["w"], s["b"])
        d = heads.layer_norm_backward(s["dy"], s["x"], s["w"], c.mean, c.rstd)
    for rep in range(3):
        fresh, _ = _state(20 + rep, 20, 300, 70001, BF16)
        for key in s:
            s[key].copy_(fresh[key])
        gr.replay()
        ea = heads.label_logprobs(fresh["logits"], fresh["y"], 9)
        eb = heads.distill_loss(fresh["logits"], fresh["ti"], fresh["tv"])
        ec = heads.layer_norm(fresh["x"], fresh["w"], fresh["b"])
        ed = heads.layer_norm_backward(fresh["dy"], fresh["x"], fresh["w"], ec.mean, ec.rstd)
        torch.cuda.synchronize()
        for got, want in ((a[:5], ea[:5]), (b[:2], eb[:2]), (c, ec), (d[:3], ed[:3])):
            assert all(torch.equal(p, q) for p, q in zip(got, want)), rep


@pytest.mark.parametrize("temp", [1e-6, 1e-3, 1e3, 1e6])
def test_extreme_temperatures(temp):
    """From one class's share to equal shares: differences come before the division."""
    from wfd_gan_amd import heads
    for t, v in ((F32, 100), (BF16, 5003)):
        x = logits_of(4, v, t, seed=6)
        x[1] = torch.finfo(t).min
        x[2, ::3] = torch.finfo(t).min
        y = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
        got = check_scores(x, y, 5, temp, x.to(DEV))
        d = heads.label_logprobs_backward(x.to(DEV), y.to(DEV), got, torch.ones(4, device=DEV), temperature=temp)
        want, bound = R.scores_backward(x, y, got.stat, got.entropy, torch.ones(4), None, temp)
        R.check(d, want, bound, t, "dlogits")
        ti = torch.tensor([[0, 1, 2], [1, 2, 3], [4, 5, 7], [9, 8, 7]], dtype=torch.int32)
        tv = torch.tensor([[0.0, 1.0, 2.0]]).repeat(4, 1)
        if temp >= 1e-3:                                       # below, T^2 times a difference / T is what is left of fp32's range
            check_distill(x[[0, 3]], ti[[0, 3]], tv[[0, 3]], y[[0, 3]], temp, 0.5, 0.5, torch.ones(2), 1.0, x[[0, 3]].to(DEV))
