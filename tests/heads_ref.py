"""Classifier-head operators from their definitions, in 64 bits on the CPU, with bounds of what fp32 arithmetic may be off.

U = 2^-24 is half a step of fp32; half(t) is half a step of a row type, relative to the value (one rounding of a result)."""
import math

import torch

U = 2.0 ** -24
INF = float("inf")


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the distance between two subnormals: what a rounding near zero may be off."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def layer_norm(x, w, b, eps):
    """(y, mean, rstd, bound of y before its rounding).  A thread adds at most 64 elements in a row before the tree, the
    long form at most N / 1024 more: the mean is off by (80 + N / 1024) U mean|x| at most, the variance by that much relative
    (halved in rstd), and each of the three operations on the way out adds a rounding."""
    x = x.double().cpu()
    n = x.shape[-1]
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.double().cpu()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    c = (80 + n / 1024) * U
    off_mean = c * x.abs().mean(-1, keepdim=True)
    # (x - mean) carries the mean's error and its own rounding; the variance sees the mean's error squared and its own sum
    rel_r = c + off_mean.square() / (var + eps) + 4 * U
    bound = w.abs() * (rstd * (off_mean + U * (x.abs() + mean.abs())) + xh.abs() * rel_r) + 4 * U * ((xh * w).abs() + b.abs())
    return xh * w + b, mean[..., 0], rstd[..., 0], bound, off_mean[..., 0], rel_r[..., 0]


def layer_norm_backward(dy, x, w, mean, rstd):
    """(dx, dw, db, bounds of the three).  Products carry up to 6 roundings, row sums (80 + N / 1024) more; a column sum is at
    most M additions in a row."""
    dy, x = dy.double().cpu(), x.double().cpu()
    mean, rstd = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    m, n = x.shape
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    xh, v = (x - mean) * rstd, dy * w
    c1, c2 = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    c = (88 + n / 1024) * U
    # what the rounding of x - mean leaves in xh
    off_xh = rstd * U * (x.abs() + mean.abs()) + 2 * U * xh.abs()
    o1 = c * v.abs().mean(1, keepdim=True)
    o2 = c * (v * xh).abs().mean(1, keepdim=True) + (v.abs() * off_xh).mean(1, keepdim=True)
    bdx = rstd * (o1 + xh.abs() * o2 + off_xh * c2.abs() + 6 * U * (v.abs() + c1.abs() + (xh * c2).abs()))
    k = (m + 80) * U
    bdw = k * (dy * xh).abs().sum(0) + (dy.abs() * off_xh).sum(0)
    return rstd * (v - c1 - xh * c2), (dy * xh).sum(0), dy.sum(0), bdx, bdw, k * dy.abs().sum(0)


def _exp_sum(x, inv_t):
    """max, z, sum of exp z (all -inf: sum 0 and z = -inf), and the relative bound of that sum in fp32: an exponential is off
    by 4 U and by 3 U |z| through its argument, a thread adds at most max(64, V / 128) of them in a row, 20 more on the way
    to the row's sum."""
    top = x.amax(-1, keepdim=True)
    none = top == -INF
    z = torch.where(none, torch.full_like(x, -INF), (x - top) * inv_t)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    ez = torch.where(e > 0, e * z, torch.zeros_like(z)).sum(-1, keepdim=True)
    one = torch.where(none, torch.ones_like(s), s)
    rel = U * (max(64, x.shape[-1] / 128) + 24 + 3 * (-ez / one))
    return top, none, z, s, ez, rel


def scores(x, y, k, temperature):
    """logprob, entropy, top logprob, top index with the bounds of the first three."""
    x = x.double().cpu()
    v = x.shape[-1]
    top, none, z, s, ez, rel = _exp_sum(x, 1.0 / temperature)
    ln = torch.where(none, torch.zeros_like(s), s.log())
    lp = torch.where(none, torch.full_like(z, -INF), z - ln)
    b_lp = rel + 4 * U * (z.abs() + ln.abs()) + 2 * U
    one = torch.where(none, torch.ones_like(s), s)
    ent = torch.where(none, torch.zeros_like(s), ln - ez / one)[..., 0]
    b_ent = (rel * (1 + 2 * (ez / one).abs()) + 6 * U * (ln.abs() + (ez / one).abs()))[..., 0]
    out = dict(entropy=ent, b_entropy=b_ent, lp=lp, b_lp=b_lp)
    if y is not None:
        yy = y.long().cpu()
        at = yy.clamp(0, v - 1)[..., None]
        g = lp.gather(-1, at)[..., 0]
        g = torch.where(yy < 0, torch.zeros_like(g), torch.where(yy >= v, torch.full_like(g, math.nan), g))
        out.update(logprob=g, b_logprob=b_lp.gather(-1, at)[..., 0])
    if k:
        # NaN first, -0 = 0, equal values by lower index
        key = torch.where(x.isnan(), torch.full_like(x, INF), x + 0.0)
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices
        if bool(x.isnan().any()):
            nan_first = torch.sort(x.isnan().to(torch.int8).gather(-1, order), dim=-1, descending=True, stable=True).indices
            order = order.gather(-1, nan_first)
        order = order[..., :k]
        out.update(top_index=order, top_logprob=lp.gather(-1, order), b_top=b_lp.gather(-1, order))
    return out


def scores_backward(x, y, stat, entropy, d_lp, d_ent, temperature):
    """The gradient, and its bound before the result's rounding, from the statistics as handed in."""
    x = x.double().cpu()
    m, v = x.shape
    top, ln = stat.double().cpu()[:, :1], stat.double().cpu()[:, 1:]
    none = (top == -INF) & (ln == 0)
    z = torch.where(none, torch.full_like(x, -INF), (x - top) / temperature)
    lp = z - ln
    p = lp.exp()
    h = torch.zeros(m, 1, dtype=torch.float64) if entropy is None else entropy.double().cpu()[:, None]
    dl = torch.zeros(m, 1, dtype=torch.float64) if d_lp is None else d_lp.double().cpu()[:, None].clone()
    dh = torch.zeros(m, 1, dtype=torch.float64) if d_ent is None else d_ent.double().cpu()[:, None]
    if y is not None:
        yy = y.long().cpu()[:, None]
        dl = torch.where(yy < 0, torch.zeros_like(dl), torch.where(yy >= v, torch.full_like(dl, math.nan), dl))
    mix = torch.where(p > 0, p * (lp + h), torch.zeros_like(p))
    d = -dl * p - dh * mix
    a = (dl.abs() * p + dh.abs() * torch.where(p > 0, p * (lp.abs() + h.abs()), torch.zeros_like(p)))
    rel = 12 * U + 6 * U * torch.where(p > 0, z.abs() + ln.abs(), torch.zeros_like(p))
    b = a * rel + dh.abs() * p * rel
    if y is not None:
        hot = torch.zeros_like(x).scatter_(1, yy.clamp(0, v - 1), 1.0)
        d = d + torch.where(hot > 0, dl * (yy >= 0), torch.zeros_like(d))
        b = b + 3 * U * hot * dl.abs()
    d, b = d / temperature, b / temperature
    # exponentials below the normal range of fp32 may be flushed to zero
    flush = (dl.abs() + dh.abs() * (110.0 + h.abs())) * 2.0 ** -125 / temperature
    d = torch.where(none.expand_as(d), torch.zeros_like(d), d)
    return d, b + 4 * U * d.abs() + flush


def distill(x, ti, tv, y, temperature, w, u, scale):
    """(loss, its bound, gradient, its bound).  ``scale``: (rows,) factor of the gradient."""
    x = x.double().cpu()
    m, v = x.shape
    k = ti.shape[1]
    ti, tv = ti.long().cpu(), tv.double().cpu()
    wrong = (ti >= v).any(1) if w != 0 and k else torch.zeros(m, dtype=torch.bool)
    here = (ti >= 0) & (ti < v)
    at = ti.clamp(0, v - 1)
    t = torch.where(here, tv, torch.full_like(tv, -INF))
    tm = t.amax(1, keepdim=True) if k else torch.full((m, 1), -INF, dtype=torch.float64)
    taught = tm > -INF
    tz = torch.where(taught, (t - tm) / temperature, torch.full_like(t, -INF))
    es = tz.exp().sum(1, keepdim=True)
    q = torch.where(taught, tz.exp() / es, torch.zeros_like(t))
    log_q = tz - es.log()
    top, none, z, s, ez, rel = _exp_sum(x, 1.0 / temperature)
    _, _, z1, s1, ez1, rel1 = _exp_sum(x, 1.0)
    lp = torch.where(none, torch.full_like(z, -INF), z - s.log())
    lp1 = torch.where(none, torch.full_like(z1, -INF), z1 - s1.log())
    lpt = lp.gather(1, at)
    term = torch.where(q > 0, q * (log_q - lpt), torch.zeros_like(q))
    loss = w * temperature ** 2 * term.sum(1) if w != 0 else torch.zeros(m, dtype=torch.float64)
    relq = U * (2 * k + 24) + 6 * U * torch.where(q > 0, tz.abs(), torch.zeros_like(tz))
    one = torch.where(none, torch.ones_like(s), s)
    mag = torch.where(q > 0, q * ((log_q.abs() + lpt.abs()) * (relq + U * (2 * k + 24)) + relq + rel
                                  + 6 * U * (z.gather(1, at).abs() + one.log().abs() + tz.abs())), torch.zeros_like(q))
    b = abs(w) * temperature ** 2 * torch.nan_to_num(mag, posinf=0.0).sum(1)
    given = torch.zeros(m, dtype=torch.bool)
    if u != 0:
        yy = y.long().cpu()
        wrong = wrong | (yy >= v)
        given = (yy >= 0) & (yy < v)
        ya = yy.clamp(0, v - 1)[:, None]
        loss = loss - torch.where(given, u * lp1.gather(1, ya)[:, 0], torch.zeros_like(loss))
        b = b + abs(u) * torch.where(given, (rel1 + 6 * U * (z1.gather(1, ya).abs() + s1.log().abs()))[:, 0],
                                     torch.zeros_like(loss)).nan_to_num(posinf=0.0)
    b = b + 8 * U * loss.abs().nan_to_num(posinf=0.0) + 1e-37
    p, p1 = lp.exp(), lp1.exp()
    d, bd = torch.zeros_like(x), torch.zeros_like(x)
    if w != 0:
        target = torch.zeros_like(x).scatter_add_(1, at, torch.where(here, q, torch.zeros_like(q)))
        offq = torch.zeros_like(x).scatter_add_(1, at, torch.where(here, q * relq, torch.zeros_like(q)))
        d = torch.where(taught, w * temperature * (p - target), d)
        bd = torch.where(taught, abs(w) * temperature * (p * (rel + 6 * U * z.abs().nan_to_num(posinf=0) + 12 * U)
                                                         + offq + 8 * U * target), bd)
    if u != 0:
        hot = torch.zeros_like(x).scatter_(1, ya, 1.0)
        on = given[:, None].double()
        d = d + u * on * (p1 - hot)
        bd = bd + abs(u) * on * (p1 * (rel1 + 6 * U * z1.abs().nan_to_num(posinf=0) + 12 * U) + 8 * U * hot)
    d = torch.where(none, torch.zeros_like(d), d)
    sc = scale.double().cpu()[:, None]
    d = torch.where(wrong[:, None], torch.full_like(d, math.nan), d * sc)
    loss = torch.where(wrong, torch.full_like(loss, math.nan), loss)
    flush = 2.0 ** -125 * (abs(w) * temperature + abs(u)) * sc.abs()
    return loss, b, d, bd * sc.abs() + 8 * U * d.abs().nan_to_num() + flush + 0 * one


def check(got, want, bound, t, what):
    """|got - want| <= bound + half a step of the result's type; infinities and NaN in the same places."""
    got = got.double().cpu()
    over = want.isfinite() & (want.abs() > torch.finfo(t).max)       # beyond the type's range: infinite, or its last value
    fine = want.isfinite() & ~over
    assert bool((got[over].abs() >= torch.finfo(t).max).all()), f"{what}: overflow"
    assert bool(got[fine].isfinite().all()), f"{what}: finite values in other places"
    same = ~want.isfinite() & ~want.isnan()
    assert torch.equal(got[same], want[same]), f"{what}: infinities"
    assert bool(got[want.isnan()].isnan().all()), f"{what}: NaN"
    if not bool(fine.any()):
        return
    bound = bound.expand_as(want)[fine] if isinstance(bound, torch.Tensor) else bound
    room = bound + half(t) * (want[fine].abs() + bound) + tiny(t)
    over = (got[fine] - want[fine]).abs() / room
    assert float(over.max()) <= 1.0, f"{what}: {float(over.max()):.3g} of the bound at {int(over.argmax())}"
