"""What a classifier's head does around its last product, as cases to measure: layer norm (forward, backward), the scores of
given labels over many classes (log probability, entropy, top alternatives; and their gradient), and the loss of a student that
learns from a teacher's top logits (with its gradient).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes the inputs, ``run`` is one pass:
in plain torch operations where ``own`` is false, through ``wfd_gan_amd.heads`` where it is true.  ``exact`` is the same
outputs from the definitions in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one answer's features on their way into the head: latency of a single row
        dict(name="norm_one_row", op="norm", back=False, rows=1, n=2048, t="bf16", wt="f32"),
        # a large batch of the generator's widest hidden layer
        dict(name="norm_hidden", op="norm", back=False, rows=4096, n=2048, t="f32", wt="f32"),
        # trace rows of 1401 values: an odd width, rows that begin off every 16-byte border
        dict(name="norm_traces_odd", op="norm", back=False, rows=8191, n=1401, t="bf16", wt="f32"),
        # backward of a training batch in mixed precision: 16-bit activations, 32-bit weights
        dict(name="norm_back_hidden", op="norm", back=True, rows=4096, n=1024, t="bf16", wt="f32"),
        # backward over many rows with everything in 16 bits
        dict(name="norm_back_large", op="norm", back=True, rows=16384, n=4096, t="bf16", wt="bf16"),
        # one answer over a large vocabulary, with the alternatives that an interface shows
        dict(name="score_one_answer", op="score", back=False, rows=1, classes=131072, k=20, t="bf16", temp=0.7, mask=0.0),
        # the observer's accuracy pass: batches of 2048 traces, 100 sites
        dict(name="score_observer", op="score", back=False, rows=2048, classes=100, k=5, t="f32", temp=1.0, mask=0.0),
        # scoring a corpus: odd class count, so each row begins elsewhere between two 16-byte borders
        dict(name="score_corpus_odd", op="score", back=False, rows=4096, classes=50257, k=10, t="bf16", temp=1.0, mask=0.0),
        # policy-style update: gradients of log probability and entropy together
        dict(name="score_back", op="score", back=True, rows=4096, classes=32000, k=0, t="bf16", temp=1.0, mask=0.0),
        # a step of the observer's training from a larger one: batch 128, 100 sites, labels mixed in
        dict(name="distill_observer", op="distill", back=True, rows=128, classes=100, k=8, t="f32", temp=2.0, labels=0.5),
        # loss alone on a held-out batch
        dict(name="distill_held_out", op="distill", back=False, rows=61, classes=32000, k=16, t="f16", temp=1.0, labels=0.0),
        # training from stored top logits over a large vocabulary
        dict(name="distill_large", op="distill", back=True, rows=2048, classes=128000, k=64, t="bf16", temp=1.0, labels=0.0),
    ]


def _between(rng, a, b):
    """A whole number of [a, b], spread over its logarithm."""
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 0.49)))))))


def draw(rng):
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    op = rng.choice(["norm", "score", "distill"])
    limit = 400_000_000 // SIZE[t]                          # elements of one operand: below the largest listed case
    if op == "norm":
        n = _between(rng, 1, 16384)
        rows = _between(rng, 1, min(32768, max(1, 100_000_000 // n)))
        return dict(op=op, back=rng.random() < 0.5, rows=rows, n=n, t=t, wt=rng.choice([t, "f32"]))
    classes = _between(rng, 2, 200_000)
    rows = _between(rng, 1, min(16384, max(1, limit // classes)))
    back = rng.random() < 0.5
    temp = rng.choice([0.5, 0.7, 1.0, 1.0, 2.0, 3.0])
    if op == "score":
        k = 0 if back else min(classes, rng.choice([0, 1, 5, 20, 64]))
        return dict(op=op, back=back, rows=rows, classes=classes, k=k, t=t, temp=temp, mask=rng.choice([0.0, 0.0, 0.5, 0.95]))
    return dict(op=op, back=back, rows=rows, classes=classes, k=_between(rng, 1, min(64, classes)), t=t, temp=temp,
                labels=rng.choice([0.0, 0.0, 0.3, 0.5]))


def work(case):
    m, e = case["rows"], SIZE[case["t"]]
    if case["op"] == "norm":
        n, w = case["n"], SIZE[case["wt"]]
        if case["back"]:
            return {"bytes": 3 * m * n * e + 8 * m + 3 * n * w, "flops": 14 * m * n}
        return {"bytes": 2 * m * n * e + 8 * m + 2 * n * w, "flops": 8 * m * n}
    c = case["classes"]
    if case["op"] == "score":
        if case["back"]:
            return {"bytes": 2 * m * c * e + 24 * m, "flops": 8 * m * c}
        return {"bytes": m * c * e + m * (20 + 8 * case["k"]), "flops": 6 * m * c}
    rows = m * c * e * (2 if case["back"] else 1)
    return {"bytes": rows + m * (12 + 8 * case["k"]), "flops": (8 if case["back"] else 4) * m * c}


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1_000_003 + 17)
    t, m = TYPES[case["t"]], case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case=dict(case))
    if case["op"] == "norm":
        n, wt = case["n"], TYPES[case["wt"]]
        # features have a spread and an offset of their own
        s["x"] = (normal(m, n) * 1.5 + normal(n)).to(t)
        s["w"] = (1 + 0.2 * normal(n)).to(wt)
        s["b"] = (0.2 * normal(n)).to(wt)
        s["eps"] = 1e-5
        if case["back"]:
            s["dy"] = normal(m, n).to(t)
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + s["eps"])
        if own:
            from wfd_gan_amd import heads
            s["out"] = heads.norm_gradients_like(s["x"], s["w"], s["b"]) if case["back"] else heads.norm_output_like(s["x"])
        return s
    c = case["classes"]
    labels = torch.randint(0, c, (m,), generator=g, device=DEV, dtype=torch.int32)
    logits = normal(m, c) * 2.0
    # a trained head is sure of the label more often than not
    logits.scatter_add_(1, labels.long()[:, None], 8.0 * torch.rand(m, 1, generator=g, device=DEV))
    if m > 8:
        labels[:: 16] = -1                                  # padding rows carry no label
    s["labels"] = labels
    if case["op"] == "score":
        if case["mask"]:
            # answers that are held to some of the classes; a few rows are left with none
            gone = torch.rand(m, c, generator=g, device=DEV) < case["mask"]
            gone[3::97] = True
            logits.masked_fill_(gone, -math.inf)
        s["logits"] = logits.to(t)
        if case["back"]:
            s["stat"], s["entropy"] = _statistics(s["logits"], case["temp"])
            s["d_logprob"], s["d_entropy"] = normal(m), 0.01 * normal(m)
        if own:
            from wfd_gan_amd import heads
            if case["back"]:
                s["scores"] = heads.LabelScores(None, s["entropy"], s["stat"], None, None, None)
                s["out"] = torch.empty_like(s["logits"])
            else:
                s["out"] = heads.scores_like(s["logits"], case["k"])
        return s
    s["logits"] = logits.to(t)
    k = case["k"]
    # the teacher: its own view of the same row, of which the k largest are kept, some rows with fewer
    teacher = logits + normal(m, c)
    s["t_value"], at = teacher.topk(k, dim=1)
    s["t_index"] = at.to(torch.int32)
    if m > 8 and k > 1:
        s["t_index"][5::32, k // 2:] = -1
    s["row_scale"] = (labels >= 0).float()
    s["scale"] = 1.0 if t == torch.float16 else 1.0 / m     # 16-bit floats of the narrow range train with a scaled loss
    if own:
        from wfd_gan_amd import heads
        s["out"] = heads.distill_output_like(s["logits"], grad=case["back"])
    return s


def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from wfd_gan_amd import heads
    case = s["case"]
    if case["op"] == "norm":
        if case["back"]:
            r = heads.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], out=s["out"])
            return r.dx, r.dweight, r.dbias
        r = heads.layer_norm(s["x"], s["w"], s["b"], s["eps"], out=s["out"])
        return r.y, r.mean, r.rstd
    if case["op"] == "score":
        if case["back"]:
            return heads.label_logprobs_backward(s["logits"], s["labels"], s["scores"], s["d_logprob"], s["d_entropy"],
                                                 temperature=case["temp"], out=s["out"])
        r = heads.label_logprobs(s["logits"], s["labels"], case["k"], temperature=case["temp"], out=s["out"])
        return (r.logprob, r.entropy, r.top_logprob, r.top_index) if case["k"] else (r.logprob, r.entropy)
    ce = case["labels"]
    r = heads.distill_loss(s["logits"], s["t_index"], s["t_value"], s["labels"] if ce else None, temperature=case["temp"],
                           weight=1.0 - ce, label_weight=ce, row_scale=s["row_scale"], grad_scale=s["scale"], grad=case["back"],
                           out=s["out"])
    return (r.loss, r.dlogits) if case["back"] else r.loss


def _statistics(logits, temp):
    """([row maximum, log of the sum of exp((x - maximum) / temp)], entropy), 32 bits; a row of nothing but -inf has
    -inf, 0 and entropy 0."""
    x = logits.float()
    top = x.amax(1, keepdim=True)
    none = top == -math.inf
    z = torch.where(none, torch.full_like(x, -math.inf), (x - top) / temp)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log = torch.where(none, torch.zeros_like(total), total.log())
    share = e / torch.where(none, torch.ones_like(total), total)
    entropy = -torch.where(share > 0, share * (z - log), torch.zeros_like(z)).sum(1)
    return torch.cat([top, log], 1), entropy


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        x, w = s["x"].float(), s["w"].float()
        if case["back"]:
            dy, n = s["dy"].float(), x.shape[1]
            unit = (x - s["mean"][:, None]) * s["rstd"][:, None]
            v = dy * w
            dx = s["rstd"][:, None] * (v - v.sum(1, keepdim=True) / n - unit * ((v * unit).sum(1, keepdim=True) / n))
            return dx.to(s["x"].dtype), (dy * unit).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)
        mean = x.sum(1) / x.shape[1]
        d = x - mean[:, None]
        rstd = 1.0 / ((d * d).sum(1) / x.shape[1] + s["eps"]).sqrt()
        return (d * rstd[:, None] * w + s["b"].float()).to(s["x"].dtype), mean, rstd
    logits, temp = s["logits"], case["temp"]
    x, labels = logits.float(), s["labels"].long()
    m, c = x.shape
    given = labels >= 0
    at = labels.clamp(min=0)[:, None]
    if case["op"] == "score":
        if case["back"]:
            top, log = s["stat"][:, :1], s["stat"][:, 1:]
            none = top == -math.inf
            lp = torch.where(none, torch.full_like(x, -math.inf), (x - top) / temp - log)
            p = lp.exp()
            dl = torch.where(given, s["d_logprob"], torch.zeros_like(s["d_logprob"]))[:, None]
            down = torch.where(p > 0, p * (lp + s["entropy"][:, None]), torch.zeros_like(p))
            d = -dl * p - s["d_entropy"][:, None] * down
            d.scatter_add_(1, at, torch.where(none, torch.zeros_like(dl), dl))
            return (d / temp).to(logits.dtype)
        stat, entropy = _statistics(logits, temp)
        top, log = stat[:, :1], stat[:, 1:]
        none = top == -math.inf

        def logprob(v):
            return torch.where(none, torch.full_like(v, -math.inf), (v - top) / temp - log)

        lp = torch.where(given, logprob(x.gather(1, at))[:, 0], torch.zeros_like(entropy))
        if not case["k"]:
            return lp, entropy
        # order of (value, lowest index first): whole numbers that rise with the value, the index below them
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        del bits
        key = key.mul_(1 << 32).add_(c - 1 - torch.arange(c, device=x.device))
        best = key.topk(case["k"], dim=1).values
        idx = c - 1 - (best & 0xFFFFFFFF)
        return lp, entropy, logprob(x.gather(1, idx)), idx.to(torch.int32)
    ce = case["labels"]

    def log_softmax(scale):
        z = x * scale
        z = z - z.amax(1, keepdim=True)
        return z - z.exp().sum(1, keepdim=True).log()

    here = s["t_index"] >= 0
    idx = s["t_index"].long().clamp(min=0)
    tv = torch.where(here, s["t_value"], torch.full_like(s["t_value"], -math.inf)) / temp
    tv = tv - tv.amax(1, keepdim=True)
    q = tv.exp()
    total = q.sum(1, keepdim=True)
    log_q = tv - total.log()
    q = q / total
    lp = log_softmax(1.0 / temp)
    loss = (1.0 - ce) * temp * temp * torch.where(here, q * (log_q - lp.gather(1, idx)), torch.zeros_like(q)).sum(1)
    d = None
    if case["back"]:
        d = lp.exp()
        d.scatter_add_(1, idx, -q)
        d *= (1.0 - ce) * temp
    if ce:
        lp = log_softmax(1.0)
        loss = loss - ce * torch.where(given, lp.gather(1, at)[:, 0], torch.zeros_like(loss))
        if d is not None:
            hot = torch.zeros_like(lp).scatter_(1, at, 1.0)
            d = d + ce * given.float()[:, None] * (lp.exp() - hot)
    if d is None:
        return loss
    return loss, (d * (s["row_scale"] * s["scale"])[:, None]).to(logits.dtype)


def _blocks(m, c):
    """Rows at a time that keep a block of 64-bit values near 256 MB."""
    step = max(1, 32_000_000 // c)
    return [slice(a, min(m, a + step)) for a in range(0, m, step)]


def exact(case, seed):
    s = prepare(case, seed)
    D = torch.float64
    if case["op"] == "norm":
        w, b, n = s["w"].to(D), s["b"].to(D), case["n"]
        parts, dw, db = [], torch.zeros(n, dtype=D, device=DEV), torch.zeros(n, dtype=D, device=DEV)
        for r in _blocks(case["rows"], n):
            x = s["x"][r].to(D)
            if case["back"]:
                mean, rstd = s["mean"][r].to(D).unsqueeze(1), s["rstd"][r].to(D).unsqueeze(1)
                dy, xh = s["dy"][r].to(D), (x - mean) * rstd
                parts.append(rstd * (dy * w - (dy * w).mean(1, keepdim=True) - xh * (dy * w * xh).mean(1, keepdim=True)))
                dw += torch.einsum("mn,mn->n", dy, xh)
                db += dy.sum(0)
            else:
                var, mean = torch.var_mean(x, dim=1, unbiased=False)
                rstd = (var + s["eps"]).pow(-0.5)
                parts.append(((x - mean[:, None]) * rstd[:, None] * w + b, mean, rstd))
        if case["back"]:
            return torch.cat(parts), dw, db
        return tuple(torch.cat(p) for p in zip(*parts))
    temp, c, k = case["temp"], case["classes"], case["k"]
    parts = []
    for r in _blocks(case["rows"], c):
        x, y = s["logits"][r].to(D), s["labels"][r].long()
        row = torch.arange(x.shape[0], device=DEV)
        lse = torch.logsumexp(x / temp, 1)
        empty = torch.isinf(lse) & (lse < 0)
        lp = torch.where(empty[:, None], -math.inf, x / temp - lse[:, None])
        p = lp.exp()
        if case["op"] == "score":
            ent = -torch.nan_to_num(p * lp, nan=0.0).sum(1)
            if case["back"]:
                # the statistics are inputs here: entropy as it was handed in
                dl = torch.where(y >= 0, s["d_logprob"][r].to(D), 0.0)
                dh = s["d_entropy"][r].to(D)
                d = -dl[:, None] * p - dh[:, None] * torch.nan_to_num(p * (lp + s["entropy"][r].to(D)[:, None]), nan=0.0)
                d[row, y.clamp(min=0)] += dl * (~empty)
                parts.append((d / temp,))
                continue
            got = torch.where(y >= 0, lp[row, y.clamp(min=0)], 0.0)
            if not k:
                parts.append((got, ent))
                continue
            value, idx = torch.sort(x, dim=1, descending=True, stable=True)
            parts.append((got, ent, lp.gather(1, idx[:, :k]), idx[:, :k].to(torch.int32)))
            continue
        ti, tv, ce = s["t_index"][r].long(), s["t_value"][r].to(D), case["labels"]
        tv = torch.where(ti < 0, -math.inf, tv) / temp
        log_q = tv - torch.logsumexp(tv, 1, keepdim=True)
        q = log_q.exp()
        pair = torch.where(ti < 0, 0.0, q * (log_q - lp.gather(1, ti.clamp(min=0))))
        loss = (1 - ce) * temp ** 2 * pair.sum(1)
        lp1 = torch.log_softmax(x, 1)
        loss -= ce * torch.where(y >= 0, lp1[row, y.clamp(min=0)], 0.0)
        if not case["back"]:
            parts.append((loss,))
            continue
        target = torch.zeros_like(p).scatter_add_(1, ti.clamp(min=0), torch.where(ti < 0, 0.0, q))
        d = (1 - ce) * temp * (p - target)
        hot = torch.zeros_like(p)
        hot[row, y.clamp(min=0)] = 1.0
        d += ce * (y >= 0).to(D)[:, None] * (lp1.exp() - hot)
        parts.append((loss, d * (s["row_scale"][r].to(D) * s["scale"])[:, None]))
    out = tuple(torch.cat(p) for p in zip(*parts))
    return out[0] if len(out) == 1 else out
