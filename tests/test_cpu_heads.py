"""CPU: what the classifier-head entry points refuse, at the tensor level (wfd_gan_amd.heads) and at the C ABI, before anything
reaches a GPU."""
import pytest
import torch

from wfd_gan_amd import heads
from wfd_gan_amd._lib import WfdError, lib

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
X = torch.zeros(4, 10)
Y = torch.zeros(4, dtype=torch.int32)
TI, TV = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)


def test_there_is_no_cpu_path():
    m = torch.zeros(4)
    for call in (lambda: heads.layer_norm(X), lambda: heads.layer_norm_backward(X, X, None, m, m),
                 lambda: heads.label_logprobs(X, Y, 2),
                 lambda: heads.label_logprobs_backward(X, Y, heads.LabelScores(None, m, torch.zeros(4, 2), None, None, None), m),
                 lambda: heads.distill_loss(X, TI, TV)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("bad", [torch.zeros(4, 10, dtype=torch.float64), torch.zeros(4, 10, dtype=torch.int32)])
def test_row_types(bad):
    m = torch.zeros(4)
    for call in (lambda: heads.layer_norm(bad), lambda: heads.layer_norm_backward(bad, bad, None, m, m),
                 lambda: heads.label_logprobs(bad, Y), lambda: heads.distill_loss(bad, TI, TV)):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            call()
    with pytest.raises(TypeError, match="expected a tensor"):
        heads.layer_norm([1.0])


@pytest.mark.parametrize("bad", [torch.zeros(()), torch.zeros(4, 0)])
def test_rows_need_an_element(bad):
    for call in (lambda: heads.layer_norm(bad), lambda: heads.label_logprobs(bad, Y), lambda: heads.distill_loss(bad, TI, TV)):
        with pytest.raises(ValueError, match="at least one element"):
            call()


def test_layer_norm_refusals():
    m = torch.zeros(4)
    with pytest.raises(ValueError, match="weight has 9"):
        heads.layer_norm(X, torch.ones(9))
    with pytest.raises(TypeError, match="one dtype"):
        heads.layer_norm(X, torch.ones(10), torch.ones(10, dtype=BF16))
    with pytest.raises(TypeError, match="float32 or have the rows' dtype"):
        heads.layer_norm(X, torch.ones(10, dtype=BF16))
    with pytest.raises(TypeError, match="float32 or have the rows' dtype"):
        heads.layer_norm(X.to(BF16), torch.ones(10, dtype=F16))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            heads.layer_norm(X, eps=eps)
    with pytest.raises(ValueError, match="does not match"):
        heads.layer_norm_backward(X[:3], X, None, m, m)
    with pytest.raises(ValueError, match="does not match"):
        heads.layer_norm_backward(X.to(BF16), X, None, m, m)
    with pytest.raises(ValueError, match="mean has 3"):
        heads.layer_norm_backward(X, X, None, m[:3], m)
    with pytest.raises(TypeError, match="rstd must be"):
        heads.layer_norm_backward(X, X, None, m, m.double())
    with pytest.raises(ValueError, match="needs the mean and rstd"):
        heads.layer_norm_backward(X, X, None, None, None)


def test_label_logprobs_refusals():
    for k in (-1, 11, 65):
        with pytest.raises(ValueError, match="k must be"):
            heads.label_logprobs(X, Y, k)
    with pytest.raises(ValueError, match="0 .. 64"):
        heads.label_logprobs(torch.zeros(4, 100), Y, 65)
    with pytest.raises(TypeError, match="labels must be"):
        heads.label_logprobs(X, Y.long())
    with pytest.raises(ValueError, match="labels has 3"):
        heads.label_logprobs(X, Y[:3])
    for t in (0.0, -1.0, 9e-7, 2e6, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            heads.label_logprobs(X, Y, temperature=t)
    m, stat = torch.zeros(4), torch.zeros(4, 2)
    full = heads.LabelScores(m, m, stat, None, None, None)
    with pytest.raises(ValueError, match="lacks"):
        heads.label_logprobs_backward(X, Y, full._replace(stat=None), m)
    with pytest.raises(ValueError, match="lacks"):
        heads.label_logprobs_backward(X, Y, full._replace(entropy=None), m, m)
    with pytest.raises(ValueError, match="needs the labels"):
        heads.label_logprobs_backward(X, None, full, m)
    with pytest.raises(ValueError, match="scores.stat has 4"):
        heads.label_logprobs_backward(X, Y, full._replace(stat=m), m)
    with pytest.raises(ValueError, match="d_entropy has 3"):
        heads.label_logprobs_backward(X, Y, full, m, m[:3])


def test_distill_refusals():
    with pytest.raises(TypeError, match="teacher_index must be"):
        heads.distill_loss(X, TI.long(), TV)
    with pytest.raises(TypeError, match="teacher_value must be"):
        heads.distill_loss(X, TI, TV.to(BF16))
    with pytest.raises(ValueError, match="go with"):
        heads.distill_loss(X, TI[:3], TV[:3])
    with pytest.raises(ValueError, match="go with"):
        heads.distill_loss(X, TI, TV[:, :2])
    with pytest.raises(ValueError, match="at most 256"):
        heads.distill_loss(X, torch.zeros(4, 257, dtype=torch.int32), torch.zeros(4, 257))
    with pytest.raises(ValueError, match="label_weight needs labels"):
        heads.distill_loss(X, TI, TV, label_weight=0.5)
    with pytest.raises(ValueError, match="must be finite"):
        heads.distill_loss(X, TI, TV, weight=float("nan"))
    with pytest.raises(ValueError, match="temperature"):
        heads.distill_loss(X, TI, TV, temperature=0.0)
    with pytest.raises(ValueError, match="row_scale has 3"):
        heads.distill_loss(X, TI, TV, row_scale=torch.ones(3))


def test_abi_refusals_and_empty_calls():
    """Codes of the C entry points; the addresses are never followed."""
    L = lib()
    P = 4096                                                   # stands for an aligned device address

    def refused(fn, *a):
        with pytest.raises(WfdError, match="bad argument"):
            fn(*a)
    fwd = lambda **o: [o.get(k, d) for k, d in dict(X=P, ldx=8, dt=1, w=P, b=P, wt=0, M=2, N=8, eps=1e-5, Y=P, ldy=8, mean=P,
                                                    rstd=P, st=0).items()]
    for o in (dict(X=0), dict(Y=0), dict(ldx=7), dict(ldy=7), dict(dt=3), dict(dt=-1), dict(wt=2), dict(M=-1), dict(N=0),
              dict(N=(1 << 24) + 1), dict(X=P + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(dt=0, Y=P + 2), dict(ldy=9)):
        refused(L.layer_norm_fwd, *fwd(**o))
    L.layer_norm_fwd(*fwd(M=0, X=0, Y=0))
    bwd = lambda **o: [o.get(k, d) for k, d in dict(DY=P, lddy=8, X=P, ldx=8, dt=1, w=P, wt=0, mean=P, rstd=P, M=2, N=8, DX=P,
                                                    lddx=8, dw=P, db=P, work=P, st=0).items()]
    for o in (dict(DY=0), dict(X=0), dict(DX=0), dict(mean=0), dict(rstd=0), dict(work=0), dict(lddy=7), dict(lddx=7), dict(wt=2),
              dict(N=0), dict(M=-2), dict(dt=5), dict(lddx=9)):
        refused(L.layer_norm_bwd, *bwd(**o))
    sc = lambda **o: [o.get(k, d) for k, d in dict(x=P, ld=9, dt=1, M=2, V=9, y=P, T=1.0, k=3, lp=P, e=P, s=P, tl=P, ti=P, work=P,
                                                   st=0).items()]
    for o in (dict(x=0), dict(ld=8), dict(dt=3), dict(V=0), dict(k=10), dict(k=65, V=100, ld=100), dict(k=-1), dict(T=0.0),
              dict(T=float("inf")), dict(T=float("nan")), dict(tl=0), dict(ti=0), dict(y=0), dict(M=-1), dict(x=P + 1),
              dict(V=(1 << 23) + 1, ld=(1 << 23) + 1)):
        refused(L.label_scores, *sc(**o))
    L.label_scores(*sc(M=0, x=0))
    sb = lambda **o: [o.get(k, d) for k, d in dict(x=P, ld=9, dt=1, M=2, V=9, y=P, T=1.0, s=P, e=P, dl=P, dh=P, dx=P, lddx=9,
                                                   st=0).items()]
    for o in (dict(x=0), dict(dx=0), dict(s=0), dict(e=0), dict(y=0), dict(ld=8), dict(lddx=8), dict(T=-1.0), dict(V=0), dict(lddx=10)):
        refused(L.label_scores_bwd, *sb(**o))
    L.label_scores_bwd(*sb(M=0, x=0, dx=0, s=0))
    ds = lambda **o: [o.get(k, d) for k, d in dict(x=P, ld=9, dt=1, M=2, V=9, ti=P, tv=P, ldt=4, K=4, y=P, T=1.0, w=1.0, u=0.5, rs=0,
                                                   gs=1.0, loss=P, dx=P, lddx=9, work=P, st=0).items()]
    for o in (dict(x=0), dict(loss=0), dict(ti=0), dict(tv=0), dict(ldt=3), dict(K=257, ldt=300), dict(K=-1), dict(y=0), dict(T=0.0),
              dict(w=float("inf")), dict(u=float("nan")), dict(lddx=8), dict(ld=8), dict(dt=3), dict(V=0), dict(lddx=10), dict(T=1e-7)):
        refused(L.distill, *ds(**o))
    L.distill(*ds(M=0, x=0, loss=0))


def test_more_threads_than_a_launch_counts():
    """A launch counts its threads in 32 bits; calls that would need more are refused, not cut off."""
    L = lib()
    P, M = 4096, (1 << 31) - 1
    calls = ((L.label_scores, lambda m, v: (P, v, 1, m, v, P, 1.0, 1, P, P, P, P, P, P, 0), (9, 4000, 20000)),
             (L.label_scores_bwd, lambda m, v: (P, v, 1, m, v, P, 1.0, P, P, P, P, P, v, 0), (9, 4000, 20000)),
             (L.distill, lambda m, v: (P, v, 1, m, v, P, P, 4, 4, P, 1.0, 1.0, 0.5, 0, 1.0, P, P, v, P, 0), (9, 300, 200000)),
             (L.layer_norm_fwd, lambda m, n: (P, n, 1, P, P, 0, m, n, 1e-5, P, n, P, P, 0), (200000,)))
    for fn, args, sizes in calls:
        for v in sizes:
            with pytest.raises(WfdError, match="bad argument"):
                fn(*args(M, v))


def test_scratch_sizes():
    L = lib()
    for m, n in ((0, 5), (1, 1), (4096, 1024), (100000, 100), (3, 1 << 20)):
        for dt in (0, 1, 2):
            assert L.layer_norm_bwd_floats(m, n, dt) >= 2 * n
            assert L.distill_floats(m, n, dt) >= 0
            for k in (0, 1, min(n, 64)):
                assert L.label_scores_floats(m, n, dt, k) >= 0
    assert L.layer_norm_bwd_floats(4096, 1 << 24, 0) == 1 << 30 and L.layer_norm_bwd_floats(4096, (1 << 24) + 1, 0) < 0
    assert L.layer_norm_bwd_floats(4, 0, 0) < 0 and L.layer_norm_bwd_floats(4, 8, 7) < 0
    assert L.label_scores_floats(4, 8, 0, 9) < 0 and L.distill_floats(-1, 8, 0) < 0


def test_train_df_flags():
    from wfd_gan_amd import train_df
    ns = train_df.parse_args(["X.npz"])
    assert ns.teacher is None and ns.top_k == 0
    ns = train_df.parse_args(["X.npz", "--teacher", "t.ckpt", "--teacher_k", "5", "--teacher_weight", "0.5", "--temperature", "3"])
    assert (ns.teacher, ns.teacher_k, ns.teacher_weight, ns.temperature) == ("t.ckpt", 5, 0.5, 3.0)
    for bad in (["--teacher_weight", "1.5"], ["--temperature", "0"], ["--teacher_k", "0"], ["--teacher_k", "65"], ["--top_k", "-1"]):
        with pytest.raises(SystemExit):
            train_df.parse_args(["X.npz"] + bad)
