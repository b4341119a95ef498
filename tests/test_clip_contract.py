"""clip_grad_norm_ takes what torch.nn.utils.clip_grad_norm_ takes, by place and by name; other norms are refused."""
import inspect
import math

import pytest
import torch


@pytest.fixture
def formulas(monkeypatch):
    """The kernels replaced by their formulas in torch, so that CPU tensors will do."""
    from fp8_gmm_b200 import backend

    def squares(grads):
        return sum((g.double().square().sum() for g in grads), torch.zeros((), dtype=torch.float64))

    def clip(grads, sum_squares, max_norm, outputs=None):
        for g in grads:
            g.mul_(torch.clamp(max_norm / (sum_squares.sqrt() + 1e-6), max=1.0).to(g.dtype))
        return sum_squares.sqrt().float()

    monkeypatch.setattr(backend, "multi_sum_squares", squares)
    monkeypatch.setattr(backend, "multi_clip", clip)
    monkeypatch.setattr(backend, "multi_clip_grad_norm", lambda grads, max_norm, outputs=None: clip(grads, squares(grads), max_norm))


def _params(values=((3.0, 0.0), (0.0, 4.0))):
    ps = [torch.nn.Parameter(torch.zeros(len(v))) for v in values]
    for p, v in zip(ps, values):
        p.grad = torch.tensor(v)
    return ps


def test_arguments_stand_where_torchs_stand():
    import fp8_gmm_b200 as fg

    ours, theirs = (list(inspect.signature(f).parameters.values()) for f in (fg.clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
    for a, b in zip(ours, theirs):
        assert (a.name, a.kind, a.default) == (b.name, b.kind, b.default)
    assert len(ours) > len(theirs) and all(a.kind is a.KEYWORD_ONLY for a in ours[len(theirs):])


@pytest.mark.parametrize("args,kw", [((1.0,), {}), ((1.0, 2.0), {}), ((1.0, 2), {}), ((1.0,), dict(norm_type=2.0)), ((1.0, 2.0, True), {}),
                                     ((1.0, 2.0, False, True), {}), ((1.0,), dict(norm_type=2, error_if_nonfinite=True, foreach=False))])
def test_the_2_norm_in_every_spelling(formulas, args, kw):
    import fp8_gmm_b200 as fg

    ours, theirs = _params(), _params()
    got, want = fg.clip_grad_norm_(ours, *args, **kw), torch.nn.utils.clip_grad_norm_(theirs, *args, **kw)
    assert float(got) == float(want) == 5.0
    assert all(torch.allclose(a.grad, b.grad, rtol=2.0 ** -22, atol=0) for a, b in zip(ours, theirs))


@pytest.mark.parametrize("norm_type", [1.0, float("inf"), 0, 3, "inf", True, float("nan")])
def test_other_norms_are_refused(formulas, norm_type):
    import fp8_gmm_b200 as fg

    for call in (lambda p: fg.clip_grad_norm_(p, 1.0, norm_type), lambda p: fg.clip_grad_norm_(p, 1.0, norm_type=norm_type)):
        ps = _params()
        with pytest.raises(RuntimeError, match="norm_type"):
            call(ps)
        assert ps[0].grad.tolist() == [3.0, 0.0]


@pytest.mark.parametrize("values", [((math.inf, 0.0), (1.0, 1.0)), ((math.nan, 0.0), (1.0, 1.0)), ((3e38, 3e38), (3e38, 1.0))])
def test_a_norm_that_is_not_finite_raises_if_asked_for(formulas, values):
    """Also one whose square is finite in 64 bits and that is itself outside fp32: the norm that would be returned is inf."""
    import fp8_gmm_b200 as fg

    ps = _params(values)
    with pytest.raises(RuntimeError, match="left as they are"):
        fg.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(p.grad, torch.tensor(v)) or math.isnan(v[0]) for p, v in zip(ps, values))


@pytest.mark.gpu
def test_a_gradient_listed_twice_is_refused(cuda):
    import fp8_gmm_b200 as fg

    p = torch.nn.Parameter(torch.zeros(4, device=cuda))
    p.grad = torch.full((4,), 2.0, device=cuda)
    with pytest.raises(RuntimeError, match="share memory"):
        fg.clip_grad_norm_([p, p], 1.0)
    assert (p.grad == 2.0).all()
    assert float(fg.clip_grad_norm_([p], 1.0, 2.0, True)) == 4.0 and torch.allclose(p.grad, torch.full_like(p.grad, 0.5))
