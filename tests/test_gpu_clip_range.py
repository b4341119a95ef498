"""GPU: clipping where the factor itself is below fp32's normal numbers, though the clipped elements are not.

A factor of 2^-126 and more is rounded to fp32 and so is the product (2^-24 each), then the output's type (half a step); a smaller
factor is multiplied in 64 bits, and the product rounded once to fp32 and once to the output's type: the first bound holds for both.
The norm's relative error, below 2^-22, moves the factor by as much."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _check(outs, before, factor):
    for o, g in zip(outs, before):
        want = g.double() * factor
        tiny = {BF: 2.0 ** -134, HF: 2.0 ** -25, F32: 2.0 ** -150}[o.dtype]      # half the smallest subnormal
        bound = want.abs() * (torch.finfo(o.dtype).eps / 2 + 2 * 2.0 ** -24 + 2.0 ** -22) + tiny + 2.0 ** -149
        assert ((o.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("value,dtype,max_norm", [(3e38, F32, 1.0), (1e38, BF, 1.0), (1e38, BF, 1e-3), (3e38, F32, 1e-7), (1e25, BF, 1e-20),
                                                  (1e25, BF, 1.0), (3e38, BF, 1e4), (6e4, HF, 1e-38), (6e4, HF, 1e-33)])
def test_clipped_elements_of_large_gradients(cuda, value, dtype, max_norm):
    from fp8_gmm_b200 import backend

    g = torch.Generator().manual_seed(1)
    grads = [((torch.rand(n, generator=g) - 0.5) * 2 * value).to(dtype).to(cuda) for n in (5000, 70001, 3)]
    grads.append(grads[0][:1].clone().float() * 1e-3)
    before = [x.clone() for x in grads]
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    factor = max_norm / (norm + 1e-6)
    for out_type in (F32, BF, HF):
        outs = [torch.full(x.shape, float("nan"), dtype=out_type, device=cuda) for x in grads]
        backend.multi_clip_grad_norm(grads, max_norm, outputs=outs)
        _check(outs, before, factor)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    squares = backend.multi_sum_squares(grads)
    backend.multi_clip(grads, squares, max_norm)                 # in place, the norm from elsewhere
    _check(grads, before, factor)


def test_every_offset_and_the_elements_beside(cuda):
    """Tiles that start inside a vector: each element once, none beside the tensor."""
    from fp8_gmm_b200 import backend

    buf = ((torch.rand(20000, generator=torch.Generator().manual_seed(2)) - 0.5) * 2 * 3e38).to(BF).to(cuda)
    for first in range(9):
        work = buf.clone()
        view = work[first:first + 8200]
        before = view.clone()
        backend.multi_clip([view], torch.tensor(1e82, dtype=torch.float64, device=cuda), 1.0)
        _check([view], [before], 1.0 / (1e41 + 1e-6))
        assert torch.equal(work[:first], buf[:first]) and torch.equal(work[first + 8200:], buf[first + 8200:])


def test_zero_and_special_elements_with_a_small_factor(cuda):
    from fp8_gmm_b200 import backend

    g = torch.tensor([0.0, -0.0, 1e38, float("inf"), -float("inf"), float("nan")], device=cuda)
    backend.multi_clip([g], torch.tensor(1e82, dtype=torch.float64, device=cuda), 1.0)
    assert g[:2].tolist() == [0.0, 0.0] and abs(float(g[2]) - 1e-3) < 1e-9
    assert float(g[3]) == math.inf and float(g[4]) == -math.inf and math.isnan(float(g[5]))
