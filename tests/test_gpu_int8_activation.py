"""GPU: codes and scales of rows behind an activation, at the borders between two codes and over all bf16 arguments.

v = a / (1 + e), e = 2^p, is computed as in the kernel's comment.  In units of 2^-24: exp2 is off by up to 4 (its documented
2^-22).  Behind SiLU the factor for the rest of p adds a rounding, and what 1 + x leaves out of 2^(x / ln 2), x^2 / 2 <= 1.6 units for
x <= 90 * 4.9e-6.  Behind GELU p is off by 3 |p| (two constants of half a unit each, two roundings), which moves e by ln 2
of that: 2.1 |p|.  An error of e moves v by e / (1 + e) of it; the sum's rounding and v's own add 1 each.
The product with `up` and the division by 127 add 1 each."""
import pytest
import torch

from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def _power(a, act):
    a = a.double()
    return a * -1.4426950408889634 * (2 * 0.79788456 * (1 + 0.044715 * a * a) if act == "gelu" else 1.0)


def _act64(a, act):
    return a.double() / (1 + torch.exp2(_power(a, act)))


def _tolerance(a, act):
    """Relative bound of v, of the definition's value for the bf16 argument a."""
    p = _power(a, act)
    return UNIT * (2 + (4 + 2.1 * p.abs() if act == "gelu" else 6.6) * torch.sigmoid(p * 0.6931471805599453))


def test_half_way_quotients_behind_gelu(cuda):
    """GELU is the identity from 8 up (exp(-2u) < 2^-64 of it), so quotients are half-way as often as without it: all of
    (m + 1/2) / 127 for a largest element of 127 * 2^e, and one half for any.  They go to the even code."""
    from fp8_gmm_b200 import backend

    ties = torch.arange(0, 127) + 0.5
    rows = [torch.cat([torch.tensor([127.0]), ties]) * 2.0 ** e for e in (4, 5, 17, 60, 119)]
    rows += [torch.cat([torch.tensor([t, t / 2]), torch.full((126,), 8.0)]) for t in (16 + torch.arange(0, 128) / 8).tolist()]
    x = torch.stack(rows).to(torch.bfloat16)
    v = x.double()
    want = torch.round(127 * v / v.amax(1, keepdim=True))
    for view in (x.to(cuda), torch.nn.functional.pad(x, (1, 0)).to(cuda)[:, 1:]):      # both kernels: aligned rows, and others
        q, s = backend.quantize_rows_int8(view, activation="gelu")
        assert torch.equal(q.cpu().double(), want)
        assert torch.equal(s.cpu(), x.float().amax(1) / 127)


def test_half_way_quotients_behind_swiglu(cuda):
    """SiLU is the identity from 45 up; times a power of two it stays short, and half-way quotients go to the even code."""
    from fp8_gmm_b200 import backend

    ties = torch.arange(0, 127) + 0.5
    gate = torch.stack([torch.cat([torch.tensor([127.0]), ties]) * 2.0 ** e for e in (7, 8, 30, 90)])
    up = torch.tensor([2.0, -0.25, 1.0, 2.0 ** -20])[:, None].expand_as(gate)
    x = torch.cat([gate, up], 1).to(torch.bfloat16)
    v = gate.double() * up.double()
    want = torch.round(127 * v / v.abs().amax(1, keepdim=True))
    for view in (x.to(cuda), torch.nn.functional.pad(x, (1, 0)).to(cuda)[:, 1:]):
        q, _ = backend.quantize_rows_int8(view, activation="swiglu")
        assert torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("cols", [1, 8])
def test_activation_of_every_bf16_number(cuda, act, cols):
    """A row of one value has scale |v| / 127."""
    from fp8_gmm_b200 import backend

    a = (torch.arange(65536, dtype=torch.int32) - 32768).to(torch.int16).view(torch.bfloat16)
    a = a[torch.isfinite(a)]
    x = a[:, None].expand(-1, cols)
    if act == "swiglu":
        x = torch.cat([x, torch.ones_like(x)], 1)
    q, s = backend.quantize_rows_int8(x.contiguous().to(cuda), activation=act)
    got, want, p = s.cpu().double() * 127, _act64(a, act).abs(), _power(a, act)
    # the scale's own rounding, and that of subnormal values (half of 2^-149, times 127 for the scale's)
    bound = want * (_tolerance(a, act) + UNIT) + 64 * 2.0 ** -149
    inside = p <= 126
    assert ((got - want).abs() <= bound)[inside].all()
    # further out 1 + e leaves the range of the reciprocal: v is 0, or still right
    assert ((got == 0) | ((got - want).abs() <= bound))[~inside].all()
    nonzero = got > 0
    assert torch.equal(q.cpu()[nonzero].abs().unique(), torch.tensor([127], dtype=torch.int8)) and (q.cpu()[~nonzero] == 0).all()
    assert torch.equal(q.cpu()[nonzero][:, 0] > 0, a[nonzero] > 0)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("rows,cols,std", [(700, 4096, 1.0), (64, 14336, 1.0), (300, 1040, 4.0), (33, 677, 2.0), (3, 20000, 1.0)])
def test_codes_next_to_a_border(cuda, act, rows, cols, std):
    """No code is further from the quotient than one half and what the values' own errors come to."""
    from fp8_gmm_b200 import backend

    x = randn_bf16((rows, cols * (2 if act == "swiglu" else 1)), rows, std)
    big = torch.rand(x.shape, generator=torch.Generator().manual_seed(cols)) < 0.002
    x = torch.where(big, x * 20, x)                       # few large values set the row's scale, as in trained models
    q, s = backend.quantize_rows_int8(x.to(cuda), activation=act)
    a = x[:, :cols]
    v, tol = _act64(a, act), _tolerance(a, act)
    if act == "swiglu":
        v, tol = v * x[:, cols:].double(), tol + UNIT
    top, at = v.abs().max(1, keepdim=True)
    tol_top = tol.gather(1, at)
    quotient = 127 * v / top
    assert ((q.cpu().double() - quotient).abs() <= 0.5 + quotient.abs() * (tol + tol_top) * 1.001).all()
    assert ((s.cpu().double() - top[:, 0] / 127).abs() <= top[:, 0] / 127 * (tol_top[:, 0] + UNIT) * 1.001).all()
