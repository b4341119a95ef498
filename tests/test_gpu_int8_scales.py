"""GPU: the int8 product with scales of any size.

Where the product of a row's and a channel's scale is a normal fp32 number (or one of them is 0) the result is
bf16(fp32(sum) * fp32(scale * scale)), elsewhere the three factors are multiplied in 64 bits: both are compared bit for bit."""
import pytest
import torch

from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu
ROWS = [1e-2, 2e-33, 0.0, 1e25, 1e-30, 3e38, 1.4e-45, 1e-38, 1.0, float("nan"), float("inf"), 2.0 ** -62, 2.0 ** 63, -1e-3, 5e-20]
CHANNELS = [1e-3, 3e-11, 1e20, 1e-12, 0.0, 3e38, 2e-39, 1.0, 2.0 ** -63, 2.0 ** 64, 1e-20, 1.4e-45, 7e12, -2e-2, 1e30, 6e-8]


def _want(a, b, sizes, sa, sb):
    out, r = [], 0
    for g, m in enumerate(sizes):
        acc = a[r:r + m].double() @ b[g].double().t()
        rows, channels = sa[r:r + m, None], sb[g][None]
        s = rows * channels
        normal = (s.abs() >= torch.finfo(torch.float32).tiny) & torch.isfinite(s)
        wide = (acc * rows.double() * channels.double()).float()
        out.append(torch.where(normal, acc.float() * s, wide).to(torch.bfloat16))
        r += m
    return torch.cat(out)


def _same(got, want):
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("tile_rows,tile_channels", [(0, 0), (128, 128), (256, 256)])
@pytest.mark.parametrize("sizes,n,k", [([15], 16, 64), ([40, 0, 33], 272, 48), ([300, 1], 144, 272)])
def test_scales_of_any_size(cuda, sizes, n, k, tile_rows, tile_channels):
    from fp8_gmm_b200 import backend

    rows, G = sum(sizes), len(sizes)
    g = torch.Generator().manual_seed(rows)
    a = torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int32).to(torch.int8)
    b = torch.randint(-128, 128, (G, n, k), generator=g, dtype=torch.int32).to(torch.int8)
    a[::7] = 0                                                       # sums of 0, under every scale
    sa = torch.tensor(ROWS)[torch.arange(rows) % len(ROWS)]
    sb = torch.tensor(CHANNELS)[torch.arange(G * n) % len(CHANNELS)].view(G, n)
    want = _want(a, b, sizes, sa, sb)
    backend.set_int8_variant(tile_rows, tile_channels)
    try:
        _same(backend.int8_gmm(a.to(cuda), b.to(cuda), sizes, sa.to(cuda), sb.to(cuda)).cpu(), want)
        backend.device_status()
    finally:
        backend.set_int8_variant()


@pytest.mark.parametrize("where", ["row", "channel"])
def test_one_scale_out_of_range_changes_no_other_result(cuda, where):
    """Rows and channels that share a tile with it keep their bits; its own sums of 0 are 0."""
    from fp8_gmm_b200 import backend

    sizes, n, k = [200], 272, 128
    g = torch.Generator().manual_seed(3)
    a = torch.randint(-127, 128, (200, k), generator=g, dtype=torch.int32).to(torch.int8)
    b = torch.randint(-127, 128, (1, n, k), generator=g, dtype=torch.int32).to(torch.int8)
    a[33], b[0, 50] = 0, 0
    sa, sb = torch.rand(200, generator=g) * 0.01 + 1e-4, torch.rand(1, n, generator=g) * 0.01 + 1e-4
    before = backend.int8_gmm(a.to(cuda), b.to(cuda), sizes, sa.to(cuda), sb.to(cuda)).cpu()
    if where == "row":
        sa[33], sb[0, 50] = 3e38, 1e30
    else:
        sb[0, 50], sa[33] = 3e38, 1e30
    got = backend.int8_gmm(a.to(cuda), b.to(cuda), sizes, sa.to(cuda), sb.to(cuda)).cpu()
    keep = torch.ones(200, n, dtype=torch.bool)
    keep[33], keep[:, 50] = False, False
    assert torch.equal(got[keep], before[keep]) and (got[33] == 0).all() and (got[:, 50] == 0).all()


def test_tiny_activations_through_the_whole_call(cuda):
    """int8_linear of rows near the bottom of bf16's range: normal results that a rounded product of the scales would miss by up
    to a per cent."""
    from fp8_gmm_b200 import backend

    x = (randn_bf16((20, 256), 1).float() * 2.0 ** -116).to(torch.bfloat16)
    w = (randn_bf16((1, 64, 256), 2).float() * 2.0 ** -10).to(torch.bfloat16)
    codes, scales = backend.quantize_rows_int8(w.to(cuda))
    q, s = backend.quantize_rows_int8(x.to(cuda))
    got = backend.int8_linear(x.to(cuda), codes, [20], scales).cpu()
    exact = (q.cpu().double() * s.cpu().double()[:, None]) @ (codes[0].cpu().double() * scales[0].cpu().double()[:, None]).t()
    _same(got, _want(q.cpu(), codes.cpu(), [20], s.cpu(), scales.cpu()))
    # bf16's half step, the two scales' and the sum's fp32 roundings, and half of fp32's smallest number where results are subnormal
    assert ((got.double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 2.0 ** -22) + 2.0 ** -134).all()
