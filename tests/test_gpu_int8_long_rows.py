"""GPU: the row quantisation's other kernel (rows over 16384 columns, or not aligned to 16 bytes) behind the router's gather, with
indices that name no row, and in the whole call."""
import pytest
import torch

from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu


def _quantize64(x):
    v = x.double()
    top = v.abs().amax(-1, keepdim=True)
    q = torch.round(v * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return q.to(torch.int8), top[..., 0].float() / 127


@pytest.mark.parametrize("cols,offset", [(20000, 0), (28672, 8), (1040, 1), (272, 3), (16392, 0)])
def test_gather_and_indices_that_name_no_row(cuda, cols, offset):
    from fp8_gmm_b200 import _lib, backend

    x = randn_bf16((7, cols + offset), cols)
    view, cpu = x.to(cuda)[:, offset:], x[:, offset:]
    idx = torch.tensor([0, 13, 13, 6, 2, 9, 1, 12], dtype=torch.int32)
    want_q, want_s = _quantize64(cpu[idx.long() // 2])
    q, s = backend.quantize_rows_int8(view, idx.to(cuda), 2)
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    backend.device_status()
    idx[2], idx[4], idx[7] = -1, 14, 2 ** 31 - 1
    q, s = backend.quantize_rows_int8(view, idx.to(cuda), 2)
    assert _lib.lib.fp8gmm_device_status(torch.cuda.current_stream().cuda_stream) == 4
    bad = [2, 4, 7]
    keep = [i for i in range(8) if i not in bad]
    assert (q[bad] == 0).all() and (s[bad] == 0).all()
    assert torch.equal(q.cpu()[keep], want_q[keep]) and torch.equal(s.cpu()[keep], want_s[keep])


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_both_kernels_give_the_same_codes_behind_an_activation(cuda, act):
    """The same rows aligned and not, and with more rows than blocks run at once."""
    from fp8_gmm_b200 import backend

    rows, cols = 3000, 272
    x = randn_bf16((rows, cols * (2 if act == "swiglu" else 1)), 5, std=2.0)
    shifted = torch.nn.functional.pad(x, (1, 0)).to(cuda)[:, 1:]
    idx = torch.randint(0, 2 * rows, (4001,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(cuda)
    for kw in ({}, dict(indices=idx, top_k=2)):
        a, b = backend.quantize_rows_int8(x.to(cuda), activation=act, **kw), backend.quantize_rows_int8(shifted, activation=act, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_long_rows_through_the_whole_call(cuda):
    from fp8_gmm_b200 import backend

    tokens, top_k, k, n = 9, 2, 28672, 48
    x = randn_bf16((tokens, k), 1).to(cuda)
    w, ws = backend.quantize_rows_int8(randn_bf16((3, n, k), 2).to(cuda))
    idx = torch.randperm(tokens * top_k, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(cuda)
    sizes = [7, 0, 11]
    q, s = backend.quantize_rows_int8(x, idx, top_k)
    want = backend.int8_gmm(q, w, sizes, s, ws)
    assert torch.equal(backend.int8_linear(x, w, sizes, ws, indices=idx, top_k=top_k), want)
    assert torch.equal(backend.int8_linear(x, w, torch.tensor(sizes, device=cuda), ws, indices=idx, top_k=top_k), want)
    backend.device_status()
