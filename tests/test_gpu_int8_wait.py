"""GPU: the limit of the product's bounded waits does not count the quantisation that int8_linear runs in front of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_wait_limit_counts_from_the_end_of_the_quantisation(cuda):
    """Rows that are not aligned go through the kernel whose blocks walk many rows, eight to an SM, of which six fit: the product may
    start beside the last two, milliseconds before the codes are there.  Its own waits are for single stages and tiles of 4080
    bytes, some microseconds each; the limit is a third of a millisecond."""
    from fp8_gmm_b200 import backend

    rows, k, n = 300000, 4080, 16
    x = torch.empty(rows, k + 1, dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(device=cuda).manual_seed(1))[:, 1:]
    w, ws = backend.quantize_rows_int8(torch.randn(1, n, k, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda))
    q, s = backend.quantize_rows_int8(x)
    want = backend.int8_gmm(q, w, [rows], s, ws)
    backend.device_status()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    backend.quantize_rows_int8(x, codes=q, scales=s)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) > 1.0      # ms: far more than the limit
    backend.set_wait_limits(gemm_wait_s=3e-4)
    try:
        for _ in range(3):
            got = backend.int8_linear(x, w, [rows], ws)
            backend.device_status()
            assert torch.equal(got, want)
    finally:
        backend.set_wait_limits(gemm_wait_s=1.0)
