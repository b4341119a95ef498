"""The device status word tells bounded waits that ran out (results undefined) from input that a kernel left out (results
defined): what the host makes of each bit, on the CPU, and what the library reports for bad input, on the GPU."""
import ctypes
import re
import types

import pytest
import torch

INDEX, SIZES, WAIT, PEER = 0x200, 0x400, 0x4, 0x100


def _watch(word):
    from fp8_gmm_b200 import backend

    w = object.__new__(backend.StatusWatch)     # without the page-locked memory, which needs a GPU
    w.host = torch.tensor([word], dtype=torch.int32)
    return w


def test_bits_match_the_header():
    import os

    from fp8_gmm_b200 import backend

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "fp8_gmm_b200.h")).read()
    bits = {name: int(v, 16) for name, v in re.findall(r"(FP8GMM_STATUS_\w+) = (0x[0-9a-fA-F]+)", text)}
    assert bits == {"FP8GMM_STATUS_GEMM_WAIT": 0xF, "FP8GMM_STATUS_PEER_WAIT": PEER, "FP8GMM_STATUS_BAD_INDEX": INDEX, "FP8GMM_STATUS_BAD_SIZES": SIZES}
    assert backend.STATUS_WAITS == 0xF | PEER


@pytest.mark.parametrize("word", [WAIT, PEER, WAIT | INDEX, PEER | SIZES])
def test_watch_reports_waits(word):
    for waits_only in (False, True):
        with pytest.raises(RuntimeError, match="bounded wait"):
            _watch(word).check(waits_only)


@pytest.mark.parametrize("word", [INDEX, SIZES, INDEX | SIZES])
def test_watch_reports_bad_input_as_such(word):
    with pytest.raises(RuntimeError) as e:
        _watch(word).check()
    assert "input" in str(e.value) and "bounded wait" not in str(e.value) and "peer" not in str(e.value)
    _watch(word).check(waits_only=True)
    _watch(0).check()


class _Reached(Exception):
    pass


@pytest.mark.parametrize("word,fails", [(0, False), (INDEX, False), (SIZES, False), (PEER, True), (WAIT, True), (PEER | SIZES, True)])
def test_expert_parallel_exchange_is_given_up_for_waits_only(monkeypatch, word, fails):
    """A serving call's bad index or sizes on the same device leave the exchange of the training job as it is."""
    from fp8_gmm_b200 import ep_peer

    ctx = types.SimpleNamespace(failed=False, status=_watch(word))
    monkeypatch.setattr(ep_peer.EpContext, "setup", classmethod(lambda cls, device, group: ctx))

    def reached(*_):
        raise _Reached

    module = types.SimpleNamespace(group=None, mlp=types.SimpleNamespace(get_fp8_weights_scratchpad=reached))
    x = torch.zeros(2, 2)
    with pytest.raises(RuntimeError if fails else _Reached):
        ep_peer.forward(module, x, None, None, 1)
    assert ctx.failed == fails
    ctx.status.host[0] = 0
    with pytest.raises(RuntimeError if fails else _Reached):     # given up for good, or as before
        ep_peer.forward(module, x, None, None, 1)


@pytest.mark.gpu
def test_library_names_bad_input(cuda):
    from fp8_gmm_b200 import _lib, backend

    stream = torch.cuda.current_stream().cuda_stream
    backend.device_status()
    x = torch.ones(4, 32, dtype=torch.bfloat16, device=cuda)
    w, ws = backend.quantize_rows_int8(torch.ones(2, 16, 32, dtype=torch.bfloat16, device=cuda))
    watch = backend.StatusWatch()
    for call, word in ((lambda: backend.quantize_rows_int8(x, torch.tensor([0, 9], dtype=torch.int32, device=cuda)), INDEX),
                       (lambda: backend.int8_linear(x, w, torch.tensor([3, 2], device=cuda), ws), SIZES)):
        call()
        watch.record()
        torch.cuda.synchronize()
        assert int(watch.host[0]) == word
        watch.check(waits_only=True)
        with pytest.raises(RuntimeError, match="input"):
            watch.check()
        assert _lib.lib.fp8gmm_device_status(stream) == 4
        message = ctypes.string_at(_lib.lib.fp8gmm_last_error()).decode()
        assert "input" in message and "bounded wait" not in message and f"0x{word:x}" in message
        backend.device_status()
