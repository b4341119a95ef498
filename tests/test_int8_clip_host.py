"""CPU: argument checks of the int8 product, the row quantisation and the gradient clip (nothing reaches the GPU), and the
host side of clipping over ranks."""
import ctypes

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _lib():
    from fp8_gmm_b200 import _lib

    return _lib


def test_struct_layouts_match_the_header():
    import os
    import re

    L = _lib()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "fp8_gmm_b200.h")).read(), flags=re.S)
    for cname, cls in [("fp8gmm_quantize_rows_args", L.QuantizeRowsArgs), ("fp8gmm_int8_gemm_args", L.Int8GemmArgs), ("fp8gmm_grad_desc", L.GradDesc)]:
        body = re.search(r"typedef struct \{([^{}]*)\}\s*" + cname + ";", text).group(1)
        fields = [re.search(r"(\w+)\s*$", f.strip()).group(1) for f in body.split(";") if f.strip()]
        assert fields == [f[0].rstrip("_") for f in cls._fields_]
    assert ctypes.sizeof(L.GradDesc) == 32   # backend packs it as four int64


def _gemm_args(**kw):
    L = _lib()
    sizes = (ctypes.c_int64 * 2)(3, 5)
    a = L.Int8GemmArgs(a=256, b=256, c=256, a_scales=256, b_scales=256, num_groups=2, rows=8, n=32, k=64)
    a.m_sizes = ctypes.cast(sizes, ctypes.POINTER(ctypes.c_int64))
    for key, v in kw.items():
        setattr(a, key, v)
    return a, sizes


@pytest.mark.parametrize("change,message", [
    (dict(n=24), b"multiples of 16"), (dict(k=72), b"multiples of 16"), (dict(k=0), b"multiples of 16"), (dict(k=1 << 17), b"overflow"),
    (dict(rows=9), b"sum to 8"), (dict(rows=7), b"bad size"), (dict(rows=-1), b"number of rows"), (dict(num_groups=513), b"num_groups"),
    (dict(num_groups=-1), b"num_groups"), (dict(device_m_sizes=256), b"not both"), (dict(m_sizes=None), b"not both"),
    (dict(a=None), b"NULL"), (dict(b_scales=None), b"NULL"), (dict(b=264), b"aligned"), (dict(n=16 << 27), b"weight rows"),
    (dict(a_ld=48), b"pitch"), (dict(a_ld=72), b"pitch"), (dict(a_ld=-64), b"pitch"), (dict(a_ld=1 << 31), b"pitch"),
])
def test_int8_gemm_refusals(change, message):
    L = _lib()
    a, keep = _gemm_args(**change)
    assert L.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(a), None) == 1
    assert message in L.lib.fp8gmm_last_error(), L.lib.fp8gmm_last_error()


def test_int8_gemm_negative_group_is_refused_and_no_rows_are_fine():
    L = _lib()
    a, _ = _gemm_args()
    sizes = (ctypes.c_int64 * 2)(9, -1)
    a.m_sizes = ctypes.cast(sizes, ctypes.POINTER(ctypes.c_int64))
    assert L.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(a), None) == 1
    a, _ = _gemm_args(rows=0, a=None, b=None, c=None)
    sizes = (ctypes.c_int64 * 2)(0, 0)
    a.m_sizes = ctypes.cast(sizes, ctypes.POINTER(ctypes.c_int64))
    assert L.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(a), None) == 0


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), b"negative"), (dict(activation=3), b"activation"), (dict(in_ld=63), b"pitch"), (dict(activation=2), b"pitch"),
    (dict(in_rows=5), b"row counts"), (dict(indices=256, top_k=0), b"top_k"), (dict(codes=None), b"NULL"), (dict(cols=0, in_ld=0), b"no columns"),
    (dict(codes_ld=63), b"pitch"), (dict(codes_ld=-64), b"pitch"),
])
def test_quantize_rows_refusals(change, message):
    L = _lib()
    a = L.QuantizeRowsArgs(in_=256, in_ld=64, top_k=1, in_rows=4, rows=4, cols=64, activation=0, codes=256, scales=256)
    for key, v in change.items():
        setattr(a, key + "_" if key == "in" else key, v)
    assert L.lib.fp8gmm_quantize_rows_int8(ctypes.byref(a), None) == 1
    assert message in L.lib.fp8gmm_last_error(), L.lib.fp8gmm_last_error()


def _descs(*rows):
    L = _lib()
    arr = (L.GradDesc * len(rows))()
    for d, (i, o, n, it, ot) in zip(arr, rows):
        d.in_, d.out, d.numel, d.in_type, d.out_type = i, o, n, it, ot
    return arr


BF16, F16, F32 = 0, 1, 2


@pytest.mark.parametrize("rows,message", [
    ([(4096, 4096, 10, BF16, BF16), (4096, 4096, 10, BF16, BF16)], b"share"),            # the same gradient twice
    ([(4096, 4096, 10, BF16, BF16), (4096 + 18, 4096 + 18, 10, BF16, BF16)], b"share"),  # overlap by one element
    ([(4096, 8192, 10, BF16, F32), (6000, 8192 + 36, 10, BF16, F32)], b"share"),         # two outputs, one element
    ([(4096, 8192, 100, BF16, BF16), (8192 + 100, 20000, 10, BF16, BF16)], b"share"),    # an input inside another's output
    ([(4096, 4096, 10, BF16, F32)], b"share"),                                           # in place with another type
    ([(4096, 4098, 10, BF16, BF16)], b"share"),                                          # shifted by one
    ([(4096, 4096, -1, BF16, BF16)], b"negative"), ([(4096, 4096, 1, 3, BF16)], b"type"), ([(4096, 4096, 1, BF16, 7)], b"type"),
    ([(None, 4096, 1, BF16, BF16)], b"NULL"), ([(4097, 4097, 1, BF16, BF16)], b"aligned"), ([(4098, 4098, 1, F32, F32)], b"aligned"),
])
def test_clip_refusals(rows, message):
    L = _lib()
    d = _descs(*rows)
    addr = ctypes.addressof(d)
    assert L.lib.fp8gmm_multi_clip(addr, len(rows), 256, 1.0, None, None) == 1
    assert message in L.lib.fp8gmm_last_error(), L.lib.fp8gmm_last_error()
    need = L.lib.fp8gmm_sum_squares_workspace_bytes(len(rows))
    assert L.lib.fp8gmm_multi_clip_grad_norm(addr, len(rows), 1.0, 256, need, 256, None) == 1
    assert message in L.lib.fp8gmm_last_error()


def test_clip_refuses_bad_norms_and_workspaces():
    L = _lib()
    d = _descs((4096, 4096, 10, BF16, BF16), (4096 + 20, 4096 + 20, 0, BF16, BF16))
    addr = ctypes.addressof(d)
    for bad in (-1.0, float("nan")):
        assert L.lib.fp8gmm_multi_clip(addr, 2, 256, bad, None, None) == 1
        assert b"max_norm" in L.lib.fp8gmm_last_error()
    assert L.lib.fp8gmm_multi_clip(addr, 2, None, 1.0, None, None) == 1
    need = L.lib.fp8gmm_sum_squares_workspace_bytes(2)
    for ws, size in ((None, need), (256, need - 1), (260, need)):
        assert L.lib.fp8gmm_multi_sum_squares(addr, 2, ws, size, 256, None, None) == 1
        assert b"workspace" in L.lib.fp8gmm_last_error()
    assert L.lib.fp8gmm_multi_sum_squares(addr, 2, 256, need, None, None, None) == 1
    assert L.lib.fp8gmm_sum_squares_workspace_bytes(2000) > need


def test_python_entries_refuse_cpu_tensors_and_wanted_gradients():
    from fp8_gmm_b200 import backend

    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    w = torch.zeros(2, 16, 32, dtype=torch.int8)
    for call in (lambda: backend.quantize_rows_int8(x), lambda: backend.int8_linear(x, w, [2, 2], torch.zeros(2, 16)),
                 lambda: backend.int8_gmm(w[0], w, [8, 8], torch.zeros(16), torch.zeros(2, 16)), lambda: backend.multi_grad_norm([x]),
                 lambda: backend.multi_clip_grad_norm([x], 1.0), lambda: backend.multi_sum_squares([x]), lambda: backend.multi_clip([x], x, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA|GPU"):
            call()
    with pytest.raises(RuntimeError, match="max_norm"):
        backend.multi_clip_grad_norm([x], -1.0)
    with pytest.raises(RuntimeError, match="no gradient"):
        backend._no_grad_wanted("int8_linear", x.requires_grad_(True))
    with torch.no_grad():
        backend._no_grad_wanted("int8_linear", x)


def test_launches_go_to_the_device_of_the_tensors(monkeypatch):
    """With another device current, the call runs inside torch.cuda.device(the tensors' device) and takes that device's stream."""
    from fp8_gmm_b200 import backend

    seen = []

    class Device:
        def __init__(self, device):
            seen.append(("enter", device.index))

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            seen.append("exit")

    monkeypatch.setattr(backend, "_raw_device", lambda: 0)
    monkeypatch.setattr(backend, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(backend, "_stream", lambda: 777)
    monkeypatch.setattr(torch.cuda, "device", Device)
    backend._enqueue(torch.device("cuda", 0), "a", lambda *args: seen.append(args) or 0, 1, 2)
    assert seen == [(1, 2, 100)]
    seen.clear()
    backend._enqueue(torch.device("cuda", 1), "b", lambda *args: seen.append(args) or 0, 3)
    assert seen == [("enter", 1), (3, 777), "exit"]
    with pytest.raises(RuntimeError, match="status 1"):
        backend._enqueue(torch.device("cuda", 1), "c", lambda *args: 1)


def test_dense_layouts():
    from fp8_gmm_b200 import backend

    t = torch.zeros(4, 6, 5)
    assert backend._dense(t) and backend._dense(t.permute(2, 0, 1)) and backend._dense(t[:, :, None]) and backend._dense(t[1:3])
    assert not backend._dense(t[:, 1:]) and not backend._dense(t[..., ::2]) and not backend._dense(torch.zeros(1, 5).expand(4, 5))
    assert backend._dense(torch.zeros(0, 5)) and backend._dense(torch.zeros(()))


# ---- clipping over ranks: the kernels replaced by their formulas in torch, the all-reduce real (gloo)
def _fake_sum_squares(grads):
    return sum((g.double().square().sum() for g in grads), torch.zeros((), dtype=torch.float64))


def _fake_clip(grads, squares, max_norm, outputs=None):
    norm = squares.sqrt()
    for g in grads:
        g.mul_(torch.clamp(max_norm / (norm + 1e-6), max=1.0).to(g.dtype))
    return norm.float()


def _rank(rank, world, path, out):
    from fp8_gmm_b200 import backend, clip

    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=world)
    backend.multi_sum_squares, backend.multi_clip = _fake_sum_squares, _fake_clip
    p = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2))]
    if rank == 0:
        p[0].grad = torch.tensor([3.0, 0.0, 0.0])   # rank 1 holds no gradient of this one
    else:
        p[1].grad = torch.tensor([0.0, 4.0])
    norm = clip.clip_grad_norm_(p, 1.0, group=dist.group.WORLD)
    out[rank] = (float(norm), [None if q.grad is None else q.grad.tolist() for q in p])
    if rank == 0:
        p[0].grad[1] = float("inf")
    try:
        clip.clip_grad_norm_(p, 1.0, error_if_nonfinite=True, group=dist.group.WORLD)
        out[rank + 10] = "no error"
    except RuntimeError as e:
        out[rank + 10] = str(e)
    dist.destroy_process_group()


def test_clip_over_ranks_uses_the_norm_of_all_shards(tmp_path):
    with mp.Manager() as m:
        out = m.dict()
        mp.spawn(_rank, args=(2, str(tmp_path / "store"), out), nprocs=2)
        out = dict(out)
    assert out[0][0] == out[1][0] == 5.0
    assert out[0][1][0] == pytest.approx([0.6, 0, 0], rel=1e-5) and out[1][1][1] == pytest.approx([0, 0.8], rel=1e-5)
    assert "inf" in out[10] and "inf" in out[11]   # both ranks refuse, also the one whose own gradients are finite
