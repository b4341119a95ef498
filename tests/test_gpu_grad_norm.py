"""GPU: global gradient norm and clipping against 64 bits.

Eight squares at a time are summed in fp32 by fused multiply-adds, the rest in double: step k rounds a sum of k squares, so if all
steps err the same way on equal elements eight squares are off by (1 + ... + 8) / 8 = 4.5 halves of a unit, 4.5 * 2^-24 relative,
the norm by half of that, and its own rounding to fp32 adds 2^-24: 3.25 * 2^-24 < 2^-22.  A clipped element is g * coef with coef rounded to fp32 (2^-24) and the
product rounded to fp32 (2^-24) and to the output's type (half a step)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# the package's own odd shapes, single elements, an empty one, and a tensor of several tiles
SHAPES = [(1,), (3,), (0, 4), (8, 8), (1, 3221), (2333, 1), (1481, 677), (120, 2080), (16384,), (16385,), (2, 3, 5), (4, 256, 1024)]


def _grads(shapes, dtypes, seed, dev, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).to(dev) for i, s in enumerate(shapes)]


def _norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check(outs, grads, coef):
    for o, g in zip(outs, grads):
        want = g.double() * coef
        tiny = {BF: 2.0 ** -134, HF: 2.0 ** -25, F32: 2.0 ** -150}[o.dtype]     # half the smallest subnormal
        assert ((o.double() - want).abs() <= want.abs() * (torch.finfo(o.dtype).eps / 2 + 2.0 ** -22) + tiny + 2.0 ** -149).all()


@pytest.mark.parametrize("dtypes", [(BF,), (F32,), (HF,), (BF, F32, HF)])
def test_norm_and_clip_in_place(cuda, dtypes):
    from fp8_gmm_b200 import backend

    grads = _grads(SHAPES, dtypes, 1, cuda, 0.1)
    before = [g.clone() for g in grads]
    want = _norm64(grads)
    norm = backend.multi_grad_norm(grads)
    assert norm.dtype == F32 and norm.dim() == 0 and abs(float(norm) - want) <= want * 2.0 ** -22
    got = backend.multi_clip_grad_norm(grads, 1.5)
    assert torch.equal(got, norm)
    _check(grads, before, 1.5 / (want + 1e-6))
    # a second call finds the norm at the limit; its result is again min(1, ..)
    after = _norm64(grads)
    backend.multi_clip_grad_norm(grads, after * 2)
    assert abs(_norm64(grads) - after) == 0.0


@pytest.mark.parametrize("in_types,out_type", [((BF,), F32), ((F32,), BF), ((HF, BF), F32), ((BF, F32), HF)])
def test_clip_into_other_types(cuda, in_types, out_type):
    from fp8_gmm_b200 import backend

    grads = _grads(SHAPES, in_types, 2, cuda, 0.05)
    before = [g.clone() for g in grads]
    outs = [torch.full(g.shape, float("nan"), dtype=out_type, device=cuda) for g in grads]
    want = _norm64(grads)
    norm = backend.multi_clip_grad_norm(grads, 0.25, outputs=outs)
    assert abs(float(norm) - want) <= want * 2.0 ** -22
    _check(outs, grads, 0.25 / (want + 1e-6))
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    # below the limit the values pass unchanged (one rounding to the output's type)
    backend.multi_clip_grad_norm(grads, want * 1.5, outputs=outs)
    assert all(torch.equal(o, g.to(out_type)) for o, g in zip(outs, grads))


def test_clip_into_a_flat_buffer(cuda):
    """bf16 gradients of any shape into consecutive pieces of one fp32 buffer, at whatever element they start."""
    from fp8_gmm_b200 import backend

    grads = _grads([s for s in SHAPES if 0 not in s], (BF, HF), 8, cuda)
    flat = torch.full((sum(g.numel() for g in grads) + 3,), 7.0, device=cuda)
    pieces, at = [], 1
    for g in grads:
        pieces.append(flat[at:at + g.numel()])
        at += g.numel()
    want = _norm64(grads)
    backend.multi_clip_grad_norm(grads, 2.0, outputs=pieces)
    _check([p.view(g.shape) for p, g in zip(pieces, grads)], grads, 2.0 / (want + 1e-6))
    assert flat[0] == 7.0 and (flat[-2:] == 7.0).all()


def test_two_steps_with_the_sum_in_between(cuda):
    """multi_sum_squares -> (sum over ranks) -> multi_clip equals the one-call form, and a sum from elsewhere is obeyed."""
    from fp8_gmm_b200 import backend

    grads = _grads(SHAPES, (BF, F32), 3, cuda)
    a = [g.clone() for g in grads]
    squares = backend.multi_sum_squares(grads)
    assert squares.dtype == torch.float64 and abs(float(squares) - _norm64(grads) ** 2) <= float(squares) * 2.0 ** -21
    norm = backend.multi_clip(grads, squares, 2.0)
    assert torch.equal(norm, backend.multi_clip_grad_norm(a, 2.0)) and all(torch.equal(x, y) for x, y in zip(grads, a))
    before = [g.clone() for g in grads]
    norm = backend.multi_clip(grads, torch.tensor(1e4, dtype=torch.float64, device=cuda), 50.0)
    assert float(norm) == 100.0
    _check(grads, before, 50.0 / (100.0 + 1e-6))


@pytest.mark.parametrize("value,dtype", [(1e38, BF), (3e38, F32), (1e-30, BF), (1e-42, F32), (1e25, BF), (1e-22, F32), (6e-8, HF)])
def test_squares_outside_fp32(cuda, value, dtype):
    """Squares that overflow or vanish in fp32 count all the same."""
    from fp8_gmm_b200 import backend

    grads = [torch.full((5000,), value, dtype=dtype, device=cuda), torch.full((70001,), -value, dtype=dtype, device=cuda)]
    want = _norm64(grads)
    got = float(backend.multi_grad_norm(grads))
    if want > torch.finfo(F32).max:
        assert got == float("inf")
        squares = float(backend.multi_sum_squares(grads))
        assert abs(math.sqrt(squares) - want) <= want * 2.0 ** -22
    else:
        assert abs(got - want) <= want * 2.0 ** -22 + 2.0 ** -150


def test_mixed_magnitudes_lose_nothing(cuda):
    """One large element among many tiny ones, and the other way round."""
    from fp8_gmm_b200 import backend

    g = torch.full((300000,), 1e-21, device=cuda)
    assert abs(float(backend.multi_grad_norm([g])) - _norm64([g])) <= _norm64([g]) * 2.0 ** -22
    g[12345] = 1e-18
    assert abs(float(backend.multi_grad_norm([g])) - _norm64([g])) <= _norm64([g]) * 2.0 ** -22
    g[12345] = 1e20
    assert abs(float(backend.multi_grad_norm([g])) - 1e20) <= 1e20 * 2.0 ** -22


def test_zero_infinite_and_nan_gradients(cuda):
    from fp8_gmm_b200 import backend

    inf, nan = float("inf"), float("nan")
    z = [torch.zeros(1000, dtype=BF, device=cuda), torch.zeros(3, device=cuda)]
    assert float(backend.multi_clip_grad_norm(z, 1.0)) == 0.0 and all((g == 0).all() for g in z)
    for bad, norm_is in ((inf, inf), (-inf, inf), (nan, nan)):
        g = [torch.ones(40000, dtype=BF, device=cuda), torch.ones(5, device=cuda)]
        g[0][39999] = bad
        ref = [torch.nn.Parameter(x.clone()) for x in g]
        for p, x in zip(ref, g):
            p.grad = x.clone()
        want = torch.nn.utils.clip_grad_norm_(ref, 1.0)
        got = backend.multi_clip_grad_norm(g, 1.0)
        assert math.isnan(float(got)) if norm_is != norm_is else float(got) == norm_is == float(want)
        assert all(torch.equal(x.isnan(), p.grad.isnan()) and torch.equal(x.nan_to_num(), p.grad.nan_to_num()) for x, p in zip(g, ref))


def test_limits_of_zero_and_infinity(cuda):
    from fp8_gmm_b200 import backend

    g = _grads([(777,), (5, 5)], (BF, F32), 4, cuda)
    before = [x.clone() for x in g]
    backend.multi_clip_grad_norm(g, float("inf"))
    assert all(torch.equal(a, b) for a, b in zip(g, before))
    backend.multi_clip_grad_norm(g, 0.0)
    assert all((x == 0).all() for x in g)


def test_views_alignments_and_layouts(cuda):
    """Gradients that start at any element of a buffer, permuted dense ones, and neighbours that must stay untouched."""
    from fp8_gmm_b200 import backend

    for dtype in (BF, F32):
        buf = torch.randn(40000, generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda)
        keep = buf.clone()
        views = [buf[1:8200], buf[8201:8204], buf[8205:30000], buf[30003:39999].view(12, 833)]
        perm = torch.randn(6, 10, 50, device=cuda).to(dtype).permute(2, 0, 1)
        grads = views + [perm]
        before = [g.clone() for g in grads]
        want = _norm64(grads)
        norm = backend.multi_clip_grad_norm(grads, 3.0)
        assert abs(float(norm) - want) <= want * 2.0 ** -22
        _check(grads, before, 3.0 / (want + 1e-6))
        for i in (0, 8200, 8204, 30000, 30001, 30002, 39999):
            assert buf[i] == keep[i]
        out = torch.empty(8200, dtype=F32, device=cuda)[1:]     # another offset than the gradient's
        backend.multi_clip_grad_norm([views[0]], 1e9, outputs=[out])
        assert torch.equal(out, views[0].float())


def test_more_tensors_than_one_launch_takes(cuda):
    from fp8_gmm_b200 import backend

    grads = _grads([(i % 97,) for i in range(1000)], (BF, F32, HF), 6, cuda)
    before = [g.clone() for g in grads]
    want = _norm64(grads)
    norm = backend.multi_clip_grad_norm(grads, 1.0)
    assert abs(float(norm) - want) <= want * 2.0 ** -22
    _check(grads, before, 1.0 / (want + 1e-6))
    assert float(backend.multi_grad_norm([])) == 0.0 and float(backend.multi_clip_grad_norm([], 1.0)) == 0.0
    assert float(backend.multi_grad_norm([torch.zeros(0, device=cuda)])) == 0.0
    assert float(backend.multi_clip_grad_norm([torch.zeros(0, device=cuda)], 1.0)) == 0.0


def test_more_than_two_to_the_31_elements(cuda):
    from fp8_gmm_b200 import backend

    n = 2 ** 31 + 12345
    g = torch.zeros(n, dtype=BF, device=cuda)
    at = torch.tensor([0, 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 1, n - 1], device=cuda)
    g[at] = torch.tensor([3.0, -1.0, 2.0, 5.0, -7.0, 1.0, 4.0], dtype=BF, device=cuda)
    before = g[at].clone()
    want = math.sqrt(105.0)
    assert abs(float(backend.multi_clip_grad_norm([g], 1.0)) - want) <= want * 2.0 ** -22
    _check([g[at]], [before], 1.0 / (want + 1e-6))
    assert int(torch.count_nonzero(g)) == 7


def test_refusals(cuda):
    from fp8_gmm_b200 import backend

    g = torch.ones(4, 6, device=cuda)
    bad = [
        (lambda: backend.multi_grad_norm([g[:, 1:]]), "gaps"), (lambda: backend.multi_grad_norm([torch.ones(1, 4, device=cuda).expand(3, 4)]), "gaps"),
        (lambda: backend.multi_grad_norm([g.double()]), "bfloat16"), (lambda: backend.multi_grad_norm([g.cpu()]), "CUDA"),
        (lambda: backend.multi_grad_norm([g, g.cpu()]), "CUDA"), (lambda: backend.multi_clip_grad_norm([g, g], 1.0), "share"),
        (lambda: backend.multi_clip_grad_norm([g, g.view(-1)[23:]], 1.0), "share"), (lambda: backend.multi_clip_grad_norm([g], 1.0, outputs=[]), "one output"),
        (lambda: backend.multi_clip_grad_norm([g], 1.0, outputs=[torch.empty(5, 4, device=cuda)]), "layout"),
        (lambda: backend.multi_clip_grad_norm([g], 1.0, outputs=[torch.empty(6, 4, device=cuda).t()]), "layout"),
        (lambda: backend.multi_clip_grad_norm([g], float("nan")), "max_norm"),
        (lambda: backend.multi_clip([g], torch.ones((), device=cuda), 1.0), "float64"),
    ]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()
    assert float(backend.multi_grad_norm([g, g])) == pytest.approx(math.sqrt(48.0))   # reading one twice is no conflict


def test_same_bits_every_time_on_any_stream_and_in_graphs(cuda):
    from fp8_gmm_b200 import backend

    grads = _grads(SHAPES * 3, (BF, F32), 7, cuda)
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    want_norm = backend.multi_clip_grad_norm(grads, 1.0, outputs=outs[0])
    want = [o.clone() for o in outs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = backend.multi_clip_grad_norm(grads, 1.0, outputs=outs[1])
    torch.cuda.synchronize()
    assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(outs[1], want))
    graphs, norms = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(backend.multi_clip_grad_norm(grads, 1.0, outputs=outs[k]))
        graphs.append(g)
    for f in (1.0, 0.5):
        for x in grads:
            x.mul_(f)
        want_norm = backend.multi_clip_grad_norm(grads, 1.0, outputs=want)
        torch.cuda.synchronize()
        for g in graphs:      # both at the same time
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(n, want_norm) for n in norms)
        assert all(torch.equal(a, b) for k in range(2) for a, b in zip(outs[k], want))


def test_module_level_clip_matches_torch(cuda):
    import fp8_gmm_b200 as fg

    torch.manual_seed(0)
    mods = [torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Linear(65, 7), torch.nn.Linear(7, 7)).to(cuda) for _ in range(2)]
    mods[1].load_state_dict(mods[0].state_dict())
    x = torch.randn(9, 33, device=cuda)
    for m in mods:
        m[:2](x).square().sum().backward()        # the last layer has no gradient
    want = torch.nn.utils.clip_grad_norm_(mods[0].parameters(), 0.7)
    got = fg.clip_grad_norm_(mods[1].parameters(), 0.7)
    # torch sums in fp32: allow its rounding (a few hundred terms, 2^-20) on top
    assert abs(float(got) - float(want)) <= float(want) * 2.0 ** -20
    for a, b in zip(mods[0].parameters(), mods[1].parameters()):
        assert (a.grad is None) == (b.grad is None) and (a.grad is None or torch.allclose(a.grad, b.grad, rtol=2.0 ** -19, atol=0))
    assert float(fg.clip_grad_norm_(mods[1][0].weight, 1e9)) > 0
    mods[1][0].weight.grad[0, 0] = float("inf")
    before = mods[1][0].weight.grad.clone()
    with pytest.raises(RuntimeError, match="left as they are"):
        fg.clip_grad_norm_(mods[1].parameters(), 0.1, error_if_nonfinite=True)
    assert torch.equal(mods[1][0].weight.grad, before)
    assert float(fg.clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device=cuda))], 1.0)) == 0.0


def test_train_clip_and_evaluate_in_int8(cuda):
    """The operators together, as a training loop uses them: FP8 step of the experts behind the router, gradients of
    experts and router clipped to a global norm, optimizer step, then the new weights evaluated in int8 without recipe
    state.  The int8 pass agrees with the new bf16 weights in 64 bits to 8-bit rounding."""
    import fp8_gmm_b200 as fg
    from fp8_gmm_b200 import routing
    from tests.helpers import randn_bf16

    E, top_k, H, F, T = 4, 2, 128, 256, 200
    torch.manual_seed(0)
    mlp = fg.GroupedMlp(H, F, E, torch.bfloat16, device=cuda, activation="swiglu")
    gate = torch.nn.Linear(H, E, bias=False).to(cuda)
    params = list(mlp.parameters()) + list(gate.parameters())
    opt = torch.optim.SGD(params, lr=0.5)
    x, target = randn_bf16((T, H), 1).to(cuda), randn_bf16((T, H), 2).to(cuda)
    experts = fg.Int8GroupedMlp.from_mlp(mlp)
    for _ in range(3):
        weights, selected = routing.topk(gate(x.float()), top_k)
        indices, bin_ids, bins, sizes = routing.indices_and_bins(selected, E)
        rows = routing.gather(x, indices, bin_ids, bins, top_k)
        with fg.fp8_autocast(enabled=True):
            y = mlp(rows, sizes.cpu())
        out = routing.scatter(y, indices, bin_ids, weights, bins, top_k)
        (out.float() - target.float()).square().sum().backward()
        grads = [p.grad.clone() for p in params]
        want = _norm64(grads)
        norm = fg.clip_grad_norm_(params, 1.0)
        assert abs(float(norm) - want) <= want * 2.0 ** -22 and want > 1.0
        _check([p.grad for p in params], grads, 1.0 / (want + 1e-6))
        opt.step()
        opt.zero_grad()
        experts.refresh(mlp)
        with torch.no_grad():
            rows8 = experts(x, sizes, indices=indices, top_k=top_k)
            parts = rows.detach().double().split(sizes.tolist())
            ref = []
            for g, p in enumerate(parts):
                a, b = (p @ mlp.fc1_weight[g].double().t()).chunk(2, dim=1)
                ref.append((a * torch.sigmoid(a) * b) @ mlp.fc2_weight[g].double().t())
            ref = torch.cat(ref)
            assert float((rows8.double() - ref).norm() / ref.norm()) < 0.05
    fg.backend.device_status()
