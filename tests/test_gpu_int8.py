"""GPU: int8 row quantisation and grouped product against the definition in 64 bits.

The codes and the integer sums are exact, so without an activation every output is compared bit for bit: codes with the
correctly rounded quotient, products with fp32(sum) * fp32(scale * scale) rounded to bf16, which fp32 torch on the CPU
reproduces.  Behind an activation the row is known to the accuracy of fp32's exp and division (relative error below 2^-17,
dominated by the argument of exp: |x| log2(e) 2^-24 at |x| <= 80), which moves a quotient of at most 127 by less than
127 * 2 * 2^-17 = 0.002."""
import pytest
import torch

from tests.helpers import randn_bf16, routed_group_sizes

pytestmark = pytest.mark.gpu
ACT_REL = 2.0 ** -17


def _act64(x, act):
    v = x.double()
    if act == "swiglu":
        g, u = v.chunk(2, dim=-1)
        return g / (1 + torch.exp(-g)) * u
    if act == "gelu":
        return v / (1 + torch.exp(-2 * 0.79788456 * v * (1 + 0.044715 * v * v)))
    return v


def _quantize64(x):
    """(codes, scales) of rows without an activation: quotients in 64 bits, the scale as one fp32 division."""
    v = x.double()
    top = v.abs().amax(-1, keepdim=True)
    q = torch.round(v * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return q.to(torch.int8), top[..., 0].float() / 127


def _product(a, b, sizes, sa, sb):
    """int64 sums, then the kernel's three fp32 roundings and the bf16 one."""
    out, r = [], 0
    for g, m in enumerate(sizes):
        acc = (a[r:r + m].double() @ b[g].double().t())    # exact: below 2^53
        out.append((acc.float() * (sa[r:r + m, None] * sb[g][None])).to(torch.bfloat16))
        r += m
    return torch.cat(out) if out else torch.empty(0, b.shape[1], dtype=torch.bfloat16)


def _codes(shape, seed, lo=-127, hi=127):
    return torch.randint(lo, hi + 1, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(torch.int8)


def _scales(shape, seed):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed)) * 0.01 + 1e-4


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (2, 33), (7, 677), (1, 1481), (33, 4096), (2, 14336), (4, 40961), (300, 128), (2, 131056)])
def test_codes_are_correctly_rounded(cuda, rows, cols):
    from fp8_gmm_b200 import backend

    x = randn_bf16((rows, cols), rows * 7 + cols, std=3.0)
    q, s = backend.quantize_rows_int8(x.to(cuda))
    want_q, want_s = _quantize64(x)
    assert q.shape == (rows, cols) and torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


def test_ties_extremes_and_special_rows(cuda):
    """Half-way quotients (top * (2 i + 1) / 254 is representable for top = 127 * 2^e), the type's extremes, rows of zeros,
    rows with infinities or NaN."""
    from fp8_gmm_b200 import backend

    ties = (torch.arange(-127, 127) + 0.5)
    inf, nan = float("inf"), float("nan")
    rows = [torch.cat([torch.tensor([127.0]), ties]) * 2.0 ** e for e in (0, 20, -40, 110, -120)]
    rows += [torch.cat([torch.tensor([1.0, 0.5, -0.5, 0.25]), torch.linspace(-1, 1, 251)]) * f for f in (1.0, 1.7, 3e38, 1e-38)]
    rows += [torch.zeros(255), torch.full((255,), -0.0), torch.full((255,), 9.2e-41), torch.full((255,), 3.3895e38)]
    x = torch.stack(rows).to(torch.bfloat16)
    q, s = backend.quantize_rows_int8(x.to(cuda))
    want_q, want_s = _quantize64(x)
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    bad = torch.ones(4, 255, dtype=torch.bfloat16)
    bad[0, 17], bad[1, 254], bad[2, 0] = inf, nan, -inf
    q, s = backend.quantize_rows_int8(bad.to(cuda))
    assert (q[:3] == 0).all() and s[:3].isnan().all() and (q[3] == 127).all() and float(s[3]) == float(torch.tensor(1.0) / 127)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (3, 1024), (2, 14336), (65, 272)])
def test_activation_in_front(cuda, act, rows, cols):
    from fp8_gmm_b200 import backend

    x = randn_bf16((rows, cols * (2 if act == "swiglu" else 1)), rows + cols, std=4.0)
    q, s = backend.quantize_rows_int8(x.to(cuda), activation=act)
    v = _act64(x, act)
    top = v.abs().amax(1, keepdim=True)
    assert torch.allclose(s.cpu().double(), top[:, 0] / 127, rtol=ACT_REL + 2.0 ** -23, atol=0)
    assert float((q.cpu().double() - v * 127 / top).abs().max()) <= 0.5 + 127 * 2 * ACT_REL


def test_activation_far_out(cuda):
    """Gates where exp overflows: the activation is 0 or the identity, never NaN."""
    from fp8_gmm_b200 import backend

    x = torch.tensor([[-1e4, 1e4, -200.0, 90.0, 0.0, -1e30, 2.0, 2.0, 2.0, 2.0, 2.0, 2.0]]).to(torch.bfloat16)
    q, s = backend.quantize_rows_int8(x.to(cuda), activation="swiglu")
    assert q.cpu().tolist() == [[0, 127, 0, 1, 0, 0]] and torch.isfinite(s).all()
    q, s = backend.quantize_rows_int8(x.to(cuda)[:, :5].contiguous(), activation="gelu")
    assert q.cpu().tolist() == [[0, 127, 0, 1, 0]] and torch.isfinite(s).all()


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_activations_near_the_end_of_fp32s_range(cuda, act):
    """Rows whose activations are all tiny: products near 1e-39, and gates at -88, where e^88 is within a factor of two of
    fp32's largest number (subnormal activations keep at least 18 bits here, more than ACT_REL asks)."""
    from fp8_gmm_b200 import backend

    width = 40
    g = torch.Generator().manual_seed(1)
    tiny = (torch.rand(2, 2 * width, generator=g) + 0.5) * (3e-20 if act == "swiglu" else 6e-39)
    deep = torch.rand(2, 2 * width, generator=g) + 0.5
    deep[:, :width] = -88.0 + torch.rand(2, width, generator=g)
    if act == "gelu":
        deep = -(torch.rand(2, 2 * width, generator=g) * 0.15 + 9.85)    # sigmoid(2u) down to e^-87 at -10
    x = torch.cat([tiny, deep]).to(torch.bfloat16)
    q, s = backend.quantize_rows_int8(x.to(cuda), activation=act)
    v = _act64(x, act)
    top = v.abs().amax(1, keepdim=True)
    # the argument of exp is about 88 here, and off by up to four roundings: 88 * 4 * 2^-24 < 2^-15
    rel = 2.0 ** -15
    assert torch.allclose(s.cpu().double(), top[:, 0] / 127, rtol=rel + 2.0 ** -23, atol=2.0 ** -149)
    assert float((q.cpu().double() - v * 127 / top).abs().max()) <= 0.5 + 127 * 2 * rel


def test_rows_with_a_pitch_an_offset_and_three_dimensions(cuda):
    from fp8_gmm_b200 import backend

    base = randn_bf16((9, 200), 1).to(cuda)
    for view in (base[:, :64], base[:, 8:72], base[:, 1:66], base[::2, 3:4], base[1:2, 5:105]):
        q, s = backend.quantize_rows_int8(view)
        want_q, want_s = _quantize64(view.cpu())
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    w = randn_bf16((3, 16, 48), 2)
    q, s = backend.quantize_rows_int8(w.to(cuda))
    want_q, want_s = _quantize64(w)
    assert q.shape == w.shape and s.shape == (3, 16) and torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    codes, scales = torch.empty_like(q), torch.empty_like(s)
    got = backend.quantize_rows_int8(w.to(cuda), codes=codes, scales=scales)
    assert got[0] is codes and torch.equal(codes, q) and torch.equal(scales, s)


def test_gather_by_indices(cuda):
    from fp8_gmm_b200 import _lib, backend

    x = randn_bf16((11, 136), 3)
    idx = torch.tensor([0, 0, 21, 5, 7, 20, 20, 13], dtype=torch.int32)    # the same row several times
    q, s = backend.quantize_rows_int8(x.to(cuda), idx.to(cuda), 2)
    want_q, want_s = _quantize64(x[idx.long() // 2])
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    backend.device_status()
    idx[3], idx[5] = -1, 22                                                # name no row: zeros, reported
    q, s = backend.quantize_rows_int8(x.to(cuda), idx.to(cuda), 2)
    assert _lib.lib.fp8gmm_device_status(torch.cuda.current_stream().cuda_stream) == 4
    for r in (3, 5):
        assert (q[r] == 0).all() and float(s[r]) == 0.0
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(q.cpu()[keep], want_q[keep])
    q, s = backend.quantize_rows_int8(x.to(cuda), idx[:0].to(cuda), 2)
    assert q.shape == (0, 136) and s.shape == (0,)


# ------------------------------------------------------------------------------------------------ product
@pytest.mark.parametrize("sizes,n,k", [
    ([1], 16, 16), ([0, 1, 0], 16, 48), ([3], 128, 128), ([2, 0, 5], 272, 144), ([16, 17, 0, 1], 144, 272), ([31, 33], 1424, 2080),
    ([64, 65, 0, 1, 127], 48, 4112), ([300, 0, 24, 17], 512, 768), ([128, 128], 256, 256), ([129, 255, 257], 400, 64), ([513], 1040, 1024),
    ([1] * 37, 64, 112), ([700, 3, 900], 528, 176), ([0, 0], 32, 32), ([2], 4096, 14336), ([1, 1], 16, 131056),
])
def test_product_is_exact(cuda, sizes, n, k):
    from fp8_gmm_b200 import backend

    rows, G = sum(sizes), len(sizes)
    a, b = _codes((rows, k), 1, -128), _codes((G, n, k), 2, -128)
    sa, sb = _scales((rows,), 3), _scales((G, n), 4)
    want = _product(a, b, sizes, sa, sb)
    dev = [t.to(cuda) for t in (a, b, sa, sb)]
    got = backend.int8_gmm(dev[0], dev[1], torch.tensor(sizes), dev[2], dev[3])
    assert torch.equal(got.cpu(), want)
    on_gpu = backend.int8_gmm(dev[0], dev[1], torch.tensor(sizes, device=cuda), dev[2], dev[3])
    backend.device_status()
    assert torch.equal(on_gpu, got)


@pytest.fixture
def any_variant():
    from fp8_gmm_b200 import backend

    yield backend.set_int8_variant
    backend.set_int8_variant()


@pytest.mark.parametrize("tile_channels", [128, 256])
@pytest.mark.parametrize("tile_rows", [128, 256])
def test_every_tile_gives_the_same_bits(cuda, any_variant, tile_rows, tile_channels):
    from fp8_gmm_b200 import backend

    any_variant(tile_rows, tile_channels)
    for sizes, n, k in [([1], 16, 16), ([5, 0, 16, 17, 33], 272, 1040), ([64, 129, 1, 255, 256, 257], 400, 2080), ([2, 7], 1424, 4112), ([300], 128, 128),
                        ([300], 128, 8192), ([7, 0, 270], 272, 14336), ([3], 48, 131056), ([40] * 20, 1040, 2064)]:
        rows, G = sum(sizes), len(sizes)
        a, b = _codes((rows, k), 1, -128), _codes((G, n, k), 2, -128)
        sa, sb = _scales((rows,), 3), _scales((G, n), 4)
        want = _product(a, b, sizes, sa, sb)
        c = torch.full((rows + 3, n), 7.0, dtype=torch.bfloat16, device=cuda)
        for m in (torch.tensor(sizes), torch.tensor(sizes, device=cuda)):
            backend.int8_gmm(a.to(cuda), b.to(cuda), m, sa.to(cuda), sb.to(cuda), c=c[:rows])
            backend.device_status()
            assert torch.equal(c[:rows].cpu(), want) and (c[rows:] == 7.0).all()


def test_largest_sums_do_not_overflow(cuda):
    from fp8_gmm_b200 import backend

    k = 131056
    a, b = torch.full((2, k), -128, dtype=torch.int8), torch.full((1, 16, k), -128, dtype=torch.int8)
    b[0, 1] = 127
    one = torch.ones(2)
    got = backend.int8_gmm(a.to(cuda), b.to(cuda), [2], one.to(cuda), torch.ones(1, 16).to(cuda))
    assert torch.equal(got.cpu(), _product(a, b, [2], one, torch.ones(1, 16)))


def test_many_rows_in_few_and_many_groups(cuda):
    """Row counts around every tile size of the kernel, compared on the GPU in 64 bits."""
    from fp8_gmm_b200 import backend

    n, k = 272, 320
    for G, rows, seed in [(1, 4097, 1), (3, 5000, 2), (64, 6144, 3), (200, 3000, 4), (512, 700, 5)]:
        sizes = routed_group_sizes(G, rows, seed)
        a, b = _codes((rows, k), seed).to(cuda), _codes((G, n, k), seed + 9).to(cuda)
        sa, sb = _scales((rows,), 3).to(cuda), _scales((G, n), 4).to(cuda)
        got = backend.int8_gmm(a, b, sizes, sa, sb)
        assert torch.equal(got, _product(a, b, sizes, sa, sb))


def test_offsets_beyond_32_bits(cuda):
    """Codes, results and weights of more than 2^32 bytes: rows and channels at both ends and around the borders."""
    from fp8_gmm_b200 import backend

    G, n, k, rows = 5, 16384, 65536, 66000          # weights 5.4 GB, codes 4.3 GB, results 2.2 GB
    g = torch.Generator(device=cuda).manual_seed(1)
    w = torch.empty(G, n, k, dtype=torch.int8, device=cuda)
    w.view(torch.int64).random_(generator=g)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    ws = _scales((G, n), 4).to(cuda)
    sizes = [65000, 0, 300, 1, 699]
    codes, scales = backend.quantize_rows_int8(x)
    pick = torch.tensor([0, 1, 32767, 32768, 64999, 65000, 65299, 65300, 65301, 65536, 65537, 65999], device=cuda)
    want_q, want_s = _quantize64(x[pick].cpu())
    assert torch.equal(codes[pick].cpu(), want_q) and torch.equal(scales[pick].cpu(), want_s)
    del x
    out = backend.int8_gmm(codes, w, sizes, scales, ws)
    backend.device_status()
    ends = torch.tensor(sizes).cumsum(0)
    for r in pick.tolist():
        grp = int((ends <= r).sum())
        cols = torch.tensor([0, 1, n // 2, n - 1], device=cuda)
        acc = codes[r].double() @ w[grp, cols].double().t()
        want = (acc.float() * (scales[r] * ws[grp, cols])).to(torch.bfloat16)
        assert torch.equal(out[r, cols], want), r


def test_sizes_on_the_gpu_leave_the_rows_behind_alone(cuda):
    from fp8_gmm_b200 import _lib, backend

    a, b = _codes((50, 64), 1).to(cuda), _codes((3, 48, 64), 2).to(cuda)
    sa, sb = _scales((50,), 3).to(cuda), _scales((3, 48), 4).to(cuda)
    for sizes in ([10, 0, 23], [0, 0, 0], [50, 0, 0]):
        c = torch.full((50, 48), 7.0, dtype=torch.bfloat16, device=cuda)
        backend.int8_gmm(a, b, torch.tensor(sizes, device=cuda), sa, sb, c=c)
        backend.device_status()
        m = sum(sizes)
        assert torch.equal(c[:m].cpu(), _product(a.cpu(), b.cpu(), sizes, sa.cpu(), sb.cpu())) and (c[m:] == 7.0).all()
    # sizes that do not fit are cut off and reported
    for sizes, cut in ([20, 40, 5], [20, 30, 0]), ([-3, 20, 1 << 40], [0, 20, 30]):
        c = torch.full((50, 48), 7.0, dtype=torch.bfloat16, device=cuda)
        backend.int8_gmm(a, b, torch.tensor(sizes, device=cuda), sa, sb, c=c)
        assert _lib.lib.fp8gmm_device_status(torch.cuda.current_stream().cuda_stream) == 4
        assert torch.equal(c.cpu(), _product(a.cpu(), b.cpu(), cut, sa.cpu(), sb.cpu()))


def test_a_bad_row_spoils_no_other(cuda):
    from fp8_gmm_b200 import backend

    x = randn_bf16((6, 64), 1)
    w = _codes((2, 32, 64), 2).to(cuda)
    ws = _scales((2, 32), 3).to(cuda)
    good = backend.int8_linear(x.to(cuda), w, [4, 2], ws)
    x[1, 5], x[5, 0] = float("nan"), float("inf")
    got = backend.int8_linear(x.to(cuda), w, [4, 2], ws)
    assert got[[1, 5]].isnan().all() and torch.equal(got[[0, 2, 3, 4]], good[[0, 2, 3, 4]])
    x[:] = 0
    assert (backend.int8_linear(x.to(cuda), w, [4, 2], ws) == 0).all()


def test_refusals_on_the_gpu(cuda):
    from fp8_gmm_b200 import backend

    x, w, ws = torch.zeros(4, 32, dtype=torch.bfloat16, device=cuda), torch.zeros(2, 16, 32, dtype=torch.int8, device=cuda), torch.zeros(2, 16, device=cuda)
    wide = torch.zeros(2, 32, dtype=torch.bfloat16, device=cuda)
    bad = [
        (lambda: backend.int8_linear(x, w, [2, 3], ws), "sum|bad size"), (lambda: backend.int8_linear(x, w, [4], ws), "group size"),
        (lambda: backend.int8_linear(x, w, torch.tensor([2, 2], dtype=torch.int32, device=cuda), ws), "int64"),
        (lambda: backend.int8_linear(x[:, ::2], w, [2, 2], ws), "contiguous"), (lambda: backend.int8_linear(x.float(), w, [2, 2], ws), "bfloat16"),
        (lambda: backend.int8_linear(x, w.float(), [2, 2], ws), "int8"), (lambda: backend.int8_linear(x, w, [2, 2], ws.half()), "float32"),
        (lambda: backend.int8_linear(x, w[:, :, :16].contiguous(), [2, 2], ws), "contraction"),
        (lambda: backend.int8_linear(x, w, [2, 2], ws, activation="relu"), "activation"),
        (lambda: backend.int8_linear(x, w, [2, 2], ws, c=wide), "output"),
        (lambda: backend.quantize_rows_int8(x, torch.zeros(4, dtype=torch.int64, device=cuda)), "int32"),
        (lambda: backend.quantize_rows_int8(x.expand(4, 32)[0:1].expand(4, 32)), "overlap"),
        (lambda: backend.quantize_rows_int8(x[:, :31].contiguous(), activation="swiglu"), "gate"),
        (lambda: backend.int8_linear(x.clone().requires_grad_(True), w, [2, 2], ws), "no gradient"),
    ]
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()


# ------------------------------------------------------------------------------------------------ modules, streams, graphs
def _moe(experts, gate, tokens, E, top_k):
    from fp8_gmm_b200 import routing

    weights, selected = routing.topk(tokens @ gate, top_k)
    indices, bin_ids, bins, sizes = routing.indices_and_bins(selected, E)
    rows = experts(tokens, sizes, indices=indices, top_k=top_k)
    return routing.scatter(rows, indices, bin_ids, weights, bins, top_k)


@pytest.mark.parametrize("activation", ["gelu", "swiglu"])
def test_experts_behind_the_router(cuda, activation):
    """Int8GroupedMlp behind topk -> sort -> scatter equals the same experts evaluated one by one with sizes on the host;
    against the bf16 weights in 64 bits its error is that of 8-bit rounding (each operand off by at most half a code step:
    relative error per product about 1 / 127 / sqrt(12) * (top / rms), summed over two layers: below 5 % here)."""
    import fp8_gmm_b200 as fg
    from fp8_gmm_b200 import backend, routing

    E, top_k, H, F, T = 6, 2, 256, 272, 97
    torch.manual_seed(0)
    mlp = fg.GroupedMlp(H, F, E, torch.bfloat16, device=cuda, activation=activation)
    experts = fg.Int8GroupedMlp.from_mlp(mlp)
    tokens, gate = randn_bf16((T, H), 1).to(cuda), randn_bf16((H, E), 2).to(cuda)
    with torch.no_grad():
        out = _moe(experts, gate, tokens, E, top_k)
        weights, selected = routing.topk(tokens @ gate, top_k)
        indices, bin_ids, bins, sizes = routing.indices_and_bins(selected, E)
        rows = routing.gather(tokens, indices, bin_ids, bins, top_k)
        on_host = experts(rows, sizes.cpu())
        assert torch.equal(routing.scatter(on_host, indices, bin_ids, weights, bins, top_k), out)
        parts = rows.double().split(sizes.tolist())
        want = torch.cat([_act64(p @ mlp.fc1_weight[g].double().t(), activation) @ mlp.fc2_weight[g].double().t() for g, p in enumerate(parts)])
        assert float((on_host.double() - want).norm() / want.norm()) < 0.05
        lin = fg.GroupedLinear(H, 48, E, torch.bfloat16, device=cuda)
        q = fg.Int8GroupedLinear.from_linear(lin)
        got = q(tokens, sizes, indices=indices, top_k=top_k)
        assert torch.equal(got, backend.int8_linear(rows, q.weight, sizes.cpu(), q.weight_scales))
    backend.device_status()


def test_module_state_round_trip(cuda):
    import fp8_gmm_b200 as fg

    mlp = fg.GroupedMlp(64, 96, 3, torch.bfloat16, device=cuda, activation="swiglu")
    a = fg.Int8GroupedMlp.from_mlp(mlp)
    b = fg.Int8GroupedMlp(64, 96, 3, device=cuda, activation="swiglu")
    b.load_state_dict(a.state_dict())
    x = randn_bf16((10, 64), 5).to(cuda)
    assert torch.equal(a(x, [3, 0, 7]), b(x, [3, 0, 7]))


def test_captured_experts_follow_new_tokens_routes_and_weights(cuda):
    import fp8_gmm_b200 as fg

    E, top_k, H, F, T = 8, 2, 128, 144, 13
    torch.manual_seed(1)
    mlp = fg.GroupedMlp(H, F, E, torch.bfloat16, device=cuda, activation="swiglu")
    experts = fg.Int8GroupedMlp.from_mlp(mlp)
    tokens, gate = randn_bf16((T, H), 1).to(cuda), randn_bf16((H, E), 2).to(cuda)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _moe(experts, gate, tokens, E, top_k)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for _ in range(2):     # two graphs of the same layer, replayed at the same time on two streams
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(_moe(experts, gate, tokens, E, top_k))
            graphs.append(g)
        for seed in (3, 4):
            tokens.copy_(randn_bf16((T, H), seed))
            mlp.fc1_weight.mul_(1.01 if seed == 4 else 1.0)
            experts.refresh(mlp)
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream() for _ in graphs]
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    for _ in range(5):
                        g.replay()
            torch.cuda.synchronize()
            want = _moe(experts, gate, tokens, E, top_k)
            assert all(torch.equal(o, want) for o in outs)
    fg.backend.device_status()


def test_beside_the_fp8_product_on_another_stream(cuda):
    """Both persistent products own tensor memory and most of an SM's shared memory: launched at the same time they take turns."""
    from fp8_gmm_b200 import backend

    sizes, n, k = [300, 0, 77, 900], 512, 1024
    rows = sum(sizes)
    x = randn_bf16((rows, k), 1).to(cuda)
    w16 = randn_bf16((4, n, k), 2).to(cuda)
    w8, ws = backend.quantize_rows_int8(w16)
    f8 = [t.to(torch.float8_e4m3fn) for t in (x, w16)]
    one = torch.ones(4, device=cuda)
    torch.cuda.synchronize()
    want = backend.int8_linear(x, w8, sizes, ws), backend.fp8_gmm(f8[0], f8[1], sizes, (one, 1), (one, 1))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            got[0].append(backend.int8_linear(x, w8, sizes, ws))
        with torch.cuda.stream(streams[1]):
            got[1].append(backend.fp8_gmm(f8[0], f8[1], sizes, (one, 1), (one, 1)))
    torch.cuda.synchronize()
    backend.device_status()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_fewer_sms(cuda):
    """The product keeps to the SMs that the persistent GEMMs may use."""
    from fp8_gmm_b200 import backend

    w, ws = _codes((3, 1424, 512), 2).to(cuda), _scales((3, 1424), 3).to(cuda)
    x = randn_bf16((500, 512), 1).to(cuda)
    want = backend.int8_linear(x, w, [200, 0, 300], ws)
    try:
        for sms in (1, 2, 7, 100):
            backend.set_gemm_sm_limit(sms)
            assert torch.equal(backend.int8_linear(x, w, [200, 0, 300], ws), want)
            backend.device_status()
    finally:
        backend.set_gemm_sm_limit(0)


def test_calls_on_two_streams_at_once(cuda):
    from fp8_gmm_b200 import backend

    w, ws = _codes((4, 272, 512), 2).to(cuda), _scales((4, 272), 3).to(cuda)
    xs = [randn_bf16((m, 512), m).to(cuda) for m in (5, 333)]
    sizes = [[1, 0, 2, 2], [100, 33, 0, 200]]
    want = [backend.int8_linear(x, w, m, ws) for x, m in zip(xs, sizes)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(backend.int8_linear(xs[i], w, sizes[i], ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


@pytest.mark.parametrize("k", [16, 272, 512])
def test_many_tiles_per_cta_with_short_contractions(cuda, k):
    """Ten and more tiles per CTA pair whose products are done before the tile in front of them is written: the accumulators
    change hands at the pace of the stores.  Every bit, in each of several runs, and rows behind the last group untouched."""
    from fp8_gmm_b200 import backend

    sizes, n, spare = [1300, 0, 33, 2077, 257, 1], 16 * 1025, 7
    rows = sum(sizes)
    a, b = _codes((rows, k), k).to(cuda), _codes((len(sizes), n, k), k + 1).to(cuda)
    sa, sb = _scales((rows,), k + 2).to(cuda), _scales((len(sizes), n), k + 3).to(cuda)
    # |sum| <= 512 * 127^2 < 2^23: each partial sum is exact in the double product, and so is its conversion to fp32
    want = _product(a, b, sizes, sa, sb)
    for _ in range(3):
        c = torch.full((rows + spare, n), 3.0, dtype=torch.bfloat16, device=cuda)
        backend.int8_gmm(a, b, sizes, sa, sb, c=c[:rows])
        assert torch.equal(c[:rows], want) and bool((c[rows:] == 3.0).all())


@pytest.mark.parametrize("pitch,cols", [(128, 96), (144, 144), (96, 80), (75, 75), (81, 48), (16500, 16400)])
def test_codes_and_operands_with_a_row_pitch(cuda, pitch, cols):
    """Through the C interface: codes written with a pitch leave the gaps alone, a product reads them with it."""
    import ctypes

    from fp8_gmm_b200 import _lib, backend

    rows = 37
    x = randn_bf16((rows, cols), pitch).to(cuda)
    want_q, want_s = backend.quantize_rows_int8(x)
    codes = torch.full((rows, pitch), 99, dtype=torch.int8, device=cuda)
    scales = torch.empty(rows, device=cuda)
    q = _lib.QuantizeRowsArgs(in_=x.data_ptr(), in_ld=cols, top_k=1, in_rows=rows, rows=rows, cols=cols, activation=0,
                              codes=codes.data_ptr(), scales=scales.data_ptr(), codes_ld=pitch)
    _lib.check(_lib.lib.fp8gmm_quantize_rows_int8(ctypes.byref(q), torch.cuda.current_stream().cuda_stream), "quantise")
    assert torch.equal(codes[:, :cols], want_q) and bool((codes[:, cols:] == 99).all()) and torch.equal(scales, want_s)
    if pitch % 16 or cols % 16:
        return
    sizes, n = [30, 7], 48
    b, sb = _codes((2, n, cols), 1).to(cuda), _scales((2, n), 2).to(cuda)
    want = backend.int8_gmm(want_q, b, sizes, want_s, sb)
    c = torch.zeros(rows, n, dtype=torch.bfloat16, device=cuda)
    host_sizes = (ctypes.c_int64 * 2)(*sizes)
    g = _lib.Int8GemmArgs(a=codes.data_ptr(), b=b.data_ptr(), c=c.data_ptr(), a_scales=scales.data_ptr(), b_scales=sb.data_ptr(),
                          num_groups=2, rows=rows, n=n, k=cols, a_ld=pitch)
    g.m_sizes = ctypes.cast(host_sizes, ctypes.POINTER(ctypes.c_int64))
    _lib.check(_lib.lib.fp8gmm_int8_grouped_gemm(ctypes.byref(g), torch.cuda.current_stream().cuda_stream), "product")
    assert torch.equal(c, want)


@pytest.mark.parametrize("k", [16, 48, 112, 144, 240, 272, 400, 528, 1040])
@pytest.mark.parametrize("channels", [128, 256])
def test_contractions_that_end_inside_a_stage(cuda, any_variant, k, channels):
    """Every number of 32-byte steps and boxes in the last stage, wide and narrow tiles; what lies behind a row is the next one,
    with codes that would show in the sums."""
    from fp8_gmm_b200 import backend

    sizes, n = [5, 140, 0, 33], 208
    rows = sum(sizes)
    a, b = _codes((rows, k), k + 5), _codes((4, n, k), k + 6)
    sa, sb = _scales((rows,), 7), _scales((4, n), 8)
    backend.set_int8_variant(128, channels)
    got = backend.int8_gmm(a.to(cuda), b.to(cuda), sizes, sa.to(cuda), sb.to(cuda))
    assert torch.equal(got.cpu(), _product(a, b, sizes, sa, sb))


def test_group_sizes_in_every_form_on_the_host(cuda):
    """Lists, int32 and strided tensors give what a contiguous int64 tensor gives; other shapes are refused; no groups, no rows."""
    from fp8_gmm_b200 import backend

    sizes = [3, 0, 9]
    x = randn_bf16((12, 64), 1).to(cuda)
    w, ws = backend.quantize_rows_int8(randn_bf16((3, 32, 64), 2).to(cuda))
    want = backend.int8_linear(x, w, torch.tensor(sizes), ws)
    strided = torch.tensor([[3, 7], [0, 7], [9, 7]])[:, 0]
    for form in (sizes, tuple(sizes), torch.tensor(sizes, dtype=torch.int32), strided, torch.tensor(sizes, device=cuda)):
        assert torch.equal(backend.int8_linear(x, w, form, ws), want)
    for bad in (torch.tensor([sizes, sizes, sizes]), torch.tensor([12]), torch.tensor(12), [12]):
        with pytest.raises(RuntimeError, match="group size"):
            backend.int8_linear(x, w, bad, ws)
    for none in ([], torch.empty(0, dtype=torch.int64)):
        assert backend.int8_linear(x[:0], w[:0], none, ws[:0]).shape == (0, 32)
