"""The product in 8-bit integers (hrf_linear_int8) and the rounding of rows (hrf_quantize_rows_int8) against 64 bits.

Tolerances: U = 2^-24. The integer sum is exact; its conversion to fp32 and the two products by scales are three roundings, the bias one
more: 3 U |v| + U |y|, then half a step of y's type (fp16 below 2^-14: 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(m, n, k, seed=0):
    g = _gen(seed)
    x = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sx = (torch.rand(m, generator=g, device="cuda") + 0.5) / 100
    sw = (torch.rand(n, generator=g, device="cuda") + 0.5) / (100 * k ** 0.5)
    b = torch.randn(n, generator=g, device="cuda")
    return x, w, sx, sw, b


def _holds(y, x, w, sx, sw, b, relu):
    v = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    want = v if b is None else v + b.double()
    tol = 3 * U * v.abs() + U * want.abs()
    if relu:
        want = want.clamp(min=0.0)
    if y.dtype != F32:
        tol = tol * (1 + torch.finfo(y.dtype).eps) + torch.finfo(y.dtype).eps / 2 * want.abs() + (2.0 ** -25 if y.dtype == F16 else 0.0)
    bad = (y.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 257, 65), (1, 130, 2051), (1, 4096, 1024), (2, 3, 127), (3, 200, 136), (5, 64, 5000), (8, 1000, 128), (9, 33, 64), (15, 65, 129),
          (16, 16, 1000), (17, 48, 128), (29, 520, 640), (31, 130, 64), (32, 257, 256), (33, 31, 300), (48, 1024, 512), (63, 100, 64), (64, 2048, 1024),
          (65, 63, 200), (100, 1500, 384), (127, 129, 1000), (128, 128, 128), (129, 257, 64), (255, 255, 255), (256, 512, 1024), (300, 130, 2051), (513, 1030, 640),
          (1000, 64, 64), (1021, 515, 900), (4099, 64, 63), (5000, 17, 30), (5000, 190, 250), (4200, 200, 129), (70, 500, 200), (100, 520, 100), (20_000, 100, 64), (1300, 2050, 256), (3, 40, 20_001), (70, 30, 17_000), (2100, 2300, 1024), (1030, 4100, 600), (5000, 3000, 520)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_codes(m, n, k, dtype):
    from humanrf_amd import ops
    x, w, sx, sw, b = _case(m, n, k)
    if dtype == F32:
        _holds(ops.linear_int8(x, ops.Int8Weight(w, sw), x_scale=sx), x, w, sx, sw, None, False)
    y = ops.linear_int8(x, ops.Int8Weight(w, sw, b), x_scale=sx, relu=True, out_dtype=dtype)
    assert y.dtype == dtype and y.shape == (m, n)
    _holds(y, x, w, sx, sw, b, True)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_float_rows(m, n, k, dtype):
    """The codes are within half a step of x / scale -- the factor 127 / amax and the product are two roundings, the scale two of its own:
    4 U of at most 127 --, and the product of x is the product of its codes, to the bit."""
    from humanrf_amd import ops
    _, w, _, sw, b = _case(m, n, k)
    x = (torch.randn(m, k, generator=_gen(7), device="cuda") * torch.exp(torch.randn(m, 1, generator=_gen(8), device="cuda"))).to(dtype)
    q, s = ops.quantize_int8(x)
    assert q.shape == x.shape and s.shape == (m,)
    top = x.double().abs().amax(1)
    assert bool(((s.double() - top / 127).abs() <= 2 * U * top / 127).all())
    # (values that the products of fp16 and bf16 with the factor may leave just above 127 are 127: 127 (1 + 2 U) rounds to it)
    assert int(q.abs().max()) == 127
    assert bool(((q.double() - x.double() / s.double()[:, None]).abs() <= 0.5 + 127 * 6 * U).all())
    handle = ops.Int8Weight(w, sw, b)
    y = ops.linear_int8(x, handle, relu=True)
    assert y.dtype == dtype
    assert torch.equal(y, ops.linear_int8(q.contiguous(), handle, x_scale=s, relu=True, out_dtype=dtype))
    _holds(y, q, w, s, sw, b, True)


def test_the_largest_sums():
    """131071 products of -128 * -128 are 2^31 - 2^14, the most that fits."""
    from humanrf_amd import ops
    k = ops.INT8_MAX_INNER
    for m in (1, 3, 40, 200):
        x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((5, k), -128, dtype=torch.int8, device="cuda")
        w[1] = 127
        y = ops.linear_int8(x, ops.Int8Weight(w, torch.ones(5, device="cuda")), x_scale=torch.ones(m, device="cuda"))
        assert bool((y[:, 0] == float(torch.tensor(k * 16384.0))).all()) and bool((y[:, 1] == float(torch.tensor(-k * 16256.0))).all())


@pytest.mark.parametrize("m", [1, 4, 30, 200])
def test_rows_further_apart_and_unaligned(m):
    from humanrf_amd import ops
    n, k = 70, 130
    x, w, sx, sw, b = _case(m, n, k)
    for dtype in (torch.int8, F32, F16, BF16):
        for ld, at in ((k, 0), (k + 1, 1), (192, 3), (256, 16)):
            buf = torch.full((m * ld + 64,), 99, dtype=dtype, device="cuda")
            view = buf[at:at + m * ld].as_strided((m, k), (ld, 1), storage_offset=at)
            src = x if dtype == torch.int8 else (x.float() / 7).to(dtype)
            view.copy_(src)
            scale = sx if dtype == torch.int8 else None
            a = ops.linear_int8(view, ops.Int8Weight(w, sw, b), x_scale=scale)
            assert torch.equal(a, ops.linear_int8(src.contiguous(), ops.Int8Weight(w, sw, b), x_scale=scale))
    for ld, at in ((k + 1, 1), (256, 0), (256, 16), (192, 5)):
        buf = torch.full((n * ld + 64,), 99, dtype=torch.int8, device="cuda")
        view = buf.as_strided((n, k), (ld, 1), storage_offset=at)
        view.copy_(w)
        _holds(ops.linear_int8(x, ops.Int8Weight(view, sw, b), x_scale=sx), x, w, sx, sw, b, False)


def test_shapes_of_more_axes_and_of_none():
    from humanrf_amd import ops
    x, w, sx, sw, b = _case(24, 10, 33)
    h = ops.Int8Weight(w, sw, b)
    flat = ops.linear_int8(x, h, x_scale=sx)
    assert torch.equal(ops.linear_int8(x.view(2, 3, 4, 33), h, x_scale=sx.view(2, 3, 4)), flat.view(2, 3, 4, 10))
    assert torch.equal(ops.linear_int8(x[0], h, x_scale=sx[:1]), flat[0])
    assert ops.linear_int8(torch.zeros(0, 33, device="cuda"), h).shape == (0, 10)
    assert ops.linear_int8(torch.zeros(2, 0, 33, device="cuda"), h).shape == (2, 0, 10)
    q, s = ops.quantize_int8(torch.randn(2, 3, 33, device="cuda"))
    assert q.shape == (2, 3, 33) and s.shape == (2, 3)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    from humanrf_amd import ops
    for m in (1, 4, 20, 300):
        for dtype in (F32, F16, BF16):
            _, w, _, sw, b = _case(m, 40, 100)
            x = torch.randn(m, 100, device="cuda").to(dtype)
            h = ops.Int8Weight(w, sw, b)
            clean = ops.linear_int8(x, h)
            x[0] = 0.0
            assert torch.equal(ops.linear_int8(x, h)[0], b.to(dtype))
            for bad in (float("nan"), float("inf"), -float("inf")):
                x[0, 99] = bad
                y = ops.linear_int8(x, h)
                assert bool(torch.isnan(y[0]).all()) and torch.equal(y[1:], clean[1:])
                q, s = ops.quantize_int8(x)
                assert not bool(torch.isfinite(s[0])) and int(q[0].abs().max()) == 0
            x[0, 99] = torch.finfo(dtype).max
            assert bool(torch.isfinite(ops.linear_int8(x.float(), h)).all())
    tiny = torch.full((2, 8), 1e-40, device="cuda")
    assert int(ops.quantize_int8(tiny)[0].abs().max()) == 0


def test_refusals_on_the_device():
    from humanrf_amd import ops
    x, w, sx, sw, b = _case(4, 6, 32)
    h = ops.Int8Weight(w, sw, b)
    with pytest.raises(RuntimeError, match="values a row"):
        ops.linear_int8(torch.zeros(4, 31, device="cuda"), h)
    with pytest.raises(RuntimeError, match="x_scale"):
        ops.linear_int8(x, h)
    with pytest.raises(RuntimeError, match="x_scale"):
        ops.linear_int8(x.float(), h, x_scale=sx)
    with pytest.raises(RuntimeError, match="one x_scale"):
        ops.linear_int8(x, h, x_scale=sx[:3])
    with pytest.raises(RuntimeError, match="out_dtype"):
        ops.linear_int8(x, h, x_scale=sx, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="must be float32"):
        ops.linear_int8(x.double(), h)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear_int8(x.float().requires_grad_(), h)
    with pytest.raises(RuntimeError, match="not contiguous"):
        ops.linear_int8(torch.zeros(32, 4, device="cuda").t(), h)
    with pytest.raises(RuntimeError, match="one value per channel"):
        ops.Int8Weight(w, sx)
    with pytest.raises(RuntimeError, match="another shape"):
        ops.Int8Weight.from_packed(h.packed, 17, 32, torch.ones(17, device="cuda"))
    with pytest.raises(RuntimeError, match="1 to"):
        ops.quantize_int8(torch.zeros(2, 131072, device="cuda"))
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.quantize_int8(x)


def test_codes_at_any_address():
    """The C entry writes codes with any row stride, at any address, and zeros from the row's end to the stride."""
    from humanrf_amd import _lib, ops
    from humanrf_amd._lib import check, ptr, stream_ptr
    for dtype, kind in ((F32, 0), (F16, 1), (BF16, 2)):
        for m, k, ld, at in ((5, 77, 77, 1), (5, 77, 83, 3), (3, 20_001, 20_003, 5), (9, 130, 136, 8)):
            x = torch.randn(m, k, device="cuda").to(dtype)
            q, s = ops.quantize_int8(x)
            buf, scale = torch.full((m * ld + 64,), 99, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
            check(_lib.lib().hrf_quantize_rows_int8(ptr(x), kind, m, k, k, buf.data_ptr() + at, ld, ptr(scale), stream_ptr()))
            got = buf[at:at + m * ld].view(m, ld)
            assert torch.equal(got[:, :k], q) and int(got[:, k:].abs().sum()) == 0 and torch.equal(scale, s)
            assert bool((buf[:at] == 99).all()) and bool((buf[at + m * ld:] == 99).all())


def test_packed_codes():
    from humanrf_amd import ops
    for n, k in ((1, 1), (16, 64), (17, 65), (40, 300)):
        _, w, _, sw, _ = _case(1, n, k)
        p = ops.Int8Weight(w, sw).packed
        rows, cols = -(-n // 16) * 16, ops.int8_padded(k)
        full = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
        full[:n, :k] = w
        # block (i, j), byte 256 q + 16 t + b: row 16 i + t, code 64 j + 16 q + b
        assert torch.equal(p.view(rows // 16, cols // 64, 4, 16, 16), full.view(rows // 16, 16, cols // 64, 4, 16).permute(0, 2, 3, 1, 4))


def test_what_lies_around_stays():
    """y is written inside its rows and nowhere else; x ends its storage here."""
    from humanrf_amd import _lib, ops
    from humanrf_amd._lib import check, ptr, stream_ptr
    for m, n, k in ((1, 70, 128), (20, 70, 128), (200, 130, 256), (700, 50, 64), (5000, 50, 100)):
        x, w, sx, sw, b = _case(m, n, k)
        h = ops.Int8Weight(w, sw, b)
        y = torch.full((m + 2, n + 9), 55.0, dtype=F16, device="cuda")
        ws = torch.empty(_lib.lib().hrf_linear_int8_workspace_bytes(m, n, k), dtype=torch.uint8, device="cuda")
        check(_lib.lib().hrf_linear_int8(ptr(x), 3, k, ptr(sx), ptr(h.packed), ptr(sw), ptr(b), m, n, k, y[1].data_ptr(), 1, n + 9, 0, ptr(ws) or None,
                                         stream_ptr()))
        _holds(y[1:1 + m, :n].contiguous(), x, w, sx, sw, b, False)
        y[1:1 + m, :n] = 55.0
        assert bool((y == 55.0).all())


def test_offsets_past_32_bits():
    from humanrf_amd import ops
    g = _gen(1)
    m, k = 36_000, 65_536                                    # 2.4e9 bytes of codes
    x = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    rows = [0, 17, 32_767, 32_768, 35_999]
    for r in rows:
        x[r] = torch.randint(-128, 128, (k,), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (40, k), generator=g, device="cuda", dtype=torch.int8)
    sx, sw = torch.full((m,), 1e-3, device="cuda"), torch.full((40,), 1e-3, device="cuda")
    y = ops.linear_int8(x, ops.Int8Weight(w, sw), x_scale=sx)
    _holds(y[rows], x[rows], w, sx[rows], sw, None, False)
    assert float(y.abs().sum()) == float(y[rows].abs().sum())
    del x, y
    y = ops.linear_int8(w[:, :64].contiguous().repeat(1800, 1), ops.Int8Weight(torch.ones(62_000, 64, dtype=torch.int8, device="cuda"),
                        torch.ones(62_000, device="cuda")), x_scale=torch.ones(72_000, device="cuda"), out_dtype=BF16)    # 4.5e9 outputs
    want = w[:, :64].double().sum(1).to(BF16)
    for r in (0, 34_640, 71_999):
        assert bool((y[r] == want[r % 40]).all())


@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_products_on_another_stream(m):
    from humanrf_amd import ops
    _, w, _, sw, b = _case(m, 130, 200)
    h = ops.Int8Weight(w, sw, b)
    x = torch.randn(m, 200, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_int8(x, h)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = ops.linear_int8(x, h)
    for k in range(4):
        x.copy_(torch.randn(m, 200, generator=_gen(k), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.linear_int8(x, h))


def test_two_streams_at_once():
    """One handle, calls of every kind interleaved on two streams: each has workspaces of its own."""
    from humanrf_amd import ops
    _, w, _, sw, b = _case(1, 200, 300)
    h = ops.Int8Weight(w, sw, b)
    xs = [torch.randn(m, 300, generator=_gen(m), device="cuda") for m in (1, 7, 40, 300, 1000)]
    want = [ops.linear_int8(x, h) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for k in range(6):
        for s, out in zip(streams, got):
            with torch.cuda.stream(s):
                out += [ops.linear_int8(x, h) for x in (xs if k % 2 else xs[::-1])]
    torch.cuda.synchronize()
    for out in got:
        for k in range(6):
            part = out[5 * k:5 * k + 5]
            assert all(torch.equal(y, z) for y, z in zip(part if k % 2 else part[::-1], want))


# ------------------------------------------------------------------------------------------------ modules, and all of it together
def test_networks():
    """A layer of rounded weights and rows is off by half a step of each: sum_k |w| s_x / 2 + |x| s_w / 2 + s_x s_w / 4; a network's first
    layer's bound passes through the second as sum |w|."""
    from humanrf_amd.int8 import Int8Linear, Int8MLP
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(50, 200), torch.nn.ReLU(), torch.nn.Linear(200, 130), torch.nn.ReLU(), torch.nn.Linear(130, 7)).cuda()
    served = Int8MLP.from_sequential(net)
    assert [layer.relu for layer in served] == [True, True, False]
    x = torch.randn(300, 50, device="cuda")
    a, err = x.double(), torch.zeros(300, 50, dtype=torch.float64, device="cuda")
    for layer, relu in ((net[0], True), (net[2], True), (net[4], False)):
        w = layer.weight.detach().double()
        size = a.abs() + err
        sx, sw = size.amax(1, keepdim=True) / 127, w.abs().amax(1) / 127
        err = (err + sx / 2) @ w.abs().t() + size.sum(1, keepdim=True) * sw / 2 + 0.25 * w.shape[1] * sx * sw + 1e-5
        a = a @ w.t() + layer.bias.detach().double()
        a = a.clamp(min=0.0) if relu else a
    y = served(x)
    assert bool(((y.double() - a).abs() <= err * (1 + 1e-4)).all())
    again = Int8MLP.from_sequential(torch.nn.Sequential(*[type(m)(m.in_features, m.out_features).cuda() if isinstance(m, torch.nn.Linear) else m for m in net]))
    again.load_state_dict(served.state_dict())
    assert torch.equal(again(x), y)
    assert torch.equal(served.half()(x), y) and torch.equal(served.cpu().cuda()(x), y)
    one = Int8Linear.from_linear(net[4])
    assert one(torch.randn(2, 3, 130, device="cuda").bfloat16()).dtype == BF16


def test_the_field_s_density_network_in_8_bits():
    """HumanRF's own sigma_net through the flat parameters, next to the kernel that serves it in fp16."""
    from humanrf_amd import ops
    from humanrf_amd.int8 import Int8MLP
    g = _gen(3)
    params = torch.randn(64 * 32 + 16 * 64, generator=g, device="cuda") * 0.2
    x = torch.randn(5000, 32, generator=g, device="cuda").half()
    h, _ = ops.density_mlp_fwd(x, params[:2048].half().contiguous(), params[2048:].half().contiguous(), 1.0)
    y = Int8MLP.from_flat(params, (32, 64, 16))(x)
    assert y.shape == h.shape and y.dtype == h.dtype
    w1, w2 = params[:2048].view(64, 32).double(), params[2048:].view(16, 64).double()
    xd = x.double()
    s1x, s1w = xd.abs().amax(1, keepdim=True) / 127, w1.abs().amax(1) / 127
    e = (s1x / 2) @ w1.abs().sum(1)[None] + xd.abs().sum(1, keepdim=True) * s1w / 2 + 0.25 * 32 * s1x * s1w
    a = (xd @ w1.t()).clamp(min=0.0)
    e = e + 2.0 ** -11 * (a + e)
    s2x, s2w = (a + e).amax(1, keepdim=True) / 127, w2.abs().amax(1) / 127
    e = (e + s2x / 2) @ w2.abs().t() + (a + e).sum(1, keepdim=True) * s2w / 2 + 0.25 * 64 * s2x * s2w
    want = a @ w2.t()
    assert bool(((y.double() - want).abs() <= e + 2.0 ** -10 * (want.abs() + e)).all())


def test_trained_in_few_bits_and_served_in_few():
    """All of it as it is used together: a network's steps with clipping and 8-bit states, captured copies of its weights, then its layers
    rounded to 8 bits; the served network is within its rounding bound of the trained one."""
    from humanrf_amd.int8 import Int8MLP
    from humanrf_amd.optim import AdamW
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Linear(48, 96), torch.nn.ReLU(), torch.nn.Linear(96, 5)).cuda()
    copies = {p: torch.empty_like(p, dtype=F16) for p in net.parameters()}
    opt = AdamW(net.parameters(), lr=3e-3, eps=1e-8, state_bits=8, max_grad_norm=1.0, copies=copies)
    x = torch.randn(512, 48, device="cuda")
    y = torch.tanh(x[:, :5]) + x[:, 5:10] * x[:, 10:15]
    start = [p.detach().clone() for p in net.parameters()]
    for _ in range(30):
        (net(x) - y).square().mean().backward()
        opt.step(zero_grad=True)
    for p, q in zip(net.parameters(), start):
        assert bool(torch.isfinite(p).all()) and not torch.equal(p, q) and torch.equal(copies[p], p.detach().half())
    served = Int8MLP.from_sequential(net)(x)
    w1, w2 = net[0].weight.detach().double(), net[2].weight.detach().double()
    xd = x.double()
    s1x, s1w = xd.abs().amax(1, keepdim=True) / 127, w1.abs().amax(1) / 127
    e = (s1x / 2) @ w1.abs().sum(1)[None] + xd.abs().sum(1, keepdim=True) * s1w / 2 + 0.25 * 48 * s1x * s1w + 1e-5
    a = (xd @ w1.t() + net[0].bias.detach().double()).clamp(min=0.0)
    s2x, s2w = (a + e).amax(1, keepdim=True) / 127, w2.abs().amax(1) / 127
    e = (e + s2x / 2) @ w2.abs().t() + (a + e).sum(1, keepdim=True) * s2w / 2 + 0.25 * 96 * s2x * s2w + 1e-5
    assert bool(((served.double() - (a @ w2.t() + net[2].bias.detach().double())).abs() <= e * (1 + 1e-4)).all())
