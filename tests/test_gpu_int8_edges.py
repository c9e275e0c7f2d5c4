"""The 8-bit product's entry points in calls that other tests do not make: more rows than one axis of a launch counts, codes of several axes,
scales at the ends of fp32, modules whose buffers are replaced. Tolerances: U = 2^-24 is half a step of fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(m, k, seed):
    return torch.randint(-128, 128, (m, k), generator=_gen(seed), device="cuda", dtype=torch.int8)


# ------------------------------------------------------------------------------------------------ past 2^32 threads
@pytest.mark.parametrize("m,k,ld", [(2 ** 24 + 37, 3, 3), (2 ** 28 + 5, 3, 8)], ids=["a workgroup a row", "16 rows a workgroup"])
def test_rounding_more_rows_than_an_axis_counts(m, k, ld):
    from humanrf_amd import _lib
    from humanrf_amd._lib import check, ptr, stream_ptr
    x = torch.randn(m, k, generator=_gen(0), device="cuda", dtype=F16)
    q, s = torch.full((m, ld), 99, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    check(_lib.lib().hrf_quantize_rows_int8(ptr(x), 1, m, k, k, ptr(q), ld, ptr(s), stream_ptr()))
    for at in range(0, m, 2 ** 26):         # everything, in pieces
        part = slice(at, min(m, at + 2 ** 26))
        top = x[part].float().abs().amax(1).clamp(min=2.0 ** -119)
        assert torch.equal(s[part], top * (1.0 / 127.0))
        assert bool(((q[part, :k].float() * s[part, None] - x[part].float()).abs() <= s[part, None] * (0.5 + 127 * 6 * U)).all())
        assert int(q[part, k:].ne(0).sum()) == 0


def test_products_of_more_rows_than_an_axis_counts():
    """Codes of 130 a row are padded into the workspace, a workgroup a row."""
    from humanrf_amd import ops
    m, k, n = 2 ** 24 + 37, 130, 200
    x, w = _codes(m, k, 1), _codes(n, k, 2)
    sx, sw = torch.rand(m, generator=_gen(3), device="cuda") + 0.5, torch.rand(n, generator=_gen(4), device="cuda") + 0.5
    y = ops.linear_int8(x, ops.Int8Weight(w, sw), x_scale=sx, out_dtype=BF16)
    for rows in (slice(0, 300), slice(2 ** 22 - 100, 2 ** 22 + 100), slice(2 ** 24 - 100, m)):
        v = (x[rows].double() @ w.double().t()) * sx[rows].double()[:, None] * sw.double()
        assert bool(((y[rows].double() - v).abs() <= (2.0 ** -8 + 4 * U) * v.abs()).all())


def test_packing_more_rows_than_an_axis_counts():
    """One code a row, 64 bytes a row packed: more than 2^30 pieces of 16 bytes, which is where the second axis begins."""
    from humanrf_amd import ops
    n = 2 ** 28 + 16
    w = _codes(n, 1, 5)
    p = ops.Int8Weight(w, torch.ones(n, device="cuda")).packed.view(n // 16, 64, 16)
    assert torch.equal(p[:, :16, 0].reshape(n, 1), w)       # row t of a block: the 16 bytes at 16 t
    for at in range(0, n // 16, 2 ** 22):
        part = p[at:at + 2 ** 22]
        assert int(part[:, :, 1:].ne(0).sum()) == 0 and int(part[:, 16:].ne(0).sum()) == 0


# ------------------------------------------------------------------------------------------------ axes and strides
@pytest.mark.parametrize("k", [33, 64, 130, 300])
@pytest.mark.parametrize("lead", [(), (1,), (2, 3), (40, 5), (2, 0, 3)])
def test_what_rounding_gives_is_what_the_product_takes(lead, k):
    """Codes of x with any number of axes are rows further apart than they are long."""
    from humanrf_amd import ops
    h = ops.Int8Weight(_codes(20, k, 1), torch.rand(20, generator=_gen(2), device="cuda"))
    x = torch.randn(*lead, k, generator=_gen(3), device="cuda")
    q, s = ops.quantize_int8(x)
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    y = ops.linear_int8(q, h, x_scale=s)
    assert y.shape == (*lead, 20) and torch.equal(y, ops.linear_int8(x, h))


def test_strides_that_are_no_rows_are_refused():
    from humanrf_amd import ops
    h = ops.Int8Weight(_codes(4, 32, 1), torch.ones(4, device="cuda"))
    x = torch.zeros(6, 5, 32, device="cuda")
    assert ops.linear_int8(x[:, ::5], h).shape == (6, 1, 4)
    for bad in (x.transpose(0, 1), x[:, :3], x[:, :1].expand(6, 5, 32), torch.zeros(64, device="cuda")[::2], torch.zeros(2, 3, 64, device="cuda")[..., ::2]):
        with pytest.raises(RuntimeError, match="not contiguous"):
            ops.linear_int8(bad, h)
        with pytest.raises(RuntimeError, match="not contiguous"):
            ops.quantize_int8(bad)


# ------------------------------------------------------------------------------------------------ scales at the ends of fp32
@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (3, 40, 5000), (20, 70, 300), (60, 70, 300), (200, 300, 300), (300, 130, 2051), (2100, 2300, 1024), (700, 1100, 640),
                                   (100, 70, 64), (100, 70, 128), (5000, 100, 200)])
@pytest.mark.parametrize("token,channel", [(-125, -30), (-30, -125), (-80, -60), (-70, 100), (100, -70), (110, -126), (-149, 40), (40, -140), (-60, -60), (60, 60),
                                           (-64, 64), (0, 0)])
def test_products_of_scales_beyond_fp32(m, n, k, token, channel):
    """sx sw may lie below or above what fp32 holds while sum sx sw does not: the same bound as for all other products, 3 U |v|, and half a
    step of the smallest numbers, 2^-150, for the product and for the type each. Sums of zero stay zero where sx sw is beyond fp32."""
    from humanrf_amd import ops
    x, w = _codes(m, k, 1), _codes(n, k, 2)
    x[m // 2] = 0
    sx = torch.ldexp(torch.rand(m, generator=_gen(3), device="cuda") + 1.0, torch.tensor(token, device="cuda"))
    sw = torch.ldexp(torch.rand(n, generator=_gen(4), device="cuda") + 1.0, torch.tensor(channel, device="cuda"))
    y = ops.linear_int8(x, ops.Int8Weight(w, sw), x_scale=sx)
    v = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()
    fits = v.abs() < 2.0 ** 127
    assert bool(((y.double() - v).abs() <= 3 * U * v.abs() + 2.0 ** -149)[fits].all())
    assert not bool(torch.isnan(y).any()) and int(y[m // 2].ne(0).sum()) == 0
    big = ops.linear_int8(x, ops.Int8Weight(w, torch.full_like(sw, 2.0 ** 100)), x_scale=torch.full_like(sx, 2.0 ** 100))
    assert not bool(torch.isnan(big).any()) and int(big[m // 2].ne(0).sum()) == 0 and torch.equal(torch.isinf(big), v != 0)


@pytest.mark.parametrize("m,k", [(1, 300), (20, 300), (200, 300), (100, 64), (5000, 200)])
def test_tiny_rows(m, k):
    """Rows of 1e-34 against weights of 1e-3: products of 1e-36 in fp32, their scales' product below the normal numbers."""
    from humanrf_amd import ops
    x, w = torch.randn(m, k, generator=_gen(1), device="cuda") * 1e-34, torch.randn(70, k, generator=_gen(2), device="cuda") * 1e-3
    q, s = ops.quantize_int8(x)
    h = ops.Int8Weight.from_float(w)
    v = (q.double() @ ops.quantize_int8(w)[0].double().t()) * s.double()[:, None] * h.scale.double()
    y = ops.linear_int8(x, h)
    assert bool(((y.double() - v).abs() <= 3 * U * v.abs() + 2.0 ** -149).all())
    assert torch.equal(y, ops.linear_int8(q, h, x_scale=s))
