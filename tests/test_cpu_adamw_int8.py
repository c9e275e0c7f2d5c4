"""What the AdamW step and the 8-bit integer product refuse, on the CPU: through the C entry points (arguments are looked at before
anything is launched) and through the Python wrappers."""
import pytest
import torch

FAKE = 1 << 20      # an address that is never followed: every call below is refused before a launch


def _adamw(lib, **change):
    a = dict(tensors=FAKE, tile_tensor=FAKE, num_tiles=1, count=1, state_bits=32, exp_avg=FAKE, second=FAKE, exp_avg_scale=None,
             second_scale=None, ctl=FAKE, lr=1e-2, lr_dev=None, beta1=0.9, beta2=0.99, eps=1e-15, weight_decay=0.0, grad_scale=1.0,
             max_norm=0.0, norm=None, flags=None, scaler=None, seed=0, zero_grad=0, stream=None)
    a.update(change)
    return lib.hrf_adamw_multi(*a.values())


@pytest.mark.parametrize("change,said", [
    (dict(num_tiles=-1), b"counts"), (dict(count=-1), b"counts"), (dict(state_bits=16), b"8 or in 32"),
    (dict(lr=-1.0), b"hyper"), (dict(lr=float("nan")), b"hyper"), (dict(beta1=1.0), b"hyper"), (dict(beta2=-0.1), b"hyper"),
    (dict(weight_decay=float("inf")), b"hyper"), (dict(weight_decay=-1.0), b"hyper"), (dict(grad_scale=0.0), b"hyper"),
    (dict(eps=0.0), b"eps"), (dict(eps=1e-40), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(max_norm=1.0), b"norm"),
    (dict(tensors=None), b"NULL"), (dict(tile_tensor=None), b"NULL"), (dict(exp_avg=None), b"NULL"), (dict(second=None), b"NULL"),
    (dict(ctl=None), b"NULL"), (dict(exp_avg=FAKE + 4), b"multiples of 16"), (dict(second=FAKE + 8), b"multiples of 16"), (dict(state_bits=8), b"scales"), (dict(state_bits=8, exp_avg_scale=FAKE), b"scales"),
])
def test_the_step_refuses(change, said):
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert _adamw(lib, **change) != 0
    assert b"hrf_adamw_multi" in lib.hrf_last_error() and said in lib.hrf_last_error()


def test_a_step_over_nothing_is_nothing():
    from humanrf_amd import _lib
    assert _adamw(_lib.lib(), num_tiles=0, tensors=None, tile_tensor=None, exp_avg=None, second=None, ctl=None) == 0


@pytest.mark.parametrize("args", [
    (FAKE, FAKE, -1, 1.0, None, FAKE, FAKE, None), (FAKE, FAKE, 1, 0.0, None, FAKE, FAKE, None),
    (FAKE, FAKE, 1, float("nan"), None, FAKE, FAKE, None), (None, FAKE, 1, 1.0, None, FAKE, FAKE, None),
    (FAKE, None, 1, 1.0, None, FAKE, FAKE, None), (FAKE, FAKE, 1, 1.0, None, None, FAKE, None),
    (FAKE, FAKE, 1, 1.0, None, FAKE, None, None),
])
def test_the_norm_refuses(args):
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert lib.hrf_grad_norm_multi(*args) != 0
    assert b"hrf_grad_norm_multi" in lib.hrf_last_error()


def test_the_descriptor_has_the_header_s_layout():
    """The rows that the plan writes are hrf_adamw_tensor as a C compiler lays it out."""
    from humanrf_amd import ops
    D = ops._ADAMW_TENSOR
    assert D.itemsize == 64
    assert [D.fields[f][1] for f in ("param", "grad", "copy", "n", "base", "first_tile", "kind", "lr_scale", "decay_scale")] == \
        [0, 8, 16, 24, 32, 40, 44, 48, 56]


def test_plans_refuse():
    from humanrf_amd import ops
    p = torch.zeros(8)
    with pytest.raises(RuntimeError, match="no parameters"):
        ops.AdamWPlan([])
    with pytest.raises(RuntimeError, match="state_bits"):
        ops.AdamWPlan([p], state_bits=4)
    with pytest.raises(RuntimeError, match="negative"):
        ops.AdamWPlan([p], step=-1)
    with pytest.raises(RuntimeError, match="not on the expected device"):
        ops.AdamWPlan([p])
    with pytest.raises(RuntimeError, match="not contiguous"):
        ops.AdamWPlan([torch.zeros(4, 4).t()])


def test_the_optimizer_refuses():
    from humanrf_amd.optim import AdamW
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="max_grad_norm"):
        AdamW([p], max_grad_norm=0.0)
    with pytest.raises(ValueError, match="betas and eps"):
        AdamW([{"params": [p]}, {"params": [q], "eps": 1e-8}])
    with pytest.raises(ValueError, match="tensor"):
        AdamW([{"params": [p], "lr": torch.tensor(1.0)}, {"params": [q], "lr": torch.tensor(1.0)}])
    opt = AdamW([p])
    assert opt.step() is None           # no gradients: nothing to do, and nothing is built
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="not on the expected device"):
        opt.step()


# ------------------------------------------------------------------------------------------------ 8-bit integer product
def _linear(lib, **change):
    a = dict(x=FAKE, x_type=2, ldx=100, x_scale=None, w=FAKE, w_scale=FAKE, bias=None, rows=4, cols=8, inner=100, y=FAKE, y_type=0, ldy=8, relu=0,
             workspace=FAKE, stream=None)
    a.update(change)
    return lib.hrf_linear_int8(*a.values())


@pytest.mark.parametrize("change,said", [
    (dict(x_type=4), b"x_type"), (dict(x_type=-1), b"x_type"), (dict(y_type=3), b"y_type"), (dict(y_type=-1), b"y_type"),
    (dict(rows=-1), b"sizes"), (dict(cols=-1), b"sizes"), (dict(rows=2 ** 31), b"sizes"), (dict(cols=64 * 65535 + 1, ldy=1 << 40), b"sizes"),
    (dict(inner=0), b"sizes"), (dict(inner=131072, ldx=131072), b"sizes"), (dict(rows=2 ** 31 - 300, cols=1 << 20, ldy=1 << 20), b"tiles"),
    (dict(x=None), b"NULL"), (dict(w=None), b"NULL"), (dict(y=None), b"NULL"), (dict(w_scale=None), b"NULL"), (dict(x_type=3), b"NULL"),
    (dict(ldx=99), b"stride"), (dict(ldy=7), b"stride"), (dict(w=FAKE + 8), b"multiple of 16"), (dict(workspace=None), b"workspace"),
    (dict(workspace=FAKE + 8), b"workspace"),
])
def test_the_product_refuses(change, said):
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert _linear(lib, **change) != 0
    assert b"hrf_linear_int8" in lib.hrf_last_error() and said in lib.hrf_last_error()


def test_products_of_nothing_are_nothing():
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert _linear(lib, rows=0, x=None, y=None) == 0 and _linear(lib, cols=0, w=None, y=None) == 0
    assert lib.hrf_quantize_rows_int8(None, 0, 0, 5, 5, None, 64, None, None) == 0
    assert lib.hrf_int8_pack(None, 0, 5, 5, None, None) == 0


@pytest.mark.parametrize("args", [
    (FAKE, 3, 2, 5, 5, FAKE, 64, FAKE, None), (FAKE, -1, 2, 5, 5, FAKE, 64, FAKE, None), (FAKE, 0, -1, 5, 5, FAKE, 64, FAKE, None),
    (FAKE, 0, 2, 0, 5, FAKE, 64, FAKE, None), (FAKE, 0, 2, 131072, 131072, FAKE, 131072, FAKE, None), (None, 0, 2, 5, 5, FAKE, 64, FAKE, None),
    (FAKE, 0, 2, 5, 5, None, 64, FAKE, None), (FAKE, 0, 2, 5, 5, FAKE, 64, None, None), (FAKE, 0, 2, 5, 4, FAKE, 64, FAKE, None),
    (FAKE, 0, 2, 5, 5, FAKE, 4, FAKE, None), (FAKE, 0, 2, 5, 5, FAKE, 131073, FAKE, None),
])
def test_rounding_rows_refuses(args):
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert lib.hrf_quantize_rows_int8(*args) != 0
    assert b"hrf_quantize_rows_int8" in lib.hrf_last_error()


@pytest.mark.parametrize("args", [
    (FAKE, -1, 5, 5, FAKE, None), (FAKE, 2, 0, 5, FAKE, None), (FAKE, 2, 131072, 131072, FAKE, None), (None, 2, 5, 5, FAKE, None),
    (FAKE, 2, 5, 5, None, None), (FAKE, 2, 5, 4, FAKE, None), (FAKE, 2, 5, 5, FAKE + 4, None),
])
def test_packing_refuses(args):
    from humanrf_amd import _lib
    lib = _lib.lib()
    assert lib.hrf_int8_pack(*args) != 0
    assert b"hrf_int8_pack" in lib.hrf_last_error()


def test_padded_lengths():
    from humanrf_amd import _lib, ops
    lib = _lib.lib()
    assert [lib.hrf_int8_padded(k) for k in (0, 131072)] == [-1, -1]
    for k in (1, 63, 64, 65, 127, 128, 129, 2051, 131071):
        assert lib.hrf_int8_padded(k) == ops.int8_padded(k) >= k
        assert lib.hrf_int8_packed_bytes(17, k) == 32 * ops.int8_padded(k)
    assert lib.hrf_int8_packed_bytes(-1, 5) == -1 and lib.hrf_int8_packed_bytes(5, 0) == -1
    assert lib.hrf_linear_int8_workspace_bytes(-1, 8, 100) == 0 and lib.hrf_linear_int8_workspace_bytes(4, 8, 100) == 16 * 128 + 16
    assert lib.hrf_linear_int8_workspace_bytes(10_000, 64, 64) == 0


def test_the_wrappers_refuse():
    from humanrf_amd import int8, ops
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="not on the expected device"):
        ops.quantize_int8(x)
    with pytest.raises(RuntimeError, match="int8 matrix"):
        ops.Int8Weight(x, torch.ones(3))
    with pytest.raises(RuntimeError, match="must be a matrix"):
        ops.Int8Weight.from_float(x[0])
    with pytest.raises(NotImplementedError, match="Sigmoid"):
        int8.Int8MLP.from_sequential(torch.nn.Sequential(torch.nn.Sigmoid()))
    with pytest.raises(RuntimeError, match="parameters"):
        int8.Int8MLP.from_flat(x, (4, 4))
