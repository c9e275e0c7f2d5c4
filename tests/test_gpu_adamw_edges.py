"""The AdamW step's entry points in calls that other tests do not make: captured steps next to eager ones of other gradients, loss scales without
a norm, values whose squares leave fp32, plans of empty tensors, optimizers that are copied. Tolerances: U = 2^-24 is half a step of fp32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LR = 1e-2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _params(sizes, seed):
    g = _gen(seed)
    return [torch.nn.Parameter(torch.randn(n, generator=g, device="cuda")) for n in sizes]


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_step_what_was_captured(bits):
    """A captured step, eager steps with gradient tensors of their own between its replays: the same bits as a twin that is given each
    gradient in turn."""
    from humanrf_amd.optim import AdamW
    sizes = (5000, 33)
    ps, qs = _params(sizes, 0), _params(sizes, 0)
    opt, twin = AdamW(ps, max_grad_norm=1.0, state_bits=bits), AdamW(qs, max_grad_norm=1.0, state_bits=bits)
    static = [torch.randn(n, generator=_gen(n), device="cuda") for n in sizes]
    given = lambda o, params, grads: ([setattr(p, "grad", g) for p, g in zip(params, grads)], o.step())  # noqa: E731
    given(opt, ps, static)
    given(twin, qs, static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    for k in range(4):
        graph.replay()
        given(twin, qs, [g.clone() for g in static])
        other = [torch.randn(n, generator=_gen(100 + k), device="cuda") for n in sizes]
        given(opt, ps, other)
        given(twin, qs, other)
        for p in ps:
            p.grad = None
        del other
        torch.full((50_000,), 1e9, device="cuda")           # what was freed is used by somebody else
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert opt._plan.steps.tolist() == twin._plan.steps.tolist() == [9, 9]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("through", ["optimizer", "plan"])
def test_a_loss_scale_alone_skips_what_overflowed(bits, through):
    from humanrf_amd import ops
    from humanrf_amd.optim import AdamW
    p, = _params((3000,), 1)
    scaler = ops.grad_scaler("cuda", init_scale=1024.0, growth_interval=2)
    if through == "optimizer":
        opt = AdamW([p], state_bits=bits)
        step = lambda: opt.step(scaler=scaler)  # noqa: E731
        plan = lambda: opt._plan  # noqa: E731
        p.grad = torch.randn(3000, device="cuda") * 1024.0
    else:
        grad = torch.randn(3000, device="cuda") * 1024.0
        made = ops.AdamWPlan([p.detach()], [grad], state_bits=bits)
        step = lambda: ops.adamw_multi(made, LR, scaler=scaler)  # noqa: E731
        plan = lambda: made  # noqa: E731
        p.grad = grad
    step()
    assert plan().steps.tolist() == [1] and ops.grad_scaler_state(scaler)["growth_tracker"] == 1
    old, states = p.detach().clone(), {k: v.clone() for k, v in plan().state.items()}
    for bad in (float("inf"), float("nan")):
        kept = p.grad[2999].clone()
        p.grad[2999] = bad
        step()
        p.grad[2999] = kept
        assert torch.equal(p, old) and all(torch.equal(v.float(), plan().state[k].float()) for k, v in states.items())
    assert plan().steps.tolist() == [1] and plan().skipped.item() == 2
    assert ops.grad_scaler_state(scaler)["scale"] == 256.0 and ops.grad_scaler_state(scaler)["growth_tracker"] == 0
    step()
    step()
    assert plan().steps.tolist() == [3] and ops.grad_scaler_state(scaler)["scale"] == 512.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e22, 1e25, 1e30, 3e38])
def test_gradients_whose_squares_leave_fp32(bits, size):
    """The second moment is inf, as in torch's own fp32 step: the first moment over it is 0, and the value decays and does nothing else. With
    8-bit states the scale of the block's roots is inf. In the next step the block's other codes, 0 times inf, are NaN, and so are their values;
    the code of the inf itself is the largest, 448 times inf is inf, and its value is divided by that again."""
    from humanrf_amd import ops
    p = torch.randn(600, generator=_gen(2), device="cuda")
    g = torch.randn(600, generator=_gen(3), device="cuda")
    g[300] = -size
    p0, want = p.clone(), torch.nn.Parameter(p.clone())
    want.grad = g.clone()
    torch.optim.AdamW([want], lr=LR, betas=(0.9, 0.99), eps=1e-15, weight_decay=0.1, foreach=False).step()
    plan = ops.AdamWPlan([p], [g], state_bits=bits)
    ops.adamw_multi(plan, LR, eps=1e-15, weight_decay=0.1)
    tol = 8 * U * p0.double().abs() + 40 * U * LR
    assert bool(((p.double() - want.detach().double()).abs() <= tol).all())
    assert float(p[300]) == float(p0[300] * torch.tensor(1.0 - LR * 0.1))
    if bits == 32:
        assert math.isinf(float(plan.state["exp_avg_sq"][300])) and int(torch.isfinite(plan.state["exp_avg_sq"]).sum()) == plan.numel - 1
        assert abs(float(plan.state["exp_avg"][300]) + 0.1 * size) <= 4 * U * 0.1 * size
    else:
        assert torch.isfinite(plan.state["exp_avg_root_scale"]).tolist() == [True, False, True]
    g[300] = 0.0
    ops.adamw_multi(plan, LR, eps=1e-15)
    gone = ~torch.isfinite(p)
    assert int(gone.sum()) == (0 if bits == 32 else 255) and (bits == 32 or (bool(gone[256:300].all()) and bool(gone[301:512].all())))


def test_a_root_that_is_not_finite_is_seen():
    """A second moment that is NaN, under a first moment that is finite: the root's scale, and the value, are NaN."""
    from humanrf_amd import ops
    for bits in (32, 8):
        p, g = torch.ones(600, device="cuda"), torch.ones(600, device="cuda")
        plan = ops.AdamWPlan([p], [g], state_bits=bits)
        plan.state["exp_avg_sq" if bits == 32 else "exp_avg_root_scale"][300 if bits == 32 else 1] = float("nan")
        ops.adamw_multi(plan, LR)
        gone = torch.isnan(p)
        assert int(gone.sum()) == (1 if bits == 32 else 256) and bool(gone[300])
        assert bits == 32 or torch.isnan(plan.state["exp_avg_root_scale"]).tolist() == [False, True, False]


@pytest.mark.parametrize("bits", [32, 8])
def test_second_moments_below_the_normal_numbers(bits):
    """Gradients of 1e-19 to 1e-21 under an eps that does not hide them: the root is that of the moment as fp32 holds it, v <= 2^-126 being a
    multiple of 2^-149. The update from that v is bounded as everywhere else: 24 U, and v itself by 8 U v + 2^-149."""
    from humanrf_amd import ops
    for size in (1e-19, 3e-20, 1e-20, 1e-21):
        g = torch.full((512,), size, device="cuda") * (1.0 + torch.arange(512, device="cuda") % 7 / 8)
        p = torch.zeros(512, device="cuda")
        plan = ops.AdamWPlan([p], [g], state_bits=bits)
        ops.adamw_multi(plan, LR, betas=(0.9, 0.99), eps=1e-36)
        v = g.double().square() * 0.01
        held = torch.round(v * 2.0 ** 149) * 2.0 ** -149
        if bits == 32:
            held = plan.state["exp_avg_sq"][:512].double()
            assert bool(((held - v).abs() <= 8 * U * v + 2.0 ** -149).all())
        root = held.sqrt()
        want = -LR / 0.1 * (0.1 * g.double()) / (root / 0.1)
        spread = 0.0 if bits == 32 else 2.0 ** -149 / held       # (half a multiple up or down in v, halved by the root, and as much again)
        assert bool(((p.double() - want).abs() <= (24 * U + spread) * want.abs()).all()), size
        if bits == 8:
            top = root.view(2, 256).amax(1)
            assert bool(((plan.state["exp_avg_root_scale"].double() * 448 - top).abs() <= (8 * U + 2.0 ** -149 / held.min()) * top).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_empty_tensors_alone_have_step_counts(bits):
    """As an empty tensor among others has: steps, skipped steps and the loss scale go on."""
    from humanrf_amd import ops
    empty = lambda: torch.zeros(0, device="cuda")  # noqa: E731
    plan = ops.AdamWPlan([empty(), empty()], [empty(), None], state_bits=bits)
    ops.adamw_multi(plan, LR)
    ops.adamw_multi(plan, LR, norm=ops.grad_norm_multi(plan), max_norm=1.0)
    assert plan.steps.tolist() == [2, 0] and plan.skipped.item() == 0
    scaler = ops.grad_scaler("cuda", init_scale=64.0, growth_interval=1)
    ops.adamw_multi(plan, LR, flags=torch.ones(1, dtype=torch.int32, device="cuda"), scaler=scaler)
    assert plan.steps.tolist() == [2, 0] and plan.skipped.item() == 1 and ops.grad_scaler_state(scaler)["scale"] == 32.0
    ops.adamw_multi(plan, LR, scaler=scaler, zero_grad=True)
    assert plan.steps.tolist() == [3, 0] and ops.grad_scaler_state(scaler)["scale"] == 64.0
    mixed = ops.AdamWPlan([empty(), torch.zeros(5, device="cuda")], [empty(), torch.ones(5, device="cuda")], state_bits=bits)
    ops.adamw_multi(mixed, LR)
    assert mixed.steps.tolist() == [1, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_of_the_optimizer_goes_on_as_the_original(bits):
    import copy
    from humanrf_amd.optim import AdamW
    ps = _params((3000, 7), 5)
    opt = AdamW(ps, state_bits=bits, max_grad_norm=1.0, seed=11)

    def step(o, params, seed):
        for p in params:
            p.grad = torch.randn(p.shape, generator=_gen(seed), device="cuda")
        o.step()
    step(opt, ps, 0)
    qs, other = copy.deepcopy((ps, opt))
    for k in range(1, 4):
        step(opt, ps, k)
        step(other, qs, k)
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(ps, qs))
    assert all(torch.equal(v.float(), other._plan.state[n].float()) for n, v in opt._plan.state.items())
    assert other._plan.steps.tolist() == [4, 4]


@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_storage_is_stepped_and_other_lengths_are_not(bits):
    from humanrf_amd.optim import AdamW
    ps, qs = _params((3000, 40), 7), _params((3000, 40), 7)
    opt, twin = AdamW(ps, state_bits=bits), AdamW(qs, state_bits=bits)

    def step(o, params, k):
        for p in params:
            p.grad = torch.randn(p.shape, generator=_gen(k), device="cuda")
        o.step()
    for k in range(4):
        step(opt, ps, k)
        step(twin, qs, k)
        ps[0].data = ps[0].data.clone()         # the same values somewhere else
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    held = ps[0].data
    ps[0].grad = None
    ps[0].data = held[:2999].clone()
    ps[0].grad = torch.ones(2999, device="cuda")
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="2999 values"):
        opt.step()
    assert all(torch.equal(p, b) for p, b in zip(ps, before)) and opt._plan.steps.tolist() == [4, 4]
    ps[0].grad = None
    ps[0].data = held
    step(opt, ps, 9)
    step(twin, qs, 9)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("keep", [True, False])
def test_a_device_lr_and_a_captured_step_of_the_optimizer(keep):
    """lr in one tensor on the device: replays read what a schedule wrote into it."""
    from humanrf_amd.optim import AdamW
    lr = torch.tensor([LR], device="cuda")
    ps, qs = _params((500,), 8), _params((500,), 8)
    opt, twin = AdamW(ps, lr=lr), AdamW(qs, lr=LR)
    ps[0].grad, qs[0].grad = torch.ones(500, device="cuda"), torch.ones(500, device="cuda")
    opt.step()
    twin.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(zero_grad=not keep)
    for k in range(3):
        now = float(torch.tensor(LR / (k + 2)))
        lr.fill_(now)
        twin.param_groups[0]["lr"] = now
        ps[0].grad.fill_(1.0 + k)
        qs[0].grad.fill_(1.0 + k)
        graph.replay()
        twin.step(zero_grad=not keep)
        torch.cuda.synchronize()
        # (the first step had lr in fp32 here and in fp64 there; every step rounds the value once)
        assert bool(((ps[0].double() - qs[0].double()).abs() <= 4 * U * (qs[0].double().abs() + LR)).all())
        assert torch.equal(ps[0].grad, qs[0].grad)
