"""The AdamW step over many tensors (hrf_adamw_multi), the gradients' norm (hrf_grad_norm_multi) and humanrf_amd.optim.AdamW against a
plain implementation in 64 bits.

Tolerances: U = 2^-24 is half a step of fp32. A parameter's value goes through 2 roundings of its own (decay, subtraction) and 2 of the
constants (decay, step size), the update m / den * step_size through 3 of m, 4 of v (halved by the root), root, den twice, quotient,
product and the gradient's factor, its constants among them: 8 U |p| + 24 U |update| bounds their sum. m: 6 U (|m| + |g|) covers
(g - m)(1 - b1) + m with G and the constant rounded; v is a sum of positive terms: 8 U v. A 16-bit parameter is off by half a step of
its type more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 256
B1, B2, EPS, LR, WD = 0.9, 0.99, 1e-15, 1e-2, 0.1
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tensors(sizes, dtype, seed, scale=1.0, offset=0):
    """One tensor of each length, `offset` values behind an aligned address, with a guard of 77s on both sides."""
    g = _gen(seed)
    out, guards = [], []
    for n in sizes:
        buf = torch.full((n + 64,), 77.0, dtype=dtype, device="cuda")
        at = 32 + offset
        buf[at:at + n] = (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)
        out.append(buf[at:at + n])
        guards.append((buf, at, n))
    return out, guards


def _guards_stand(guards):
    return all(bool((b[:at] == 77).all()) and bool((b[at + n:] == 77).all()) for b, at, n in guards)


def _state(sizes, bits, seed):
    """Mid-training states in the plan's flat layout, and their values in 64 bits."""
    g = _gen(seed)
    total = sum(-(-n // BLOCK) * BLOCK for n in sizes)
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    at = 0
    for n in sizes:
        inside[at:at + n] = True
        at += -(-n // BLOCK) * BLOCK
    m = torch.where(inside, torch.randn(total, generator=g, device="cuda") * 0.3, 0.0)
    v = torch.where(inside, torch.rand(total, generator=g, device="cuda") + 0.01, 0.0)
    if bits == 32:
        return {"exp_avg": m, "exp_avg_sq": v}
    st = {}
    for name, x in (("exp_avg", m), ("exp_avg_root", v.sqrt())):
        scale = (x.view(-1, BLOCK).abs().amax(1) / 448.0).clamp(min=1e-12)
        st[name] = (x.view(-1, BLOCK) / scale[:, None]).reshape(-1).to(torch.float8_e4m3fn)
        st[name + "_scale"] = scale
    return st


def _decode(st, bits):
    st = {k: v.double() for k, v in st.items()}
    if bits == 32:
        return st["exp_avg"], st["exp_avg_sq"]
    up = lambda s: s.repeat_interleave(BLOCK)  # noqa: E731
    return st["exp_avg"] * up(st["exp_avg_scale"]), (st["exp_avg_root"] * up(st["exp_avg_root_scale"])) ** 2


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _codes_follow(x, tol, code, scale, noise, keep):
    """Every e4m3 code is the value below or above |x| 448 / amax that its random bits choose. fp32 has x off by `tol`, the block's largest
    by top_tol, the scale by 3 U more (the constant 1 / 448, the product, the largest's own place). t is off by tol 448 / amax, by
    t top_tol / amax and by 4 U t (quotient, product, the sum with the lowest binade's begin): where t / gap + noise is nearer than that
    to a whole number the two may choose differently, by one gap."""
    b, bt = x.view(-1, BLOCK), tol.view(-1, BLOCK)
    top, top_tol = b.abs().amax(1), bt.amax(1)
    assert bool(((scale.double() - top / 448.0).abs() <= (top_tol + 3 * U * top) / 448.0 + 1e-45).all())
    per = torch.where(top > 0, 448.0 / top.clamp(min=1e-300), 0.0)[:, None]
    t = (b.abs() * per).reshape(-1).clamp(max=448.0)
    t_tol = (bt * per + b.abs() * per * per * top_tol[:, None] / 448.0).reshape(-1) + 4 * U * (t + 2.0 ** -6)
    gap = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
    y = t / gap + noise
    want = torch.floor(y) * gap
    if keep:
        want = torch.where((t > 0) & (want == 0), 2.0 ** -9, want)
    want = want.clamp(max=448.0)
    got = code.double().abs()
    near = (y - torch.round(y)).abs() <= t_tol / gap
    assert bool(((got == want) | (near & ((got - want).abs() <= 2 * gap))).all())
    assert bool(((x.abs() <= tol) | (torch.sign(code.double()) * torch.sign(x) >= 0)).all())


def _check(sizes, bits, p0, g, p, copies, before, plan, factor, t, pdt):
    m0, v0 = _decode(before, bits)
    for k, n in enumerate(sizes):
        s = slice(plan.offsets[k], plan.offsets[k] + n)
        G = g[k].double() * factor
        m = m0[s] + (G - m0[s]) * (1 - B1)
        v = v0[s] * B2 + (1 - B2) * G * G
        upd = LR / (1 - B1 ** t) * m / ((v / (1 - B2 ** t)).sqrt() + EPS)
        want = p0[k].double() * (1 - LR * WD) - upd
        tol = 8 * U * p0[k].double().abs() + 24 * U * upd.abs()
        m_tol = 6 * U * (m0[s].abs() + G.abs())
        tol = tol + 4 * LR / (1 - B1 ** t) * m_tol / ((v / (1 - B2 ** t)).sqrt() + EPS)      # m's own cancellation goes into the update
        half = torch.finfo(pdt).eps / 2 if pdt != F32 else 0.0
        got = p[k].double()
        assert bool(((got - want).abs() <= tol * (1 + 2 * half) + half * want.abs() + (2.0 ** -25 if pdt == F16 else 0.0)).all()), (k, n)
        if copies[k] is not None:
            assert torch.equal(copies[k], p[k].to(copies[k].dtype))
        if bits == 32:
            assert bool(((plan.state["exp_avg"][s].double() - m).abs() <= m_tol).all())
            assert bool(((plan.state["exp_avg_sq"][s].double() - v).abs() <= 8 * U * v).all())
    if bits == 8:
        full = plan.numel
        gm = torch.zeros(full, dtype=torch.float64, device="cuda")
        for k, n in enumerate(sizes):
            gm[plan.offsets[k]:plan.offsets[k] + n] = g[k].double() * factor
        m = m0 + (gm - m0) * (1 - B1)
        r = (v0 * B2 + (1 - B2) * gm * gm).sqrt()
        h = _mix(torch.arange(full, device="cuda") ^ _mix(plan.seed ^ _mix(t)))
        _codes_follow(m, 6 * U * (m0.abs() + gm.abs()), plan.state["exp_avg"], plan.state["exp_avg_scale"], (h & 0xFFFF).double() / 65536, False)
        _codes_follow(r, 6 * U * r, plan.state["exp_avg_root"], plan.state["exp_avg_root_scale"], (h >> 16).double() / 65536, True)


SIZES = (1, 255, 256, 257, 2047, 0, 2048, 2049, 7, 10_001)
TYPES = [(F32, F32, None), (F32, F32, F16), (F32, BF16, BF16), (F32, F16, None), (BF16, BF16, None), (BF16, F32, None), (F16, F16, None),
         (F16, F32, None), (F16, BF16, None), (BF16, F16, None)]


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("pdt,gdt,cdt", TYPES, ids=lambda d: str(d).replace("torch.", ""))
@pytest.mark.parametrize("bits", [32, 8])
def test_one_step(bits, pdt, gdt, cdt, offset):
    from humanrf_amd import ops
    p, pg = _tensors(SIZES, pdt, 1, 0.5, offset)
    g, gg = _tensors(SIZES, gdt, 2, 1.0, offset)
    c, cg = _tensors(SIZES, cdt, 3, 1.0, offset) if cdt is not None else ([None] * len(SIZES), [])
    st = _state(SIZES, bits, 4)
    before = {k: v.clone() for k, v in st.items()}
    p0, g0 = [x.clone() for x in p], [x.clone() for x in g]
    plan = ops.AdamWPlan(p, g, copies=c, state_bits=bits, state=st, step=6, seed=123)
    norm = ops.grad_norm_multi(plan, grad_scale=4.0)
    want = math.sqrt(sum(float(x.double().square().sum()) for x in g)) / 4.0
    assert abs(float(norm) - want) <= 2 * U * want
    max_norm = 0.5 * want
    ops.adamw_multi(plan, LR, betas=(B1, B2), eps=EPS, weight_decay=WD, norm=norm, max_norm=max_norm, grad_scale=4.0)
    torch.cuda.synchronize()
    factor = min(1.0, max_norm / (float(norm) + 1e-6)) / 4.0
    _check(SIZES, bits, p0, g0, p, c, before, plan, factor, 7, pdt)
    assert all(torch.equal(a, b) for a, b in zip(g, g0))
    assert plan.steps.tolist() == [7] * len(SIZES) and plan.skipped.item() == 0
    assert _guards_stand(pg + gg + cg)
    # a second step from where the first one ended, gradients zeroed behind it
    before, p0 = {k: v.clone() for k, v in plan.state.items()}, [x.clone() for x in p]
    ops.adamw_multi(plan, LR, betas=(B1, B2), eps=EPS, weight_decay=WD, zero_grad=True)
    _check(SIZES, bits, p0, g0, p, c, before, plan, 1.0, 8, pdt)
    assert all(float(x.float().abs().sum()) == 0.0 for x in g) and _guards_stand(pg + gg + cg)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_a_gradient_stay(bits):
    from humanrf_amd import ops
    sizes = (300, 5000, 40)
    p, _ = _tensors(sizes, F32, 1)
    g, _ = _tensors(sizes, F32, 2)
    plan = ops.AdamWPlan(p, [g[0], None, g[2]], state_bits=bits, state=_state(sizes, bits, 3))
    old = p[1].clone()
    s = slice(plan.offsets[1], plan.offsets[2])
    codes = plan.state["exp_avg"][s].clone()
    for _ in range(3):
        ops.adamw_multi(plan, LR, weight_decay=WD)
    assert torch.equal(p[1], old) and torch.equal(plan.state["exp_avg"][s].float(), codes.float())
    assert plan.steps.tolist() == [3, 0, 3]
    want = math.sqrt(sum(float(x.double().square().sum()) for x in (g[0], g[2])))
    assert abs(float(ops.grad_norm_multi(plan)) - want) <= 2 * U * want
    plan.set_grads(g)
    ops.adamw_multi(plan, LR, weight_decay=WD)
    assert plan.steps.tolist() == [4, 1, 4] and not torch.equal(p[1], old)


@pytest.mark.parametrize("bits", [32, 8])
def test_factors_per_tensor(bits):
    from humanrf_amd import ops
    sizes = (3000, 3000)
    p, _ = _tensors(sizes, F32, 1)
    g, _ = _tensors(sizes, F32, 2)
    q, p0 = [x.clone() for x in p], [x.clone() for x in p]
    plan = ops.AdamWPlan(p, g, state_bits=bits, seed=9, lr_scales=[0.5, 1.0], decay_scales=[0.0, 2.0])
    ops.adamw_multi(plan, LR, weight_decay=WD)
    for k, (lr, wd) in enumerate(((LR * 0.5, 0.0), (LR, 2 * WD))):
        G = g[k].double()
        upd = lr * G / (G.abs() + EPS)            # first step from zero: m / (1 - b1) over sqrt(v / (1 - b2)) is the sign
        tol = 8 * U * p0[k].double().abs() + 40 * U * lr
        assert bool(((p[k].double() - (p0[k].double() * (1 - lr * wd) - upd)).abs() <= tol).all())
    del q


def test_plans_refuse_on_the_device():
    from humanrf_amd import ops
    buf, g = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
    for p in ([buf, buf], [buf[:60], buf[59:]]):
        with pytest.raises(RuntimeError, match="share memory"):
            ops.AdamWPlan(p)
    with pytest.raises(RuntimeError, match="share memory"):
        ops.AdamWPlan([buf[:50], buf[50:]], [g[:50], g[:50]])
    with pytest.raises(RuntimeError, match="length and device"):
        ops.AdamWPlan([buf], [g[:99]])
    with pytest.raises(RuntimeError, match="must be float32"):
        ops.AdamWPlan([buf.double()])
    with pytest.raises(RuntimeError, match="gradients must be"):
        ops.AdamWPlan([buf], [g.double()])
    with pytest.raises(RuntimeError, match="copies of float32"):
        ops.AdamWPlan([buf.half()], copies=[g.half()])
    with pytest.raises(RuntimeError, match="one gradient"):
        ops.AdamWPlan([buf], [g, g])
    with pytest.raises(RuntimeError, match="one finite factor"):
        ops.AdamWPlan([buf], lr_scales=[-1.0])
    plan = ops.AdamWPlan([buf], [g])
    with pytest.raises(RuntimeError, match="state must hold"):
        ops.AdamWPlan([buf], [g], state_bits=8, state=plan.state)
    with pytest.raises(RuntimeError, match="must have 256 values"):
        ops.AdamWPlan([buf], [g], state={k: v[:128] for k, v in plan.state.items()})
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.adamw_multi(plan, LR, max_norm=1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.adamw_multi(plan, LR, norm=ops.grad_norm_multi(plan), max_norm=0.0)
    with pytest.raises(RuntimeError, match="not on the expected device"):
        ops.adamw_multi(plan, LR, norm=torch.zeros(1))
    with pytest.raises(RuntimeError, match="eps"):
        ops.adamw_multi(plan, LR, eps=0.0)
    with pytest.raises(RuntimeError, match="hyper"):
        ops.adamw_multi(plan, LR, betas=(1.0, 0.9))


def test_the_norm():
    from humanrf_amd import ops
    p, _ = _tensors((70_001, 3, 999_999), F32, 1)
    g, _ = _tensors((70_001, 3, 999_999), F32, 2)
    g[1].copy_(torch.tensor([1e30, -2e30, 0.0]))           # squares beyond fp32
    plan = ops.AdamWPlan(p, g)
    a = ops.grad_norm_multi(plan)
    want = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    assert abs(float(a) - want) <= 2 * U * want
    assert all(torch.equal(a, ops.grad_norm_multi(plan)) for _ in range(3))
    g[2][-1] = float("inf")
    assert float(ops.grad_norm_multi(plan)) == float("inf")
    g[0][5] = float("nan")
    assert math.isnan(float(ops.grad_norm_multi(plan)))
    empty = ops.AdamWPlan([torch.zeros(0, device="cuda")], [torch.zeros(0, device="cuda")])
    assert float(ops.grad_norm_multi(empty)) == 0.0
    ops.adamw_multi(empty, LR)
    none = ops.AdamWPlan(p)
    assert float(ops.grad_norm_multi(none)) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_skipped_steps_and_the_loss_scale(bits):
    from humanrf_amd import ops
    p, _ = _tensors((5000,), F32, 1)
    g, _ = _tensors((5000,), F32, 2, 1024.0)
    plan = ops.AdamWPlan(p, g, state_bits=bits, state=_state((5000,), bits, 3))
    scaler = ops.grad_scaler("cuda", init_scale=1024.0, growth_interval=2)
    twin = ops.AdamWPlan([p[0].clone()], [g[0] / 1024.0], state_bits=bits, state={k: v.clone() for k, v in plan.state.items()})
    norm = ops.grad_norm_multi(plan, scaler=scaler)
    ops.adamw_multi(plan, LR, weight_decay=WD, norm=norm, scaler=scaler)
    ops.adamw_multi(twin, LR, weight_decay=WD)              # a power of two: the same gradients to the bit
    assert torch.equal(p[0], twin.params[0]) and torch.equal(plan.state["exp_avg"].float(), twin.state["exp_avg"].float())
    old, states = p[0].clone(), {k: v.clone() for k, v in plan.state.items()}
    g[0][17] = float("nan")
    norm = ops.grad_norm_multi(plan, scaler=scaler)
    ops.adamw_multi(plan, LR, weight_decay=WD, norm=norm, scaler=scaler, zero_grad=True)
    assert torch.equal(p[0], old) and all(torch.equal(v.float(), plan.state[k].float()) for k, v in states.items())
    assert float(g[0].abs().sum()) == 0.0 and plan.steps.tolist() == [1] and plan.skipped.item() == 1
    assert ops.grad_scaler_state(scaler)["scale"] == 512.0 and ops.grad_scaler_state(scaler)["growth_tracker"] == 0
    flags = torch.tensor([1], dtype=torch.int32, device="cuda")
    ops.adamw_multi(plan, LR, flags=flags)
    assert torch.equal(p[0], old) and plan.skipped.item() == 2
    for _ in range(2):
        ops.adamw_multi(plan, LR, flags=torch.zeros_like(flags), scaler=scaler)
    assert ops.grad_scaler_state(scaler)["scale"] == 1024.0 and plan.steps.tolist() == [3]


def test_what_is_not_finite_is_seen():
    """Without a norm a NaN gradient goes where it goes in torch's step: into the value; with 8-bit states its block of 256 is lost and
    no other."""
    from humanrf_amd import ops
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            p, _ = _tensors((1000,), F32, 1)
            g, _ = _tensors((1000,), F32, 2)
            g[0][300] = bad
            plan = ops.AdamWPlan(p, g, state_bits=bits, state=_state((1000,), bits, 3))
            ops.adamw_multi(plan, LR)
            assert not math.isfinite(float(p[0][300])) and int(torch.isfinite(p[0]).sum()) == 999
            g[0][300] = 0.0
            ops.adamw_multi(plan, LR)
            gone = ~torch.isfinite(p[0])
            assert bool(gone[300]) and int(gone.sum()) == (1 if bits == 32 else 256)
            assert bits == 32 or bool(gone[256:512].all())


def test_moments_without_gradients_decay():
    """e4m3 codes rounded to nearest would keep 0.9 m = m for every code whose neighbour is over 10 % away, and 0.995 r for all of them.
    Rounded at random the mean decays as in fp32. Each rounding of a value x to a gap d has a variance of d^2 / 4 at most, d <= x / 8:
    a relative variance of 1 / 256 a step, (1 + 1/256)^40 - 1 = 0.17 over 40 steps, over 2^16 values (their own spread, E[x^4]^(1/2) /
    E[x^2] < 2, included) a standard deviation of the mean's under 0.0033: 2 % is 6 of them. What lies below the smallest normal code
    (2^-6 / 448 of the block's largest) adds less than 1e-4 of the mean."""
    from humanrf_amd import ops
    n = 1 << 16
    p = torch.zeros(n, device="cuda")
    st = _state((n,), 8, 5)
    m0, v0 = _decode(st, 8)
    plan = ops.AdamWPlan([p], [torch.zeros(n, device="cuda")], state_bits=8, state={k: v.clone() for k, v in st.items()}, seed=3)
    for _ in range(40):
        ops.adamw_multi(plan, 0.0, betas=(0.9, 0.99))
    m, v = _decode(plan.state, 8)
    assert abs(float(m.abs().mean() / m0.abs().mean()) / 0.9 ** 40 - 1) < 0.02
    assert abs(float(v.sqrt().mean() / v0.sqrt().mean()) / 0.99 ** 20 - 1) < 0.02
    assert bool((v[:n] > 0).all())
    assert float(p.abs().sum()) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_the_same_call_gives_the_same_bits(bits):
    from humanrf_amd import ops

    def go(seed):
        p, _ = _tensors((100_000, 77), F32, 1)
        g, _ = _tensors((100_000, 77), F32, 2)
        plan = ops.AdamWPlan(p, g, state_bits=bits, seed=seed)
        for _ in range(4):
            ops.adamw_multi(plan, LR, norm=ops.grad_norm_multi(plan), max_norm=1.0)
        return torch.cat([x for x in p] + [v.float() for v in plan.state.values()])
    a = go(1)
    assert torch.equal(a, go(1))
    assert bits == 32 or not torch.equal(a, go(2))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_on_another_stream(bits):
    """Norm and step in a graph, lr on the device, replayed with eager work of its own between: the same bits as an eager twin. Two
    graphs over two plans replay in turn."""
    from humanrf_amd import ops
    plans, twins, lrs = [], [], []
    for k in range(2):
        p, _ = _tensors((70_000, 33), F32, 10 + k)
        g, _ = _tensors((70_000, 33), F32, 20 + k)
        plans.append(ops.AdamWPlan(p, g, state_bits=bits, seed=k))
        twins.append(ops.AdamWPlan([x.clone() for x in p], g, state_bits=bits, seed=k))
        lrs.append(torch.tensor([LR], device="cuda"))

    def step(plan, lr):
        ops.adamw_multi(plan, lr, weight_decay=WD, norm=ops.grad_norm_multi(plan), max_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for plan, lr in zip(plans, lrs):
            step(plan, lr)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(plan, lr)
            graphs.append(graph)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capture"):
        dead = torch.cuda.CUDAGraph()
        with torch.cuda.graph(dead):
            plans[0].set_grads(plans[0].grads)
    for k in range(2):
        step(twins[k], lrs[k])
    for it in range(5):
        for k in range(2):
            lrs[k].fill_(LR / (it + 1))
            graphs[k].replay()
            step(twins[k], lrs[k])
            torch.randn(1000, device="cuda").sum()
        torch.cuda.synchronize()
        for plan, twin in zip(plans, twins):
            assert all(torch.equal(a, b) for a, b in zip(plan.params, twin.params))
            assert all(torch.equal(v.float(), twin.state[n].float()) for n, v in plan.state.items())
            assert plan.steps.tolist() == twin.steps.tolist() == [it + 2] * 2


def test_two_plans_on_two_streams_at_once():
    from humanrf_amd import ops

    def make(k):
        p, _ = _tensors((300_000, 5), F32, 30 + k)
        g, _ = _tensors((300_000, 5), F32, 40 + k)
        return ops.AdamWPlan(p, g, state_bits=8, seed=k)
    plans, twins, streams = [make(0), make(1)], [make(0), make(1)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(8):
        for plan, s in zip(plans, streams):
            with torch.cuda.stream(s):
                ops.adamw_multi(plan, LR, norm=ops.grad_norm_multi(plan), max_norm=1.0)
    torch.cuda.synchronize()
    for plan, twin in zip(plans, twins):
        for _ in range(8):
            ops.adamw_multi(twin, LR, norm=ops.grad_norm_multi(twin), max_norm=1.0)
        assert all(torch.equal(a, b) for a, b in zip(plan.params, twin.params)) and plan.steps.tolist() == [8, 8]


def test_offsets_past_32_bits():
    """A tensor of 2^31 + 777 values: its last block, and one at 2^31, are stepped as any other."""
    from humanrf_amd import ops
    n = 2 ** 31 + 777
    p = torch.zeros(n, dtype=BF16, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    for at in (0, 2 ** 31 - 1, 2 ** 31 + 5, n - 1):
        g[at] = -2.0
    plan = ops.AdamWPlan([p], [g], state_bits=8)
    assert abs(float(ops.grad_norm_multi(plan)) - 4.0) <= 4 * U * 4.0
    ops.adamw_multi(plan, LR)
    # the first step is lr * sign, rounded to bf16
    want = torch.tensor(LR).to(BF16)
    for at in (0, 2 ** 31 - 1, 2 ** 31 + 5, n - 1):
        assert abs(float(p[at]) - float(want)) <= 2 ** -8 * LR
        assert float(plan.state["exp_avg"][at].float()) == -448.0
        assert abs(float(plan.state["exp_avg_scale"][at // 256]) - 2.0 * 0.1 / 448) < 1e-8
    assert int((p != 0).sum()) == 4
    assert int((plan.state["exp_avg"].view(torch.uint8) != 0).sum()) == 4


# ------------------------------------------------------------------------------------------------ the optimizer object
def _net(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(24, 65), torch.nn.ReLU(), torch.nn.Linear(65, 3)).cuda()


def _loss(net, x, y):
    return (net(x) - y).square().mean()


@pytest.mark.parametrize("keep", [True, False])
def test_the_optimizer_follows_torch_s_adamw(keep):
    """Six steps of both from the same start, the gradients given (not recomputed, so that rounding does not feed back): every step adds
    less than the bound of one step. Groups with their own lr and decay, a schedule, clipping."""
    from humanrf_amd.optim import AdamW
    net = _net()
    ref = [torch.nn.Parameter(p.detach().double()) for p in net.parameters()]
    group = lambda ps: [{"params": ps[:2], "lr": 3e-3}, {"params": ps[2:], "weight_decay": 0.0}]  # noqa: E731
    ours = AdamW(group(list(net.parameters())), lr=1e-2, eps=1e-8, weight_decay=0.05, max_grad_norm=0.7)
    theirs = torch.optim.AdamW(group(ref), lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05, foreach=False)
    sched = [torch.optim.lr_scheduler.LambdaLR(o, lambda k: 0.8 ** k) for o in (ours, theirs)]
    for k in range(6):
        g = _gen(k)
        for p, q in zip(net.parameters(), ref):
            d = torch.randn(p.shape, generator=g, device="cuda")
            if keep and p.grad is not None:
                p.grad.copy_(d)
            else:
                p.grad = d
            q.grad = d.double()
        if k == 3:
            list(net.parameters())[1].grad, ref[1].grad = None, None
        torch.nn.utils.clip_grad_norm_(ref, 0.7)
        versions = [p._version for p in net.parameters()]
        ours.step()
        theirs.step()
        for s in sched:
            s.step()
        for p, q, ver in zip(net.parameters(), ref, versions):
            assert bool(((p.double() - q).abs() <= (k + 1) * (8 * U * q.abs() + 100 * U * 1e-2)).all())
            assert (p._version > ver) == (p.grad is not None)
        if k == 3:
            list(net.parameters())[1].grad = torch.zeros(65, device="cuda")


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints(bits):
    from humanrf_amd.optim import AdamW

    def run(opt, net, first, count):
        for k in range(first, first + count):
            g = _gen(100 + k)
            for p in net.parameters():
                p.grad = torch.randn(p.shape, generator=g, device="cuda")
            opt.step()
    a, b = _net(), _net()
    oa, ob = AdamW(a.parameters(), state_bits=bits), AdamW(b.parameters(), state_bits=bits)
    run(oa, a, 0, 6)
    run(ob, b, 0, 3)
    saved = ob.state_dict()
    c = _net(1)
    c.load_state_dict(b.state_dict())
    oc = AdamW(c.parameters(), lr=1.0, state_bits=bits)
    oc.load_state_dict(saved)
    run(oc, c, 3, 3)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), c.parameters()))
    with pytest.raises(RuntimeError, match="other bits|another shape"):
        AdamW(_net().parameters(), state_bits=40 - bits).load_state_dict(saved)
    if bits == 32:      # the layout is torch's
        ref = torch.optim.AdamW(_net().parameters())
        ref.load_state_dict(saved)
        od = AdamW(_net().parameters())
        od.load_state_dict(ref.state_dict())
        assert torch.equal(od._plan.state["exp_avg_sq"], ob._plan.state["exp_avg_sq"]) and od._plan.steps.tolist() == [3] * 4


def test_a_captured_training_step():
    """Forward, backward, norm and step captured and replayed, with eager steps of a twin between; an eager autograd graph over copies of
    the parameters is alive all the while and is differentiated after the replays."""
    from humanrf_amd.optim import AdamW
    net, twin = _net(), _net()
    x, y = torch.randn(128, 24, device="cuda"), torch.randn(128, 3, device="cuda")
    opt, ref = AdamW(net.parameters(), max_grad_norm=1.0, state_bits=8), AdamW(twin.parameters(), max_grad_norm=1.0, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _loss(net, x, y).backward()
        opt.step(zero_grad=True)
    torch.cuda.current_stream().wait_stream(side)
    _loss(twin, x, y).backward()
    ref.step(zero_grad=True)
    torch.cuda.synchronize()
    w = [p.detach().clone().requires_grad_() for p in net.parameters()]
    alive = sum((q * q).sum() for q in w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _loss(net, x, y).backward()
        opt.step(zero_grad=True)
    for _ in range(4):
        graph.replay()
        _loss(twin, x, y).backward()
        ref.step(zero_grad=True)
        torch.cuda.synchronize()
    alive.backward()
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters()))
    assert opt._plan.steps.tolist() == [5] * 4


def test_the_field_model_trains_with_it():
    """HumanRF.get_params under the optimizer, 8-bit states: the 16-bit copies that the kernels read are renewed after the step."""
    from humanrf_amd.optim import AdamW
    from humanrf_amd.scene_representation import HumanRF
    frames = tuple(range(12))
    model = HumanRF(density_scale=100, sorted_frame_numbers=frames, n_features_per_level=2, log2_hashmap_size=12, n_levels=16,
                    coarsest_resolution=16, finest_resolution=256, geometry_feature_dim=15, n_neurons=64, n_hidden_layers_density=1,
                    n_hidden_layers_color=2, sh_degree=4, segment_sizes=(12,), camera_embedding_dim=0, device="cuda")
    opt = AdamW(model.get_params(1e-2), state_bits=8, weight_decay=0.0)
    g = _gen(0)
    xyzt = torch.rand(500, 4, generator=g, device="cuda")
    seg = torch.zeros(500, dtype=torch.int32, device="cuda")
    dirs = torch.randn(500, 3, generator=g, device="cuda")
    idx = torch.arange(500, device="cuda")
    sigma0 = model.field(xyzt, seg, dirs, idx, None, True)[0].detach()
    for _ in range(3):
        sigma, rgb, _ = model.field(xyzt, seg, dirs, idx, None, True)
        (sigma.mean() * 1e-2 + rgb.square().mean()).backward()
        opt.step(zero_grad=True)
    sigma1 = model.field(xyzt, seg, dirs, idx, None, True)[0].detach()
    assert torch.equal(model._tables_h[:model.table_params.numel()], model.table_params.detach().half())
    assert torch.isfinite(sigma1).all() and not torch.equal(sigma0, sigma1)
