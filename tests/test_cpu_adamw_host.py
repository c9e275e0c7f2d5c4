"""What humanrf_amd.optim.AdamW and ops.AdamWPlan put into the descriptors that the kernels follow, on the CPU: the library's calls are
recorded instead of made, so that nothing is launched and a wrong address or length is seen without anybody following it."""
import contextlib

import numpy as np
import pytest
import torch


class Recorder:
    """Stands for the library: keeps what each call was given, the descriptors as they were at that moment."""

    def __init__(self):
        self.calls = []

    def hrf_adamw_workspace_bytes(self):
        return 64

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args, self.rows(args[0])))
            return 0
        return call

    def rows(self, address):
        from humanrf_amd import ops
        import ctypes
        raw = (ctypes.c_uint8 * (self.count * ops._ADAMW_TENSOR.itemsize)).from_address(address)
        return np.frombuffer(bytes(raw), dtype=ops._ADAMW_TENSOR)


@pytest.fixture
def host(monkeypatch):
    from humanrf_amd import _lib, ops
    lib, chk = Recorder(), ops._chk
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_chk", lambda t, name, dtype=None, cuda=True: chk(t, name, dtype, False))
    monkeypatch.setattr(ops, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "stream_of", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    return lib


def _stepped(host, tensors, **kw):
    """An optimizer over parameters of these values that has taken one step."""
    from humanrf_amd.optim import AdamW
    params = [torch.nn.Parameter(t) for t in tensors]
    host.count = len(params)
    for p in params:
        p.grad = torch.ones_like(p)
    opt = AdamW(params, **kw)
    opt.step()
    return opt, params


@pytest.mark.parametrize("length", [1000, 99_999, 100_001])
def test_a_parameter_of_another_length_is_refused(host, length):
    opt, (p, q) = _stepped(host, [torch.zeros(100_000), torch.zeros(7)])
    assert host.calls[-1][2]["n"].tolist() == [100_000, 7]
    n = len(host.calls)
    p.grad = None
    p.data = torch.zeros(length)
    p.grad = torch.ones(length)
    for _ in range(2):
        with pytest.raises(RuntimeError, match=f"{length} values"):
            opt.step()
    assert len(host.calls) == n         # nothing was launched


def test_a_parameter_cut_short_where_it_lies_is_refused(host):
    opt, (p,) = _stepped(host, [torch.zeros(100)])
    n, g = len(host.calls), p.grad
    p.grad = None
    p.data = p.data[:60]
    p.grad = g[:60]                     # both at the addresses that they had
    with pytest.raises(RuntimeError, match="60 values"):
        opt.step()
    assert len(host.calls) == n


def test_storage_of_the_same_length_is_taken_over(host):
    opt, (p, q) = _stepped(host, [torch.zeros(4, 10), torch.zeros(7)])
    p.data = torch.full((5, 8), 2.0)
    p.grad = torch.ones(5, 8, dtype=torch.float32)
    opt.step()
    rows = host.calls[-1][2]
    assert rows["param"].tolist() == [p.data_ptr(), q.data_ptr()] and rows["grad"].tolist() == [p.grad.data_ptr(), q.grad.data_ptr()]
    assert rows["n"].tolist() == [40, 7] and rows["kind"].tolist() == [0, 0]
    p.grad = None
    p.data = p.data.bfloat16()          # a type that the step knows: the descriptor says so
    p.grad = torch.ones(5, 8, dtype=torch.bfloat16)
    opt.step()
    assert host.calls[-1][2]["kind"].tolist() == [2 | 2 << 2, 0] and host.calls[-1][2]["param"][0] == p.data_ptr()


def test_replaced_storage_is_checked_as_the_first_was(host):
    shared = torch.zeros(20)
    for bad, said in ((torch.zeros(10, dtype=torch.float64), "must be float32"), (shared[:10], "share memory"),
                      (torch.zeros(2, 5).t().contiguous().t().view(2, 5), "not contiguous")):
        opt, (p, q) = _stepped(host, [torch.zeros(2, 5) if said == "not contiguous" else torch.zeros(10), shared[5:15]])
        n = len(host.calls)
        p.grad = None
        p.data = bad
        p.grad = torch.ones_like(bad)
        with pytest.raises(RuntimeError, match=said):
            opt.step()
        assert len(host.calls) == n
    p = torch.nn.Parameter(torch.zeros(10))
    from humanrf_amd.optim import AdamW
    host.count, p.grad = 1, torch.zeros(10)
    opt = AdamW([p], copies={p: torch.zeros(10, dtype=torch.float16)})
    opt.step()
    p.grad = None
    p.data = p.data.half()
    p.grad = torch.zeros(10, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="copies of float32"):
        opt.step()


@pytest.mark.parametrize("other", [lambda b: b.view(16, 8).t(), lambda b: b[:1].expand(8, 16)], ids=["transposed", "broadcast"])
def test_a_gradient_of_other_strides_at_the_same_address_is_refused(host, other):
    opt, (p,) = _stepped(host, [torch.zeros(8, 16)])
    buf = torch.zeros(128)
    p.grad = buf.view(8, 16)
    opt.step()
    n = len(host.calls)
    p.grad = other(buf)
    assert p.grad.data_ptr() == buf.data_ptr() and p.grad.shape == (8, 16)
    with pytest.raises(RuntimeError, match="not contiguous: gradient"):
        opt.step(zero_grad=True)
    assert len(host.calls) == n
    p.grad = buf.view(8, 16)
    opt.step()
    assert len(host.calls) == n + 1


def test_plans_take_tensors_of_their_own_lengths_only(host):
    from humanrf_amd import ops
    host.count = 2
    p, g = [torch.zeros(300), torch.zeros(5)], [torch.zeros(300), torch.zeros(5)]
    plan = ops.AdamWPlan(p, g)
    with pytest.raises(RuntimeError, match="as many parameters"):
        plan.set_tensors(p[:1], g[:1])
    with pytest.raises(RuntimeError, match="299 values"):
        plan.set_tensors([p[0][:299], p[1]], [g[0][:299], g[1]])
    with pytest.raises(RuntimeError, match="length and device"):
        plan.set_tensors(p, [g[0][:299], g[1]])
    assert plan.params is not None and [x.numel() for x in plan.params] == [300, 5]
    q = [torch.ones(300), torch.ones(5)]
    plan.set_tensors(q, [None, g[1]])
    ops.adamw_multi(plan, 1e-2)
    rows = host.calls[-1][2]
    assert rows["param"].tolist() == [q[0].data_ptr(), q[1].data_ptr()] and rows["grad"].tolist() == [0, g[1].data_ptr()]


def test_a_captured_step_keeps_its_descriptors(host, monkeypatch):
    """A graph holds the address of the descriptors. Eager steps with other gradients write theirs elsewhere, so that replays neither step with
    gradients that they were not captured with nor follow addresses of tensors that are gone."""
    import gc
    import weakref
    opt, (p, q) = _stepped(host, [torch.zeros(3000), torch.zeros(7)], max_grad_norm=1.0)
    held = weakref.ref(p.grad)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step(zero_grad=True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    captured, rows = host.calls[-1][1][:2], host.calls[-1][2]
    for _ in range(3):
        p.grad, q.grad = torch.ones(3000), None
        opt.step()
        _, args, now = host.calls[-1]
        assert args[0] != captured[0] and now["grad"].tolist() == [p.grad.data_ptr(), 0]
        assert args[1] == args[0] + now.nbytes
    gc.collect()
    assert held() is not None and np.array_equal(host.rows(captured[0]), rows)
    # eager steps alone rewrite the descriptors that they have
    assert len({args[0] for _, args, _ in host.calls[-3:]}) == 1


def test_a_loss_scale_alone_has_the_norm_taken(host):
    """Without a norm and without flags nothing would see an overflowed gradient, and the scale would only grow."""
    from humanrf_amd import ops
    opt, (p,) = _stepped(host, [torch.zeros(50)])
    scaler, flags = ops.grad_scaler("cpu"), torch.zeros(1, dtype=torch.int32)
    del host.calls[:]
    opt.step(scaler=scaler, grad_scale=2.0)
    (norm, norm_args, _), (step, args, _) = host.calls
    assert norm == "hrf_grad_norm_multi" and norm_args[3:5] == (2.0, scaler.data_ptr()) and step == "hrf_adamw_multi"
    assert args[-6] == norm_args[6] and args[-4] == scaler.data_ptr()
    del host.calls[:]
    opt.step(scaler=scaler, flags=flags)
    assert [c[0] for c in host.calls] == ["hrf_adamw_multi"] and host.calls[0][1][-6:-3] == (None, flags.data_ptr(), scaler.data_ptr())


def test_the_entry_refuses_a_loss_scale_alone():
    from humanrf_amd import _lib
    lib, fake = _lib.lib(), 1 << 20      # an address that is never followed
    args = [fake, fake, 1, 1, 32, fake, fake, None, None, fake, 1e-2, None, 0.9, 0.99, 1e-15, 0.0, 1.0, 0.0, None, None, fake, 0, 0, None]
    assert lib.hrf_adamw_multi(*args) != 0 and b"loss scale" in lib.hrf_last_error()


def test_sparse_gradients_are_refused_by_name(host):
    opt, (p, q) = _stepped(host, [torch.zeros(4, 4), torch.zeros(7)])
    n = len(host.calls)
    q.grad = None
    p.grad = torch.eye(4).to_sparse()
    with pytest.raises(RuntimeError, match="sparse gradients"):
        opt.step()
    assert len(host.calls) == n


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_and_pickles_of_an_optimizer(host, how, bits):
    """A copy steps its own parameters, from the states and step counts that it was made with."""
    import copy
    import io
    net = torch.nn.Linear(20, 5)
    from humanrf_amd.optim import AdamW
    copies = {net.weight: torch.zeros(5, 20, dtype=torch.float16)}
    opt = AdamW(net.parameters(), lr=3e-3, state_bits=bits, max_grad_norm=2.0, seed=7, copies=copies)
    host.count = 2
    for p in net.parameters():
        p.grad = torch.ones_like(p)

    def again(pair):
        if how == "deepcopy":
            return copy.deepcopy(pair)
        file = io.BytesIO()
        torch.save(pair, file)
        return torch.load(io.BytesIO(file.getvalue()), weights_only=False)
    fresh_net, fresh = again((net, opt))                 # before the first step
    assert fresh._plan is None and fresh.max_grad_norm == 2.0 and fresh.state_bits == bits
    opt.step()
    for k, buf in enumerate(opt._plan.state.values()):
        buf.view(torch.uint8)[:5] = k + 1
    opt._plan.steps[:] = torch.tensor([3, 4], dtype=torch.int32)
    other_net, other = again((net, opt))
    for p in list(other_net.parameters()) + list(fresh_net.parameters()):
        p.grad = torch.ones_like(p)
    for made, made_net in ((other, other_net), (fresh, fresh_net)):
        made.step()
        rows = host.calls[-1][2]
        assert rows["param"].tolist() == [p.data_ptr() for p in made_net.parameters()]
        assert rows["copy"].tolist()[0] == made._copies[made_net.weight].data_ptr() != copies[net.weight].data_ptr()
        assert host.calls[-1][1][10] == 3e-3 and host.calls[-1][1][21] == 7
    assert other._plan.steps.tolist() == [3, 4] and fresh._plan.steps.tolist() == [0, 0]
    for name, buf in opt._plan.state.items():
        assert torch.equal(buf.view(torch.uint8), other._plan.state[name].view(torch.uint8))
        assert buf.data_ptr() != other._plan.state[name].data_ptr()
    # the original goes on, and so does loading
    opt.step()
    assert host.calls[-1][2]["param"].tolist() == [p.data_ptr() for p in net.parameters()]
    other.load_state_dict(opt.state_dict())
    assert other._plan.steps.tolist() == opt._plan.steps.tolist()


def _checkpoint(opt):
    import copy
    return copy.deepcopy(opt.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_that_does_not_fit_changes_nothing(host, bits):
    opt, params = _stepped(host, [torch.zeros(6, 5), torch.zeros(7)], lr=3e-3, state_bits=bits)
    for buf in opt._plan.state.values():
        buf.view(torch.uint8).fill_(3)
    opt._plan.steps[:] = 5
    before = {name: buf.clone() for name, buf in opt._plan.state.items()}

    def spoil(change):
        sd = _checkpoint(opt)
        for entry in sd["state"].values():
            for v in entry.values():
                v.view(torch.uint8).fill_(9) if v.dim() else None
        sd["param_groups"][0]["lr"] = 1.0
        change(sd)
        return sd
    cases = [(lambda sd: sd["state"][1].pop("exp_avg"), "has no exp_avg for parameter 1"),
             (lambda sd: sd["state"][1].update(exp_avg=sd["state"][1]["exp_avg"][:6]), "parameter 1 has another shape"),
             (lambda sd: sd["state"][0].update(exp_avg=sd["state"][0]["exp_avg"].to(torch.float32 if bits == 8 else torch.float8_e4m3fn)), "another shape or type"),
             (lambda sd: sd["state"][1].update(step=torch.tensor(-1.0)), "negative step"),
             (lambda sd: sd["param_groups"][0].update(amsgrad=True), "amsgrad"),
             (lambda sd: sd["param_groups"][0].update(maximize=True), "maximize"),
             (lambda sd: sd["param_groups"][0].update(decoupled_weight_decay=False), "coupled")]
    for change, said in cases:
        with pytest.raises((RuntimeError, ValueError), match=said):
            opt.load_state_dict(spoil(change))
        assert all(torch.equal(buf.view(torch.uint8), before[name].view(torch.uint8)) for name, buf in opt._plan.state.items())
        assert opt._plan.steps.tolist() == [5, 5] and opt.param_groups[0]["lr"] == 3e-3
    opt.load_state_dict(spoil(lambda sd: None))
    assert opt.param_groups[0]["lr"] == 1.0
    assert int(opt._plan.state["exp_avg"].view(torch.uint8)[0]) == 9


def test_groups_that_do_not_fit_change_nothing(host):
    opt, params = _stepped(host, [torch.zeros(6), torch.zeros(7)])
    from humanrf_amd.optim import AdamW
    opt = AdamW([{"params": params[:1]}, {"params": params[1:]}], lr=3e-3)
    opt.step()
    opt._plan.state["exp_avg"].fill_(2.0)
    sd = _checkpoint(opt)
    sd["param_groups"][1]["eps"] = 1e-3
    with pytest.raises(ValueError, match="betas and eps"):
        opt.load_state_dict(sd)
    assert opt.param_groups[1]["eps"] == 1e-15 and float(opt._plan.state["exp_avg"][0]) == 2.0
    torch_s = torch.optim.AdamW(params, amsgrad=True)
    torch_s.step()
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW(params).load_state_dict(torch_s.state_dict())


@pytest.mark.parametrize("bad", [dict(lr=-1e-3), dict(weight_decay=-0.1), dict(lr=float("nan")), dict(lr=float("inf")), dict(weight_decay=float("nan"))],
                         ids=str)
def test_every_group_s_lr_and_decay_are_looked_at(host, bad):
    """One negative next to a positive one became a negative factor, and the group climbed; max() of a NaN is whichever comes first."""
    from humanrf_amd.optim import AdamW
    make = lambda **kw: [{"params": [torch.nn.Parameter(torch.zeros(4))]}, {"params": [torch.nn.Parameter(torch.zeros(4))], **kw}]  # noqa: E731
    with pytest.raises(ValueError, match="finite and not negative"):
        AdamW(make(**bad))
    groups = make()
    host.count = 2
    opt = AdamW(groups)
    for g in opt.param_groups:
        g["params"][0].grad = torch.ones(4)
    opt.step()
    n = len(host.calls)
    opt.param_groups[1].update(bad)         # as a schedule would
    with pytest.raises(ValueError, match="finite and not negative"):
        opt.step()
    assert len(host.calls) == n


def test_versions_of_what_a_step_writes(host):
    """Through ops.adamw_multi as through the optimizer: a cast that is renewed by version (HumanRF's 16-bit copies) sees the step, and autograd
    refuses to go back through what was overwritten."""
    from humanrf_amd import ops
    host.count = 2
    p, q = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(5))
    c, g = torch.zeros(4, dtype=torch.float16), torch.zeros(4)
    plan = ops.AdamWPlan([p, q], [g, None], copies=[c, None])
    watched = (p, q, c, g)
    before = [t._version for t in watched]
    ops.adamw_multi(plan, 1e-2)
    assert [t._version - b for t, b in zip(watched, before)] == [1, 0, 1, 0]
    ops.adamw_multi(plan, 1e-2, zero_grad=True)
    assert [t._version - b for t, b in zip(watched, before)] == [2, 0, 2, 1]
    x = torch.ones(4, requires_grad=True)
    y = (x * c.float() * p).sum()
    ops.adamw_multi(plan, 1e-2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    flat = torch.zeros(10)
    views, version = [flat[:4], flat[4:]], flat._version
    ops.adamw_multi(ops.AdamWPlan(views, [torch.ones(4), torch.ones(6)]), 1e-2)
    assert flat._version == views[1]._version == version + 1
    opt, (p,) = _stepped(host, [torch.zeros(4)])
    before, g = (p._version, p.grad._version), p.grad
    opt.step(zero_grad=True)
    assert (p._version, g._version) == (before[0] + 1, before[1] + 1)


def test_nothing_that_a_step_writes_shares_memory(host):
    """Workgroups work on the tensors side by side: a gradient inside another tensor's values, or values inside the states, would be read
    before or after they are written."""
    from humanrf_amd import ops
    host.count = 2
    buf, g = torch.zeros(2000), torch.zeros(2000)
    p = [buf[:50], buf[50:100]]
    plan = ops.AdamWPlan(p, [g[:50], g[50:100]])
    for grads in ([buf[50:100], None], [buf[:50], None], [g[:50], g[49:99]]):
        with pytest.raises(RuntimeError, match="share memory"):
            plan.set_grads(grads)
        with pytest.raises(RuntimeError, match="share memory"):
            ops.AdamWPlan(p, grads)
    state = {"exp_avg": buf[64:576], "exp_avg_sq": g[200:712]}
    with pytest.raises(RuntimeError, match="share memory|multiple of 16"):
        ops.AdamWPlan(p, [g[:50], g[50:100]], state=state)
    big = torch.zeros(4096)
    at = (-big.data_ptr() // 4) % 4
    whole = big[at:at + 1024]
    with pytest.raises(RuntimeError, match="share memory"):
        ops.AdamWPlan(p, state={"exp_avg": whole[:512], "exp_avg_sq": whole[256:768]})
    with pytest.raises(RuntimeError, match="share memory"):
        ops.AdamWPlan([whole[:50], whole[600:650]], state={"exp_avg": whole[:512], "exp_avg_sq": big[2048 + at:2560 + at]})
    ops.AdamWPlan(p, [g[:50], g[50:100]], state={"exp_avg": whole[:512], "exp_avg_sq": whole[512:]})
    assert np.array_equal(plan._rows["grad"], [g.data_ptr(), g.data_ptr() + 200])


def test_an_lr_in_a_tensor_on_the_host_is_a_number(host):
    """As torch.optim.AdamW takes it; a schedule writes into it."""
    lr = torch.tensor(3e-3, dtype=torch.float64)
    opt, params = _stepped(host, [torch.zeros(4), torch.zeros(7)], lr=lr)
    assert host.calls[-1][1][10:12] == (3e-3, None)
    lr.fill_(1e-3)
    opt.step()
    assert host.calls[-1][1][10:12] == (1e-3, None)
    n = len(host.calls)
    lr.fill_(-1.0)
    with pytest.raises(ValueError, match="finite and not negative"):
        opt.step()
    assert len(host.calls) == n
