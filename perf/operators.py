"""What is measured of the AdamW step over many tensors and of the matrix product in 8-bit integers: their cases, inputs and plain forms.

Two operators. "step": one AdamW step over a list of tensors, with first and second moments in 32 bits, or in 8 (e4m3 codes with one
fp32 scale for every 256 values; the second moment as its square root; rounded up or down at random, unbiased, by a counter-based hash),
after a global gradient norm where the case clips. "product": y = act(x W^T + b) with W in 8-bit integers and a scale for each channel,
tokens rounded to 8 bits with a scale for each token inside the call, or handed in as integers with their scales."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BETA1, BETA2, EPS, LR, DECAY, MAX_NORM, SEED, STEP0 = 0.9, 0.99, 1e-15, 1e-2, 1e-2, 1.0, 20, 100
BLOCK = 256          # values of one tensor that share a scale; a tensor begins on a block of its own


def listed():
    return [
        # the two networks and the camera embeddings of a field model: a handful of small tensors, where latency counts
        {"name": "step32 small", "op": "step", "tensors": 5, "total": 14_000, "bits": 32, "params": "float32", "copy": True, "clip": True},
        # hash tables and vectors of seven temporal segments with the fp16 copy that the gather kernels read
        {"name": "step32 tables", "op": "step", "tensors": 15, "total": 39_000_000, "bits": 32, "params": "float32", "copy": True, "clip": False},
        # a network of many layers kept in bf16, gradients clipped
        {"name": "step32 bf16 layers", "op": "step", "tensors": 217, "total": 120_000_000, "bits": 32, "params": "bfloat16", "copy": False, "clip": True},
        # small ragged layers and biases, 8-bit states
        {"name": "step8 small", "op": "step", "tensors": 24, "total": 90_000, "bits": 8, "params": "float32", "copy": False, "clip": True},
        # the tables again, 8-bit states
        {"name": "step8 tables", "op": "step", "tensors": 15, "total": 39_000_000, "bits": 8, "params": "float32", "copy": True, "clip": False},
        # a long capture: many segments' tables, clipped
        {"name": "step8 large", "op": "step", "tensors": 161, "total": 240_000_000, "bits": 8, "params": "float32", "copy": False, "clip": True},
        # a few rows through a narrow layer: latency
        {"name": "product tiny", "op": "product", "rows": 3, "cols": 200, "inner": 136, "tokens": "float16", "out": "float16", "bias": True, "relu": True},
        # one token against a square layer: the weights' bytes
        {"name": "product one token", "op": "product", "rows": 1, "cols": 4096, "inner": 4096, "tokens": "bfloat16", "out": "bfloat16", "bias": False, "relu": False},
        # a small batch of tokens, a wide layer, already in integers
        {"name": "product 29 tokens", "op": "product", "rows": 29, "cols": 10240, "inner": 5120, "tokens": "int8", "out": "float32", "bias": True, "relu": False},
        # every sample of half a training batch through one 64-neuron layer: the bytes of x and y
        {"name": "product samples", "op": "product", "rows": 320_000, "cols": 64, "inner": 64, "tokens": "float16", "out": "float16", "bias": True, "relu": True},
        # odd sizes in every direction
        {"name": "product ragged", "op": "product", "rows": 1021, "cols": 4099, "inner": 2051, "tokens": "bfloat16", "out": "bfloat16", "bias": True, "relu": True},
        # a long prompt's or a full image's rows through a large layer: the matrix rate
        {"name": "product large", "op": "product", "rows": 8192, "cols": 8192, "inner": 8192, "tokens": "bfloat16", "out": "bfloat16", "bias": False, "relu": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        total = _log(rng, 10_000, 240_000_000)
        bits, params = rng.choice((8, 32)), rng.choice(("float32", "float32", "bfloat16", "float16"))
        return {"op": "step", "tensors": _log(rng, 1, min(220, total // 500)), "total": min(total, 240_000_000 if bits == 8 else 120_000_000),
                "bits": bits, "params": params, "copy": params == "float32" and rng.random() < 0.5, "clip": rng.random() < 0.6}
    while True:
        rows, cols, inner = _log(rng, 1, 320_000), _log(rng, 48, 10_240), _log(rng, 48, 8192)
        if rows * cols * inner <= 8192 ** 3 and rows * (cols + inner) <= 2 ** 28:
            break
    tokens = rng.choice(("float16", "bfloat16", "float32", "int8"))
    return {"op": "product", "rows": rows, "cols": cols, "inner": inner, "tokens": tokens, "out": rng.choice(("float16", "bfloat16")),
            "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}


def _sizes(case):
    """Lengths of the tensors: three in four of them about as long as each other, the others a 64th of that; odd lengths among them."""
    count, total = case["tensors"], case["total"]
    weights = [(1.0 if k % 4 else 1.0 / 64.0) * (1.0 + 0.37 * ((k * 7919) % 13) / 13.0) for k in range(count)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    return [n if k % 3 else n | 1 for k, n in enumerate(sizes)]


def _offsets(sizes):
    offsets = [0]
    for n in sizes:
        offsets.append(offsets[-1] + -(-n // BLOCK) * BLOCK)
    return offsets


def _prepare_step(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sizes = _sizes(case)
    offsets = _offsets(sizes)
    total, dtype, device = offsets[-1], DTYPES[case["params"]], "cuda"
    # every tensor in one buffer, on a block of its own, zeros behind its end; a tensor's gradients have a magnitude of their own
    inside = torch.zeros(total, dtype=torch.bool, device=device)
    size = torch.empty(total, device=device)
    scales = torch.exp(torch.randn(len(sizes), generator=gen, device=device) * 1.5) * 1e-4
    for k, n in enumerate(sizes):
        inside[offsets[k]:offsets[k] + n] = True
        size[offsets[k]:offsets[k + 1]] = scales[k]
    normal = lambda: torch.randn(total, generator=gen, device=device)  # noqa: E731
    zero = torch.zeros((), device=device)
    param = torch.where(inside, normal() * 0.1, zero).to(dtype)
    touched = torch.rand(total, generator=gen, device=device) < 0.7        # table entries that no sample of the batch reads get no gradient
    grad = torch.where(inside & touched, normal() * size, zero).to(dtype)
    first = torch.where(inside, normal() * size * 0.3, zero)
    second = torch.where(inside, (normal() * size).square() * 0.5 + (0.1 * size).square(), zero)
    s = {"op": "step", "bits": case["bits"], "clip": case["clip"], "param": param, "grad": grad, "step": STEP0,
         "copy": param.to(torch.float16) if case["copy"] else None}
    if case["bits"] == 32:
        s["state"] = {"exp_avg": first, "exp_avg_sq": second}
    else:
        s["state"] = {}
        for name, x in (("exp_avg", first), ("exp_avg_root", second.sqrt())):
            top = x.view(-1, BLOCK).abs().amax(1)
            t = x.view(-1, BLOCK) * torch.where(top > 0, torch.full_like(top, 448.0) / top, top).unsqueeze(1)
            s["state"][name] = t.reshape(-1).to(torch.float8_e4m3fn)
            s["state"][name + "_scale"] = top * (1.0 / 448.0)
    if own:
        from humanrf_amd import ops
        views = lambda x: None if x is None else [x[o:o + n] for o, n in zip(offsets, sizes)]  # noqa: E731
        s["plan"] = ops.AdamWPlan(views(param), views(grad), copies=views(s["copy"]), state_bits=case["bits"], state=s["state"],
                                  step=STEP0, seed=SEED)
    return s


def _prepare_product(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, n, k, device = case["rows"], case["cols"], case["inner"], "cuda"
    weight = torch.randint(-127, 128, (n, k), generator=gen, device=device, dtype=torch.int8)
    s = {"op": "product", "relu": case["relu"], "out": DTYPES[case["out"]], "weight": weight, "x_scale": None, "bias": None,
         "weight_scale": (torch.rand(n, generator=gen, device=device) + 0.5) * (0.02 / math.sqrt(k))}
    if case["bias"]:
        s["bias"] = torch.randn(n, generator=gen, device=device) * 0.1
    if case["tokens"] == "int8":
        s["x"] = torch.randint(-127, 128, (m, k), generator=gen, device=device, dtype=torch.int8)
        s["x_scale"] = (torch.rand(m, generator=gen, device=device) + 0.5) / 40.0
    else:
        # activations: each row of a size of its own, a few columns much larger than the rest
        x = torch.randn(m, k, generator=gen, device=device) * (torch.rand(m, 1, generator=gen, device=device) + 0.2)
        x[:, :: max(1, k // 7)] *= 6.0
        s["x"] = x.to(DTYPES[case["tokens"]])
    if own:
        from humanrf_amd import ops
        s["handle"] = ops.Int8Weight(weight, s["weight_scale"], s["bias"])
    return s


def prepare(case, seed):
    return _prepare_step(case, seed) if case["op"] == "step" else _prepare_product(case, seed)


# ------------------------------------------------------------------------------------------------ plain forms
def _mix(x):
    """32-bit integer hash, in int64 lanes."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _to_e4m3(x, random, floor):
    """Blocks of 256 values -> codes and scales: |x| * 448 / amax, then up or down to a neighbouring e4m3 value with the 16 random bits
    of each position; `floor`: what is not zero gets a code that is not zero. A block whose largest value is under 2^-100 is zeros."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1)
    top = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top)
    inverse = torch.where(top > 0, torch.full_like(top, 448.0) / top, top).unsqueeze(1)
    t = (b.abs() * inverse).clamp(max=448.0).reshape(-1)
    low = torch.where(t < 2.0 ** -6, 2.0 ** -6, 0.0)      # below 2^-6 the values are 2^-9 apart, as in the binade that this moves them to
    bits = (t + low).view(torch.int32) + (random.to(torch.int32) << 4)
    q = (bits & -0x100000).view(torch.float32) - low
    q = q.clamp(max=448.0)
    if floor:
        q = torch.where(t > 0, q.clamp(min=2.0 ** -9), q)
    return torch.where(x < 0, -q, q).to(torch.float8_e4m3fn), top * (1.0 / 448.0)


def _from_e4m3(code, scale):
    return (code.to(torch.float32).view(-1, BLOCK) * scale.unsqueeze(1)).reshape(-1)


def _plain_step(s):
    p, g, state = s["param"].float(), s["grad"].float(), s["state"]
    s["step"] += 1
    if s["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (MAX_NORM / (norm.double() + 1e-6)).clamp(max=1.0).float()
    if s["bits"] == 32:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    else:
        m = _from_e4m3(state["exp_avg"], state["exp_avg_scale"])
        r = _from_e4m3(state["exp_avg_root"], state["exp_avg_root_scale"])
        v = r * r
    m = m + (g - m) * (1.0 - BETA1)
    v = v * BETA2 + g * (1.0 - BETA2) * g
    root = v.sqrt()
    denominator = root * (1.0 / math.sqrt(1.0 - BETA2 ** s["step"])) + EPS
    p = p * (1.0 - LR * DECAY) - (m / denominator) * (LR / (1.0 - BETA1 ** s["step"]))
    s["param"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if s["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = m, v
    else:
        at = torch.arange(p.numel(), device=p.device)
        h = _mix(at ^ _mix(SEED ^ _mix(s["step"])))
        state["exp_avg"], state["exp_avg_scale"] = _to_e4m3(m, h & 0xFFFF, False)
        state["exp_avg_root"], state["exp_avg_root_scale"] = _to_e4m3(root, h >> 16, True)
    return {"param": s["param"], "copy": s["copy"], "norm": norm if s["clip"] else None, **state}


def _int_product(x, w):
    """Sums of products of 8-bit integers: exact in fp32 over 1024 of them, joined in 64 bits."""
    total = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    for k in range(0, x.shape[1], 1024):
        total += x[:, k:k + 1024].float() @ w[:, k:k + 1024].float().t()
    return total.float()


def _plain_product(s):
    x, scale = s["x"], s["x_scale"]
    if scale is None:
        x = x.float()
        top = x.abs().amax(1).clamp(min=2.0 ** -119)
        scale = top * (1.0 / 127.0)
        x = (x * (torch.full_like(top, 127.0) / top).unsqueeze(1)).round()
    y = _int_product(x, s["weight"]) * scale.unsqueeze(1) * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["relu"]:
        y = y.clamp(min=0.0)
    return y.to(s["out"])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_step(s):
    from humanrf_amd import ops
    plan, norm = s["plan"], None
    if s["clip"]:
        norm = ops.grad_norm_multi(plan)
    ops.adamw_multi(plan, LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, norm=norm, max_norm=MAX_NORM if s["clip"] else None)
    return {"param": s["param"], "copy": s["copy"], "norm": norm, **plan.state}


def _own_product(s):
    from humanrf_amd import ops
    return ops.linear_int8(s["x"], s["handle"], x_scale=s["x_scale"], relu=s["relu"], out_dtype=s["out"])


def run(state):
    if own:
        return _own_step(state) if state["op"] == "step" else _own_product(state)
    return _plain_step(state) if state["op"] == "step" else _plain_product(state)


def work(case):
    if case["op"] == "step":
        n, size = sum(_sizes(case)), DTYPES[case["params"]].itemsize
        state = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
        return {"bytes": n * (3 * size + state + (2 if case["copy"] else 0)), "flops": n * (20.0 if case["bits"] == 32 else 60.0)}
    m, n, k = case["rows"], case["cols"], case["inner"]
    item = 1 if case["tokens"] == "int8" else DTYPES[case["tokens"]].itemsize
    return {"bytes": m * k * item + n * k + m * n * DTYPES[case["out"]].itemsize + 4.0 * (n * (2 if case["bias"] else 1)), "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _code64(values, noise, keep):
    """The e4m3 value next below or above each |value| * 448 / amax, above where the fraction between them is over 1 - noise."""
    rows = values.reshape(-1, BLOCK)
    largest = rows.abs().max(dim=1).values
    largest[largest < 2.0 ** -100] = 0.0
    t = (rows.abs() * torch.nan_to_num(448.0 / largest, posinf=0.0).unsqueeze(1)).reshape(-1)
    gap = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
    q = torch.floor(t / gap + noise) * gap
    if keep:
        q[(t > 0) & (q == 0)] = 2.0 ** -9
    return torch.sign(values) * q.clamp(max=448.0), largest / 448.0


def _exact_step(s):
    t = s["step"] + 1
    g, p = s["grad"].double(), s["param"].double()
    norm = torch.linalg.vector_norm(g) if s["clip"] else None
    if norm is not None:
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    st = {k: x.double() for k, x in s["state"].items()}
    if s["bits"] == 32:
        m, v = st["exp_avg"], st["exp_avg_sq"]
    else:
        m = st["exp_avg"] * st["exp_avg_scale"].repeat_interleave(BLOCK)
        v = (st["exp_avg_root"] * st["exp_avg_root_scale"].repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    p = (1.0 - LR * DECAY) * p - LR * (m / (1.0 - BETA1 ** t)) / (torch.sqrt(v / (1.0 - BETA2 ** t)) + EPS)
    out = {"param": p, "copy": p if s["copy"] is not None else None, "norm": norm}
    if s["bits"] == 32:
        out.update(exp_avg=m, exp_avg_sq=v)
        return out
    at = torch.arange(p.numel(), device=p.device, dtype=torch.int64)

    def scramble(x):
        for shift, factor in ((16, 2146121005), (15, 2221713035), (16, 1)):
            x = ((x ^ (x >> shift)) * factor) % 2 ** 32
        return x
    h = scramble(at ^ scramble(SEED ^ scramble(t)))
    out["exp_avg"], out["exp_avg_scale"] = _code64(m, (h % 65536).double() / 65536.0, False)
    out["exp_avg_root"], out["exp_avg_root_scale"] = _code64(v.sqrt(), (h // 65536).double() / 65536.0, True)
    return out


def _exact_product(s):
    x = s["x"].double()
    scale = s["x_scale"].double() if s["x_scale"] is not None else None
    if scale is None:
        scale = x.abs().max(dim=1).values / 127.0
        x = torch.round(x / scale[:, None])
    y = torch.matmul(x, s["weight"].double().t().contiguous())
    y = y * torch.outer(scale, s["weight_scale"].double())
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return torch.relu(y) if s["relu"] else y


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_step(s) if case["op"] == "step" else _exact_product(s)
