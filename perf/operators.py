"""Operators that are measured, with their plain forms.

``layer_norm``     normalisation of each row over its channels, with an
                   optional residual and ReLU, alone or with its gradients
``newton_schulz``  the orthogonal factor of a matrix, or of a batch of them,
                   by Newton-Schulz products
``muon_step_``     one optimiser step over a flat parameter buffer: momentum,
                   the Newton-Schulz products of every matrix, the update

``own`` chooses between elementary torch operations (False) and the
framework's operators (True).  A case is a dict of plain values.
"""

import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NS_EPS = 1e-7
LN_EPS = 1e-5
DTYPES = {
    "fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
}
DEVICE = "cuda"


# ------------------------------------------------------------------- cases

def _ln(name, rows, cols, dtype, train, residual, relu):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols,
            "dtype": dtype, "train": train, "residual": residual,
            "relu": relu}


def _ns(name, batch, rows, cols, dtype):
    return {"name": name, "op": "newton_schulz", "batch": batch,
            "rows": rows, "cols": cols, "dtype": dtype}


def _muon(name, depth, width, classes, dtype):
    return {"name": name, "op": "muon_step", "depth": depth, "width": width,
            "classes": classes, "dtype": dtype}


def listed():
    return [
        # one token's activations at inference: latency alone
        _ln("ln_one_token", 1, 2048, "bf16", False, False, False),
        # the last join of a ResNet-50 stage 4 block at 32 images
        _ln("ln_stage4_join", 32 * 7 * 7, 2048, "bf16", True, True, True),
        # the join of a ResNet-50 stage 1 block at 32 images: many short
        # rows, the largest activations of the network
        _ln("ln_stage1_join", 32 * 56 * 56, 256, "bf16", True, True, True),
        # full precision, an odd width: no row but the first is aligned
        _ln("ln_odd_rows", 8191, 1001, "fp32", True, False, False),
        # long rows of a wide model, half precision
        _ln("ln_long_rows", 4096, 16384, "fp16", True, False, False),
        # the smallest matrix a network has: latency alone
        _ns("ns_small", 1, 64, 64, "fp32"),
        # the classifier of ResNet-50
        _ns("ns_classifier", 1, 1000, 2048, "fp32"),
        # a few tall matrices of odd sizes, worked on together
        _ns("ns_tall_batch", 6, 2303, 257, "bf16"),
        # a large square matrix
        _ns("ns_large", 1, 4096, 4096, "bf16"),
        # a small network with odd widths: every matrix is tiny
        _muon("muon_narrow", 18, 15, 10, "fp32"),
        # ResNet-18, full-precision weights and gradients
        _muon("muon_resnet18", 18, 64, 1000, "fp32"),
        # ResNet-50, bf16 gradients and working weights, fp32 master
        _muon("muon_resnet50", 50, 64, 1000, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.random()
    if kind < 0.5:
        cols = _log_int(rng, 8, 16384)
        rows = _log_int(rng, 1, max(1, min(131072, (1 << 26) // cols)))
        train = rng.random() < 0.75
        residual = rng.random() < 0.5
        return {"op": "layer_norm", "rows": rows, "cols": cols,
                "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "train": train, "residual": residual,
                "relu": rng.random() < 0.5}
    if kind < 0.8:
        rows = _log_int(rng, 16, 4096)
        cols = _log_int(rng, 16, 4096)
        most = 4.0 * 4096 ** 3 / (4.0 * min(rows, cols) ** 2
                                  * max(rows, cols))
        return {"op": "newton_schulz",
                "batch": _log_int(rng, 1, max(1, min(12, int(most)))),
                "rows": rows, "cols": cols,
                "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    return {"op": "muon_step", "depth": rng.choice([18, 34, 50]),
            "width": _log_int(rng, 8, 64), "classes": _log_int(rng, 10, 1000),
            "dtype": rng.choice(["fp32", "bf16"])}


# ------------------------------------------------------------------ inputs

def _resnet_shapes(depth, width, classes):
    """Weight shapes of a ResNet in the order of its modules, convolutions
    as [out, in * k * k], without its vectors."""
    blocks = {18: (2, 2, 2, 2), 34: (3, 4, 6, 3), 50: (3, 4, 6, 3)}[depth]
    bottle = depth == 50
    shapes, cin = [(width, 3 * 49)], width
    for stage, count in enumerate(blocks):
        planes = width << stage
        cout = planes * 4 if bottle else planes
        for i in range(count):
            if bottle:
                shapes += [(planes, cin), (planes, planes * 9),
                           (cout, planes)]
            else:
                shapes += [(planes, cin * 9), (planes, planes * 9)]
            if i == 0 and (stage > 0 or cin != cout):
                shapes.append((cout, cin))
            cin = cout
    shapes.append((classes, cin))
    return shapes


def _layout(case):
    """[(start, rows, cols)] of the matrices in the flat buffer, and its
    length.  bf16: the matrices lie one after another.  fp32: each is
    followed by the vectors of its normalisation (a weight and a bias of
    its rows), as a module lists its parameters."""
    at, where = 0, []
    for rows, cols in _resnet_shapes(
            case["depth"], case["width"], case["classes"]):
        where.append((at, rows, cols))
        at += rows * cols
        if case["dtype"] == "fp32":
            at += 2 * rows
    return where, at


def _gradient(gen, *shape):
    """A matrix with a few strong directions over noise, as gradients have."""
    rank = min(4, shape[-1], shape[-2])
    left = torch.randn(*shape[:-1], rank, generator=gen, device=DEVICE)
    right = torch.randn(*shape[:-2], rank, shape[-1], generator=gen,
                        device=DEVICE)
    noise = torch.randn(*shape, generator=gen, device=DEVICE)
    return noise + 0.5 * torch.matmul(left, right)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(1000003 * seed + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # rows with a mean and a scale of their own
        x = randn(rows, cols) * (0.5 + randn(rows, 1).abs()) + randn(rows, 1)
        state["x"] = x.to(dtype)
        state["weight"] = 1.0 + 0.2 * randn(cols)
        state["bias"] = 0.2 * randn(cols)
        state["res"] = randn(rows, cols).to(dtype) if case["residual"] \
            else None
        if case["train"]:
            dy = randn(rows, cols).to(dtype)
            if case["relu"]:
                # no gradient comes from where the last bit of a sum
                # decides on which side of the ReLU's border it lies
                z = _ln_parts(state, torch.float64)[0]
                dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
            state["dy"] = dy
            state["leaves"] = [
                t for t in (state["x"], state["weight"], state["bias"],
                            state["res"]) if t is not None]
            for t in state["leaves"]:
                t.requires_grad_(True)
    elif case["op"] == "newton_schulz":
        g = _gradient(gen, case["batch"], case["rows"], case["cols"])
        state["g"] = (1e-3 * g).to(dtype)
    else:
        where, total = _layout(case)
        state["where"] = where
        params, grads, buf = randn(total), randn(total), randn(total)
        for start, rows, cols in where:
            n = rows * cols
            params[start:start + n] *= math.sqrt(2.0 / cols)
            grads[start:start + n] = _gradient(gen, rows, cols).reshape(-1)
        state["params"] = params
        state["grads"] = (1e-3 * grads).to(dtype)
        state["buf"] = 1e-3 * buf
        state["shadow"] = params.to(dtype) if case["dtype"] == "bf16" \
            else None
        state["lr"] = torch.tensor([0.02], device=DEVICE)
        if own:
            from stochastic_gradient_push_amd import ops
            state["plan"] = ops.MuonPlan(where, total, DEVICE)
    return state


# ------------------------------------------------------------- plain forms

def _ln_parts(state, dtype):
    """The value before the ReLU, the normalised rows and 1 / deviation."""
    x = state["x"].detach().to(dtype)
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True)
                            + LN_EPS)
    hat = centred * rstd
    z = hat * state["weight"].detach().to(dtype) \
        + state["bias"].detach().to(dtype)
    if state["res"] is not None:
        z = z + state["res"].detach().to(dtype)
    return z, hat, rstd


def _plain_layer_norm(state):
    kind = state["x"].dtype
    z, hat, rstd = _ln_parts(state, torch.float32)
    y = torch.where(z > 0, z, torch.zeros_like(z)) if state["relu"] else z
    if not state["train"]:
        return [y.to(kind)]
    g = state["dy"].float()
    if state["relu"]:
        g = torch.where(z > 0, g, torch.zeros_like(g))
    gw = g * state["weight"].detach()
    dx = rstd * (gw - gw.mean(-1, keepdim=True)
                 - hat * (gw * hat).mean(-1, keepdim=True))
    out = [y.to(kind), dx.to(kind), (g * hat).sum(0), g.sum(0)]
    return out + [g.to(kind)] if state["res"] is not None else out


def _plain_newton_schulz(g):
    """Of [..., rows, cols] in 32 bits, not rounded."""
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    x = x / (torch.sqrt((x * x).sum((-1, -2), keepdim=True)) + NS_EPS)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2) if tall else x


MOMENTUM, DECAY = 0.95, 0.01


def _plain_muon_step(state):
    params, buf, lr = state["params"], state["buf"], state["lr"]
    g = state["grads"].float()
    whole = torch.zeros_like(params, dtype=torch.bool)
    for start, rows, cols in state["where"]:
        whole[start:start + rows * cols] = True
    # vectors: SGD with coupled decay; matrices: decay apart from momentum
    g = torch.where(whole, g, g + DECAY * params)
    buf.mul_(MOMENTUM).add_(g)
    u = g + MOMENTUM * buf
    params.copy_(torch.where(whole, params * (1 - lr * DECAY),
                             params - lr * u))
    shapes = {}
    for start, rows, cols in state["where"]:
        shapes.setdefault((rows, cols), []).append(start)
    for (rows, cols), starts in shapes.items():  # equal shapes together
        n = rows * cols
        o = _plain_newton_schulz(torch.stack(
            [u[at:at + n] for at in starts]).view(-1, rows, cols))
        o = lr * math.sqrt(max(1.0, rows / cols)) * o.reshape(-1, n)
        for at, step in zip(starts, o):
            params[at:at + n] -= step
    if state["shadow"] is not None:
        state["shadow"].copy_(params)


def run(state):
    if state["op"] == "layer_norm":
        if not own:
            return _plain_layer_norm(state)
        from stochastic_gradient_push_amd import ops
        y = ops.layer_norm(state["x"], state["weight"], state["bias"],
                           eps=LN_EPS, residual=state["res"],
                           relu=state["relu"])
        if not state["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(
            y, state["leaves"], state["dy"])]
    if state["op"] == "newton_schulz":
        if not own:
            return [_plain_newton_schulz(state["g"])
                    .to(state["g"].dtype).contiguous()]
        from stochastic_gradient_push_amd import ops
        return [ops.newton_schulz(state["g"], steps=STEPS,
                                  coefficients=COEFFICIENTS, eps=NS_EPS)]
    if own:
        from stochastic_gradient_push_amd import ops
        ops.muon_step_(state["params"], state["grads"], state["buf"],
                       state["plan"], state["lr"], momentum=MOMENTUM,
                       weight_decay=DECAY, nesterov=True, steps=STEPS,
                       coefficients=COEFFICIENTS, eps=NS_EPS,
                       shadow=state["shadow"])
    else:
        _plain_muon_step(state)
    out = [state["params"], state["buf"]]
    return out + [state["shadow"]] if state["shadow"] is not None else out


# ------------------------------------------------------------ work, oracle

def _ns_flops(rows, cols):
    """X X^T and its square are symmetric: half of each is needed."""
    n, m = min(rows, cols), max(rows, cols)
    return STEPS * (n * n * m + n * n * n + 2 * n * n * m)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # x and y, and in training dy and dx; the residual and its gradient
        each = 2 + (2 if case["train"] else 0)
        if case["residual"]:
            each += 2 if case["train"] else 1
        vectors = 4 if case["train"] else 2
        return {"bytes": each * rows * cols * size + vectors * cols * 4,
                "flops": (18 if case["train"] else 8) * rows * cols}
    if case["op"] == "newton_schulz":
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        return {"bytes": 2 * batch * rows * cols * size,
                "flops": batch * _ns_flops(rows, cols)}
    where, total = _layout(case)
    # params and momentum are read and written, gradients read, and the
    # bf16 working weights written
    return {"bytes": total * (16 + size + (2 if size == 2 else 0)),
            "flops": sum(_ns_flops(r, c) for _, r, c in where) + 8 * total}


def _exact_factor(g):
    a, b, c = COEFFICIENTS
    x = g.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True)
             + NS_EPS)
    eye = torch.eye(min(x.shape[-2:]), dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            s = x @ x.mT.contiguous()
            x = (a * eye + s @ (b * eye + c * s)) @ x
        else:
            s = x.mT.contiguous() @ x
            x = x @ (a * eye + s @ (b * eye + c * s))
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "newton_schulz":
        return [_exact_factor(state["g"])]
    if case["op"] == "muon_step":
        p, g = state["params"].double(), state["grads"].double()
        buf, lr = state["buf"].double(), state["lr"].double()
        inside = torch.zeros(p.numel(), dtype=torch.bool, device=p.device)
        for start, rows, cols in state["where"]:
            inside[start:start + rows * cols] = True
        g = g + DECAY * p * (~inside)
        buf = MOMENTUM * buf + g
        u = g + MOMENTUM * buf
        new = torch.where(inside, p - lr * DECAY * p, p - lr * u)
        for start, rows, cols in state["where"]:
            part = slice(start, start + rows * cols)
            o = _exact_factor(u[part].view(rows, cols))
            new[part] -= (lr * max(1.0, rows / cols) ** 0.5 * o).reshape(-1)
        out = [new, buf]
        return out + [new] if state["shadow"] is not None else out
    x = state["x"].detach().double().requires_grad_(True)
    w = state["weight"].detach().double().requires_grad_(True)
    b = state["bias"].detach().double().requires_grad_(True)
    leaves = [x, w, b]
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) * torch.rsqrt(var + LN_EPS) * w + b
    if state["res"] is not None:
        leaves.append(state["res"].detach().double().requires_grad_(True))
        y = y + leaves[-1]
    if state["relu"]:
        y = torch.relu(y)
    if not case["train"]:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(
        y, leaves, state["dy"].double())]
