"""The operators of a training step's tail, as cases to measure: the loss of a linear head over many classes computed without its
logits, with its gradient (``ops.linear_ce_loss``), and the orthogonalised update of an optimizer step (``ops.newton_schulz``).

``own`` selects the framework's kernels; otherwise ``run`` evaluates the same definitions with elementary torch operations."""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
IGNORE = -100

# The 3x3 and 1x1 filters of the 2D U-Net (16 .. 256 features, one input channel, two classes) as [Cout, Cin * k * k] matrices.
UNET = ((16, 9), (16, 144), (32, 144), (32, 288), (64, 288), (64, 576), (128, 576), (128, 1152), (256, 1152), (256, 2304),
        (128, 256), (128, 2304), (128, 1152), (64, 128), (64, 1152), (64, 576), (32, 64), (32, 576), (32, 288), (16, 32), (16, 288),
        (16, 144), (2, 144))


def _ns(name, shapes, dtype):
    return {"name": name, "op": "newton_schulz", "shapes": "+".join("%dx%d" % s for s in shapes), "dtype": dtype}


def _ce(name, rows, classes, width, dtype, ignored, bias, reduction, backward):
    return {"name": name, "op": "linear_ce", "rows": rows, "classes": classes, "width": width, "dtype": dtype, "ignored": ignored,
            "bias": bias, "reduction": reduction, "backward": backward}


def listed():
    return [
        # one middle filter of the U-Net: the smallest call, its launches are what counts
        _ns("ns_one_filter", [(64, 576)], "float32"),
        # every filter of the U-Net, as one optimizer step orthogonalises them
        _ns("ns_unet", UNET, "float32"),
        # odd sides in 16-bit storage: a projection of a wider network
        _ns("ns_odd_bf16", [(1000, 1537)], "bfloat16"),
        # tall, the larger side first
        _ns("ns_tall", [(4096, 1024)], "float32"),
        # a large projection
        _ns("ns_large_bf16", [(2048, 8192)], "bfloat16"),
        # a handful of rows against a thousand classes in the parity type: the smallest loss with its gradients
        _ce("ce_few_rows_f32", 16, 1000, 256, "float32", 0.0, True, "mean", True),
        # the parity type at an ordinary size, nothing a multiple of a tile
        _ce("ce_odd_f32", 4001, 8003, 384, "float32", 0.0, True, "mean", True),
        # every voxel of two 64^3 volumes against a hundred structures, from 16 features
        _ce("ce_voxels", 2 * 64 ** 3, 105, 16, "bfloat16", 0.0, True, "mean", True),
        # scribbles: 12 slices of 256^2, nine pixels of ten unlabelled
        _ce("ce_scribbles_f16", 12 * 256 ** 2, 33, 64, "float16", 0.9, True, "mean", True),
        # pixel embeddings against a memory bank
        _ce("ce_bank", 16384, 65536, 128, "bfloat16", 0.0, False, "mean", True),
        # the loss of each row alone, few rows, a large bank: the forward pass of an evaluation
        _ce("ce_rows_forward_f16", 37, 131071, 512, "float16", 0.1, True, "none", False),
        # the largest training step
        _ce("ce_large", 8192, 50000, 1024, "bfloat16", 0.1, False, "mean", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if rng.random() < 0.45:
        while True:
            shapes = [(_log(rng, 2, 4096), _log(rng, 2, 8192)) for _ in range(rng.choice([1, 1, 2, 5, 12]))]
            case = {"op": "newton_schulz", "shapes": "+".join("%dx%d" % s for s in shapes), "dtype": dtype}
            if work(case)["flops"] <= 5e11 and work(case)["bytes"] <= 1e8:
                return case
    while True:
        case = {"op": "linear_ce", "rows": _log(rng, 1, 1 << 20), "classes": _log(rng, 2, 131072), "width": _log(rng, 8, 2048),
                "dtype": dtype, "ignored": rng.choice([0.0, 0.1, 0.5, 0.9]), "bias": rng.random() < 0.5,
                "reduction": rng.choice(["mean", "sum", "none"]), "backward": rng.random() < 0.75}
        r, v, d = case["rows"], case["classes"], case["width"]
        if r * v * d <= 3e11 and r * v <= 4e8 and r * d <= 1e8 and v * d <= 1.4e8:
            return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split("+")]


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["op"] == "newton_schulz":
        flops = nbytes = 0
        for a, b in _shapes(case):
            m, n = min(a, b), max(a, b)
            # X X^T and its square are symmetric: half of each; their polynomial times X is a whole product
            flops += STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
            nbytes += 2 * m * n * size
        return {"bytes": nbytes, "flops": flops}
    r, v, d = case["rows"], case["classes"], case["width"]
    valid = max(1, round(r * (1.0 - case["ignored"])))
    product = 2 * valid * v * d
    nbytes = valid * d * size + v * d * size + 8 * r + (4 * v if case["bias"] else 0) + (4 * r if case["reduction"] == "none" else 4)
    if not case["backward"]:
        return {"bytes": nbytes, "flops": product}
    nbytes += r * d * size + v * d * size + (4 * v if case["bias"] else 0)
    return {"bytes": nbytes, "flops": 3 * product}


# ----------------------------------------------------------------------------- inputs
def _update(gen, m, n, dtype):
    """A momentum buffer as it looks in training: a few strong directions over noise, rows of unlike size."""
    dev = gen.device
    r = max(1, min(m, n) // 8)
    noise = torch.randn(m, n, generator=gen, device=dev) * (0.5 * torch.exp(0.7 * torch.randn(m, 1, generator=gen, device=dev)))
    signal = torch.randn(m, r, generator=gen, device=dev) @ torch.randn(r, n, generator=gen, device=dev) / math.sqrt(r)
    return (0.01 * (noise + signal)).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "newton_schulz":
        return {"op": "newton_schulz", "updates": [_update(gen, m, n, dtype) for m, n in _shapes(case)]}
    r, v, d = case["rows"], case["classes"], case["width"]
    labels = torch.randint(0, v, (r,), generator=gen, device=dev)
    weight = torch.randn(v, d, generator=gen, device=dev) * (1.5 / math.sqrt(d))
    # features that lean towards their own class, as those of a network in training do (its logit stands some 4 above the mean)
    x = torch.randn(r, d, generator=gen, device=dev) + 2.7 * torch.nn.functional.normalize(weight[labels], dim=1)
    drop = torch.rand(r, generator=gen, device=dev) < case["ignored"]
    drop[0] = False
    labels = torch.where(drop, torch.full_like(labels, IGNORE), labels)
    bias = torch.randn(v, generator=gen, device=dev) * 0.2 if case["bias"] else None
    each = torch.randn(r, generator=gen, device=dev)             # the upstream gradient of each row's loss
    # what reaches the loss from above: one, or the loss scale that keeps half-precision gradients in range
    above = 1.0
    if case["dtype"] == "float16":
        above = 4096.0 if case["reduction"] == "mean" else min(1.0, 4096.0 / r)
    above = each if case["reduction"] == "none" else torch.tensor(above, device=dev)
    state = {"op": "linear_ce", "x": x.to(dtype), "weight": weight.to(dtype), "bias": bias, "labels": labels, "above": above,
             "reduction": case["reduction"], "backward": case["backward"]}
    if case["backward"]:
        for k in ("x", "weight", "bias"):
            if state[k] is not None:
                state[k].requires_grad_(True)
    return state


# ----------------------------------------------------------------------------- one pass
def _plain_ns(update):
    x = update.float()
    if x.shape[0] > x.shape[1]:
        x = x.t()
    x = x / (x.double().square().sum().sqrt() + EPS).float()
    a, b, c = COEFFS
    for _ in range(STEPS):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    if update.shape[0] > update.shape[1]:
        x = x.t()
    return x.to(update.dtype).contiguous()


def _plain_ce(s):
    with torch.no_grad():
        x, w, labels = s["x"].float(), s["weight"].float(), s["labels"]
        valid = labels != IGNORE
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"]
        at = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
        top = z.max(dim=1, keepdim=True).values
        picked = z.gather(1, at)
        z = torch.exp(z - top)
        total = z.double().sum(dim=1, keepdim=True).float()
        rows = torch.where(valid, (top + torch.log(total) - picked)[:, 0], torch.zeros_like(top[:, 0]))
        if s["reduction"] == "none":
            loss, scale = rows, s["above"]
        else:
            count = valid.sum() if s["reduction"] == "mean" else torch.ones_like(valid.sum())
            loss = (rows.double().sum() / count).float()
            scale = (s["above"] / count).expand(rows.shape)
        if not s["backward"]:
            return {"loss": loss}
        z = z / total
        z.scatter_add_(1, at, torch.full_like(picked, -1.0))
        z = z * torch.where(valid, scale, torch.zeros_like(scale))[:, None]
        out = {"loss": loss, "dx": (z @ w).to(s["x"].dtype), "dweight": (z.t() @ x).to(s["weight"].dtype)}
        if s["bias"] is not None:
            out["dbias"] = z.double().sum(dim=0).float()
        return out


def _own_ce(s):
    from fedicra_amd import ops
    if not s["backward"]:
        with torch.no_grad():
            return {"loss": ops.linear_ce_loss(s["x"], s["weight"], s["bias"], s["labels"], IGNORE, s["reduction"])}
    loss = ops.linear_ce_loss(s["x"], s["weight"], s["bias"], s["labels"], IGNORE, s["reduction"])
    leaves = [s["x"], s["weight"]] + ([] if s["bias"] is None else [s["bias"]])
    grads = torch.autograd.grad(loss, leaves, s["above"])
    return dict(zip(("loss", "dx", "dweight", "dbias"), (loss.detach(), *grads)))


def run(state):
    if state["op"] == "newton_schulz":
        if own:
            from fedicra_amd import ops
            return ops.newton_schulz(state["updates"], steps=STEPS, coeffs=COEFFS, eps=EPS)
        return [_plain_ns(u) for u in state["updates"]]
    return _own_ce(state) if own else _plain_ce(state)


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _exact_ns(update):
    x = update.double()
    tall = x.shape[0] > x.shape[1]
    x = x / (torch.linalg.norm(x) + EPS)
    # the odd polynomial a s + b s^3 + c s^5 of the singular values, by Horner's rule on whichever side is the shorter
    a, b, c = COEFFS
    for _ in range(STEPS):
        g = x.t().matmul(x) if tall else x.matmul(x.t())
        poly = b * g + c * g.matmul(g)
        poly.diagonal().add_(a)
        x = x.matmul(poly) if tall else poly.matmul(x)
    return x


def _exact_ce(s):
    x, w, labels = s["x"].detach().double(), s["weight"].detach().double(), s["labels"]
    bias = None if s["bias"] is None else s["bias"].detach().double()
    r, v = x.shape[0], w.shape[0]
    count = int((labels != IGNORE).sum()) if s["reduction"] == "mean" else 1
    rows = torch.zeros(r, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros(v, dtype=torch.float64, device=x.device)
    piece = max(1, int(1.2e8) // v)
    for lo in range(0, r, piece):
        hi = min(r, lo + piece)
        keep = (labels[lo:hi] != IGNORE).nonzero()[:, 0]
        if keep.numel() == 0:
            continue
        xs, ls = x[lo:hi][keep], labels[lo:hi][keep]
        logp = torch.log_softmax(torch.nn.functional.linear(xs, w, bias), dim=1)
        rows[lo + keep] = -logp[torch.arange(len(ls), device=x.device), ls]
        if s["backward"]:
            g = logp.exp_()
            g[torch.arange(len(ls), device=x.device), ls] -= 1.0
            g.mul_((s["above"][lo:hi][keep].double()[:, None] if s["reduction"] == "none" else s["above"].double() / count))
            dx[lo + keep] = g.matmul(w)
            dw.addmm_(g.t(), xs)
            db += g.sum(0)
    out = {"loss": rows if s["reduction"] == "none" else rows.sum() / count}
    if s["backward"]:
        out.update(dx=dx, dweight=dw)
        if bias is not None:
            out["dbias"] = db
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] == "newton_schulz":
        return [_exact_ns(u) for u in state["updates"]]
    with torch.no_grad():
        return _exact_ce(state)
