"""What is measured of three operators of the training and inference path, and what they compute:

  norm   layer normalisation over the channels of feature rows, y = (x - mean) / sqrt(var + eps) * weight + bias, and its backward pass
  group  products of feature rows with the weight of the group (class, domain, expert) that each row belongs to, the groups' row counts
         known on the device only, and its backward pass: y[i] = weight[g(i)] x[i] + bias[g(i)]
  clip   the global L2 norm over a list of gradient tensors, and clipping to a largest norm

With `own` false `run` computes them from elementary torch operations in 32 bits (64 for the norm's long sum), with `own` true it makes
the calls of uemda_amd that a user makes.  `exact` gives the same in 64 bits."""
import math

import torch

own = False

EPS = 1e-5
MAX_NORM = 32.0          # the training scripts' clip_grad_norm_ bound
# what a drawn case may cost at most: the largest listed ones
NORM_MOST = 32768 * 2048
GROUP_MOST = 65536 * 2048 * 2048
CLIP_MOST = 400_000_000


# ---- cases -----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one pooled feature vector of a tile at inference: nothing but latency
        dict(name="norm_one_row", op="norm", rows=1, channels=2048, dtype="bfloat16", train=False),
        # the encoder's last map of 32 tiles of 512 x 512 (stride 16, 2048 channels) in a training step, 32-bit storage
        dict(name="norm_feature_map", op="norm", rows=32768, channels=2048, dtype="float32", train=True),
        # layer1's map of the same 32 tiles (stride 4, 256 channels) in a training step, 16-bit storage
        dict(name="norm_layer1_map", op="norm", rows=524288, channels=256, dtype="bfloat16", train=True),
        # the pixels of a cropped tile, an odd channel count: no row but the first is aligned
        dict(name="norm_odd", op="norm", rows=9409, channels=777, dtype="bfloat16", train=True),
        # a handful of pooled regions through per-class projections at inference: the weights are all there is to read
        dict(name="group_few_rows", op="group", rows=9, groups=6, k=2048, n=512, dtype="bfloat16", train=False, spread=0.5, tail=0.0),
        # the pixels of 32 tiles grouped by their pseudo label (7 classes of very unequal size, a fifth of the pixels ignored) through
        # per-class projections 2048 -> 512, training step
        dict(name="group_by_class", op="group", rows=32768, groups=7, k=2048, n=512, dtype="bfloat16", train=True, spread=1.5, tail=0.2),
        # the same kind of head in 32-bit storage on 8 tiles
        dict(name="group_fp32", op="group", rows=8192, groups=6, k=512, n=512, dtype="float32", train=True, spread=1.0, tail=0.1),
        # a layer of many experts, training step: the largest product
        dict(name="group_experts", op="group", rows=65536, groups=32, k=2048, n=2048, dtype="bfloat16", train=True, spread=0.7, tail=0.0),
        # odd everything: rows, widths, some groups empty
        dict(name="group_odd", op="group", rows=5003, groups=19, k=333, n=77, dtype="bfloat16", train=True, spread=2.5, tail=0.05),
        # the gradients of one small head: latency
        dict(name="clip_head", op="clip", kind="head", numel=4 * 55296, tensors=8, bf16_share=0.0),
        # the gradients of a ResNet-50 with its two heads as one tensor each
        dict(name="clip_encoder", op="clip", kind="encoder", numel=0, tensors=0, bf16_share=0.0),
        # many tensors of mixed type, odd sizes and alignments, the size of a large model
        dict(name="clip_mixed", op="clip", kind="mixed", numel=400_000_000, tensors=600, bf16_share=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "group", "group", "group", "clip"])
    if op == "norm":
        channels = _log_int(rng, 1, 8192)
        if rng.random() < 0.5:
            channels = max(8, channels // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(524288, NORM_MOST // channels)))
        return dict(op="norm", rows=rows, channels=channels, dtype=rng.choice(["float32", "bfloat16"]), train=rng.random() < 0.7)
    if op == "group":
        k, n = _log_int(rng, 16, 2048), _log_int(rng, 16, 2048)
        if rng.random() < 0.6:
            k, n = max(16, k // 16 * 16), max(16, n // 16 * 16)
        dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
        most = GROUP_MOST // (12 if dtype == "float32" else 1)
        rows = _log_int(rng, 1, max(1, min(65536, most // (k * n))))
        return dict(op="group", rows=rows, groups=_log_int(rng, 1, 64), k=k, n=n, dtype=dtype, train=rng.random() < 0.7,
                    spread=rng.choice([0.0, 0.7, 1.5, 2.5]), tail=rng.choice([0.0, 0.0, 0.1, 0.3]))
    return dict(op="clip", kind="mixed", numel=_log_int(rng, 1000, CLIP_MOST // 4), tensors=_log_int(rng, 1, 400),
                bf16_share=rng.choice([0.0, 0.3, 1.0]))


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _encoder_sizes():
    """(shape) of every parameter of a ResNet-50 without its classifier and of two heads of four dilated 3 x 3 convolutions to 6 classes"""
    shapes = [(64, 3, 7, 7), (64,), (64,)]
    cin = 64
    for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for b in range(blocks):
            shapes += [(width, cin, 1, 1), (width,), (width,), (width, width, 3, 3), (width,), (width,),
                       (4 * width, width, 1, 1), (4 * width,), (4 * width,)]
            if b == 0:
                shapes += [(4 * width, cin, 1, 1), (4 * width,), (4 * width,)]
            cin = 4 * width
    return shapes + [(6, 2048, 3, 3), (6,)] * 8


def _sizes(case):
    """[(elements, is bf16)] of the gradient list: a function of the case alone"""
    if case["kind"] == "encoder":
        return [(math.prod(s), False) for s in _encoder_sizes()]
    if case["kind"] == "head":
        return [(case["numel"] // 4, False), (6, False)] * (case["tensors"] // 2)
    # sizes over several orders of magnitude: shares of 1, 1/2, .. in a fixed pattern, odd remainders
    n = case["tensors"]
    shares = [1.0 / (1 + (i * 7) % 40) ** 2 for i in range(n)]
    total = sum(shares)
    return [(max(1, int(case["numel"] * s / total)), (i * 5) % 10 < 10 * case["bf16_share"]) for i, s in enumerate(shares)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _bounds(case, seed):
    """row offsets of the groups, on the host: log-normal shares, `tail` of the rows behind the last group"""
    g = torch.Generator().manual_seed(seed * 2 + 1)
    rows = case["rows"] - int(case["rows"] * case["tail"])
    share = torch.exp(case["spread"] * torch.randn(case["groups"], generator=g, dtype=torch.float64))
    ends = torch.floor(torch.cumsum(share, 0) / share.sum() * rows).to(torch.int64)
    ends[-1] = rows
    return [0] + ends.tolist()


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "norm":
        dtype = getattr(torch, case["dtype"])
        rows, c = case["rows"], case["channels"]
        # feature rows have a mean and a scale of their own
        x = torch.randn((rows, c), generator=g, device="cuda")
        x = x.mul_(torch.rand((rows, 1), generator=g, device="cuda") * 2 + 0.1).add_(torch.randn((rows, 1), generator=g, device="cuda"))
        w = 1 + _normal(g, (c,), torch.float32, 0.2)
        b = _normal(g, (c,), torch.float32, 0.2)
        state = dict(op="norm", train=case["train"], x=x.to(dtype), w=w, b=b)
        if case["train"]:
            state["dy"] = _normal(g, (rows, c), dtype)
            for name in ("x", "w", "b"):
                state[name].requires_grad_()
        return state
    if case["op"] == "group":
        dtype = getattr(torch, case["dtype"])
        rows, groups, k, n = case["rows"], case["groups"], case["k"], case["n"]
        bounds = _bounds(case, seed)
        state = dict(op="group", train=case["train"], bounds=bounds, offsets=torch.tensor(bounds, dtype=torch.int32, device="cuda"),
                     x=_normal(g, (rows, k), dtype), w=_normal(g, (groups, n, k), dtype, k ** -0.5), b=_normal(g, (groups, n), dtype, 0.1))
        if case["train"]:
            state["dy"] = _normal(g, (rows, n), dtype)
            for name in ("x", "w", "b"):
                state[name].requires_grad_()
        return state
    sizes = _sizes(case)
    flats, lists = [], []
    for dtype, is16, step in ((torch.float32, False, 4), (torch.bfloat16, True, 8)):
        mine = [n for n, b in sizes if b == is16]
        if not mine:
            continue
        # each tensor in its own place of one allocation; in the mixed list the places are not aligned to more than an element
        places, at = [], 0
        for n in mine:
            places.append((at, n))
            at += n if case["kind"] == "mixed" else (n + step - 1) // step * step
        flat = _normal(g, (at,), dtype, 0.05)
        for (a, n), nxt in zip(places, [p for p, _ in places[1:]] + [at]):
            flat[a + n:nxt] = 0                                                  # the gaps behind the tensors hold no gradient
        flats.append(flat)
        lists += [flat[a:a + n] for a, n in places]
    params = []
    for t in lists:
        p = torch.empty_like(t, memory_format=torch.contiguous_format).requires_grad_()
        p.grad = t
        params.append(p)
    # the bound falls a little from call to call, so that every call finds something to clip
    return dict(op="clip", params=params, flats=flats, max_norm=min(MAX_NORM, 0.01 * math.sqrt(sum(n for n, _ in sizes))))


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    if state["op"] == "group":
        return _group_own(state) if own else _group_plain(state)
    max_norm = state["max_norm"]
    state["max_norm"] = max_norm * 0.9999
    norm = _clip_own(state["params"], max_norm) if own else _clip_plain([p.grad for p in state["params"]], max_norm)
    return [norm] + state["flats"]


def _norm_own(s):
    from uemda_amd.norm import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], EPS)
    if not s["train"]:
        return [y]
    return [y] + list(torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))


@torch.no_grad()
def _norm_plain(s):
    x, w = s["x"].float(), s["w"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * w + s["b"].float()).to(s["x"].dtype)
    if not s["train"]:
        return [y]
    dy = s["dy"].float()
    dw, db = (dy * hat).sum(0), dy.sum(0)
    dhat = dy * w
    dx = rstd * (dhat - dhat.mean(1, keepdim=True) - hat * (dhat * hat).mean(1, keepdim=True))
    return [y, dx.to(s["x"].dtype), dw, db]


def _group_own(s):
    from uemda_amd.grouped import grouped_linear
    y = grouped_linear(s["x"], s["w"], s["offsets"], s["b"])
    if not s["train"]:
        return [y]
    return [y] + list(torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))


@torch.no_grad()
def _group_plain(s):
    x, w, b = s["x"], s["w"], s["b"]
    y = torch.zeros((x.shape[0], w.shape[1]), device=x.device, dtype=x.dtype)
    spans = [(i, lo, hi) for i, (lo, hi) in enumerate(zip(s["bounds"], s["bounds"][1:])) if hi > lo]
    for i, lo, hi in spans:
        y[lo:hi] = torch.mm(x[lo:hi].float(), w[i].float().t()) + b[i].float()
    if not s["train"]:
        return [y]
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i, lo, hi in spans:
        dy = s["dy"][lo:hi].float()
        dx[lo:hi] = torch.mm(dy, w[i].float())
        dw[i] = torch.mm(dy.t(), x[lo:hi].float())
        db[i] = dy.sum(0)
    return [y, dx, dw, db]


def _clip_own(params, max_norm):
    from uemda_amd.optim import clip_grad_norm_
    return clip_grad_norm_(params, max_norm)


@torch.no_grad()
def _clip_plain(grads, max_norm):
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    coef = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    for g in grads:
        g.copy_(g.float() * coef)
    return norm


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        rows, c, e = case["rows"], case["channels"], 4 if case["dtype"] == "float32" else 2
        # x in, y out; training: dy in, dx out, the weight's and bias's gradients
        maps = 4 if case["train"] else 2
        return dict(bytes=maps * rows * c * e + (4 if case["train"] else 2) * 4 * c, flops=(20 if case["train"] else 8) * rows * c)
    if case["op"] == "group":
        rows, e = case["rows"], 4 if case["dtype"] == "float32" else 2
        used = rows - int(rows * case["tail"])
        g, k, n = case["groups"], case["k"], case["n"]
        x, y, w = rows * k * e, rows * n * e, (k * n + n) * e * min(g, used)
        once = 2 * used * k * n
        return dict(bytes=2 * x + 2 * y + 2 * w, flops=3 * once) if case["train"] else dict(bytes=x + y + w, flops=once)
    sizes = _sizes(case)
    return dict(bytes=2 * sum(n * (2 if b else 4) for n, b in sizes) + 4, flops=3 * sum(n for n, _ in sizes))


# ---- in 64 bits --------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        c = x.shape[1]
        mu = x.sum(1) / c
        sigma = (x.sub(mu[:, None]).pow(2).sum(1) / c + EPS).sqrt()
        z = (x - mu[:, None]) / sigma[:, None]
        y = torch.addcmul(s["b"].double(), z, s["w"].double())
        if not case["train"]:
            return [y]
        g = s["dy"].double()
        out = [y, None, torch.einsum("rc,rc->c", g, z), torch.einsum("rc->c", g)]
        g = g * s["w"].double()
        # d/dx of the projection orthogonal to (1, z)
        along = torch.einsum("rc,rc->r", g, z) / c
        out[1] = (g - (g.sum(1) / c)[:, None] - z * along[:, None]) / sigma[:, None]
        return out
    if case["op"] == "group":
        ends = torch.tensor(s["bounds"][1:], device="cuda")
        rows = torch.arange(case["rows"], device="cuda")
        owner = torch.searchsorted(ends, rows, right=True)               # == groups: behind the last one
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        y = torch.zeros((case["rows"], case["n"]), device="cuda", dtype=torch.float64)
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
        for i in range(case["groups"]):
            at = (owner == i).nonzero().flatten()
            if at.numel() == 0:
                continue
            y[at] = torch.addmm(b[i], x[at], w[i].t())
            if case["train"]:
                g = s["dy"][at].double()
                dx[at] = g @ w[i]
                dw[i] = (x[at].t() @ g).t()
                db[i] = g.sum(0)
        return [y, dx, dw, db] if case["train"] else [y]
    total = math.sqrt(sum(float(f.double().pow(2).sum()) for f in s["flats"]))
    scale = min(1.0, s["max_norm"] / (total + 1e-6))
    return [torch.tensor(total, dtype=torch.float64, device="cuda")] + [f.double() * scale for f in s["flats"]]
