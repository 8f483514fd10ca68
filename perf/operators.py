"""What is measured of the token operators: layer norm, attention and the learned relative position bias.

The cases are token blocks over the feature maps of this package's detectors: 80 x 80, 40 x 40 and 20 x 20 positions of a
640 x 640 image (76, 38 and 19 at 608 x 608), the 8400 positions of all three levels together, widths of 128 to 1024 channels.
``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, through ``yolo_amd.tokens``.
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ---- cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one image, the tokens of its coarsest map, when a block is served: nothing but latency
        _norm("norm_serve_map20", rows=400, c=512, dtype="bf16", train=False),
        # a batch of 32 images at 40 x 40 when served
        _norm("norm_serve_batch", rows=32 * 1600, c=256, dtype="bf16", train=False),
        # a training step at 40 x 40 and 64 images, float32 weights beside bf16 activations
        _norm("norm_train_batch", rows=64 * 1600, c=512, dtype="bf16", train=True),
        # the head's float32 rows, a channel count that no vector width divides
        _norm("norm_train_odd", rows=17003, c=171, dtype="f32", train=True),
        # one image's coarsest map in a block with a position bias, when served
        _biased("biased_serve_map20", b=1, h=20, w=20, heads=8, d=32, buckets=16, far=20, train=False),
        # the finest map of two images when served: the longest rows
        _biased("biased_serve_map80", b=2, h=80, w=80, heads=8, d=64, buckets=16, far=80, train=False),
        # a training step of a block at 40 x 40
        _biased("biased_train_map40", b=8, h=40, w=40, heads=8, d=64, buckets=16, far=40, train=True),
        # a training step on sequences that are not maps, odd length and head width
        _biased("biased_train_row", b=3, h=1, w=1447, heads=6, d=40, buckets=32, far=128, train=True),
        # one query that pools all three levels' positions of each image, heads that share keys, padded images
        _plain("token_serve", b=8, lq=1, lk=8400, heads=16, kv_heads=4, d=64, mask="padded", train=False),
        # 300 queries of a decoder over all three levels of one image, when served
        _plain("decoder_serve", b=1, lq=300, lk=8400, heads=8, kv_heads=8, d=32, mask="none", train=False),
        # the decoder's training step over a padded batch in which one image is empty
        _plain("decoder_train", b=8, lq=300, lk=8400, heads=8, kv_heads=8, d=32, mask="empty", train=True),
        # the finest map's training step, wide heads that share keys: the largest
        _plain("map80_train", b=2, lq=6400, lk=6400, heads=8, kv_heads=4, d=128, mask="none", train=True),
    ]


def _norm(name, **k):
    return {"name": name, "op": "norm", **k}


def _plain(name, **k):
    return {"name": name, "op": "attention", **k}


def _biased(name, **k):
    return {"name": name, "op": "biased", **k}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    most = 14 * 2 * 8 * 6400 * 6400 * 128          # products of the largest listed case
    op = rng.choice(["norm", "attention", "biased"])
    train = rng.random() < 0.5
    if op == "norm":
        c = _log(rng, 8, 4096)
        if rng.random() < 0.6:
            c = max(8, c // 8 * 8)
        rows = _log(rng, 1, min(102400, 52428800 // c))
        case = {"op": op, "rows": rows, "c": c, "dtype": rng.choice(["bf16", "f32"]), "train": train}
    elif op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        case = {"op": op, "b": _log(rng, 1, 8), "lq": _log(rng, 1, 6400), "lk": _log(rng, 1, 8400),
                "heads": kv * rng.choice([1, 1, 2, 4]), "kv_heads": kv, "d": 8 * rng.randint(2, 16),
                "mask": rng.choice(["none", "padded", "empty"]), "train": train}
    else:
        flat = rng.random() < 0.3
        h = 1 if flat else rng.randint(5, 80)
        w = _log(rng, 30, 4000) if flat else rng.randint(5, 80)
        case = {"op": op, "b": _log(rng, 1, 8), "h": h, "w": w, "heads": rng.choice([1, 2, 4, 6, 8]), "d": 8 * rng.randint(2, 16),
                "buckets": rng.choice([8, 16, 32]) if flat else rng.choice([8, 16]), "far": max(16, w), "train": train}
    if op != "norm":
        while work(case)["flops"] > most // 2 and case["b"] > 1:
            case["b"] -= 1
        while work(case)["flops"] > most // 2:
            case["heads"] //= 2
            if "kv_heads" in case:
                case["kv_heads"] = max(1, min(case["kv_heads"], case["heads"]))
    return case


def _dims(case):
    """(lq, lk, key/value heads) of an attention case."""
    if case["op"] == "biased":
        n = case["h"] * case["w"]
        return n, n, case["heads"]
    return case["lq"], case["lk"], case["kv_heads"]


def _valid_keys(case):
    """How many keys each image of the batch has (the rest of its row is padding)."""
    _, lk, _ = _dims(case)
    b, kind = case["b"], case.get("mask", "none")
    if kind == "none":
        return [lk] * b
    n = [max(1, lk - (lk * i) // (2 * b)) for i in range(b)]
    if kind == "empty":
        n[-1] = 0
    return n


def work(case):
    if case["op"] == "norm":
        n, c, e = case["rows"], case["c"], 2 if case["dtype"] == "bf16" else 4
        if case["train"]:      # x and dy read, y and dx written
            return {"bytes": 4 * n * c * e + 4 * c * 4, "flops": 20 * n * c}
        return {"bytes": 2 * n * c * e + 2 * c * 4, "flops": 8 * n * c}
    lq, lk, kv = _dims(case)
    b, h, d = case["b"], case["heads"], case["d"]
    pairs = sum(_valid_keys(case)) * lq * h
    q, k = b * lq * h * d * 2, b * lk * kv * d * 2
    if case["train"]:          # q, k, v, do read; o, dq, dk, dv written
        return {"bytes": 4 * q + 4 * k, "flops": 14 * pairs * d}
    return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs * d}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _axis_bucket(delta, n, far):
    """Bucket of a signed distance along one axis: half of the n buckets for each sign; the first half of those hold one
    distance each, the others grow by a constant factor up to ``far``.  Whole-number comparisons only."""
    half = n // 2
    near = half // 2
    m = abs(delta)
    if m < near:
        f = m
    else:
        t, steps = 0, half - near
        while t + 1 < steps and m ** steps * near ** (t + 1) >= near ** steps * far ** (t + 1):
            t += 1
        f = near + t
    return (half if delta > 0 else 0) + f


def _buckets(case):
    """(n, n) bucket of every pair of positions (query row, key column), and the number of buckets."""
    h, w, nb, far = case["h"], case["w"], case["buckets"], case["far"]
    bx = torch.tensor([_axis_bucket(x, nb, far) for x in range(-(w - 1), w)], device=DEV)
    ix = torch.arange(w, device=DEV)
    ax = bx[ix[:, None] - ix[None, :] + w - 1]
    if h == 1:
        return ax, nb
    by = torch.tensor([_axis_bucket(y, nb, far) for y in range(-(h - 1), h)], device=DEV)
    iy = torch.arange(h, device=DEV)
    ay = by[iy[:, None] - iy[None, :] + h - 1]
    return (ay[:, None, :, None] * nb + ax[None, :, None, :]).reshape(h * w, h * w), nb * nb


def prepare(case, seed):
    g = _gen(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "norm":
        rows, c, train = case["rows"], case["c"], case["train"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # activations after a conv: channels differ in level and spread
        x = (normal(rows, c) * (0.5 + normal(c).abs()) + 0.5 * normal(c)).to(dt)
        s = {"case": case, "x": x, "weight": 1 + 0.2 * normal(c), "bias": 0.2 * normal(c), "eps": 1e-5}
        if train:
            s["dy"] = normal(rows, c).to(dt)
            for n in ("x", "weight", "bias"):
                s[n].requires_grad_(True)
        return s
    lq, lk, kv = _dims(case)
    b, heads, d = case["b"], case["heads"], case["d"]
    s = {"case": case, "q": (1.5 * normal(b, lq, heads, d)).bfloat16(), "k": normal(b, lk, kv, d).bfloat16(),
         "v": normal(b, lk, kv, d).bfloat16(), "scale": 1 / math.sqrt(d)}
    s["mask"] = None
    if case.get("mask", "none") != "none":
        n = torch.tensor(_valid_keys(case), device=DEV)
        s["mask"] = torch.arange(lk, device=DEV)[None, :] < n[:, None]
    names = ["q", "k", "v"]
    if case["op"] == "biased":
        # the table of a bias, in the type of the activations, and the map from distances to its rows
        n = case["buckets"] if case["h"] == 1 else case["buckets"] ** 2
        s["table"] = (0.5 * normal(n, heads)).bfloat16()
        names.append("table")
        if own:
            from yolo_amd import tokens
            s["position"] = tokens.RelativePosition(case["h"], case["w"], case["buckets"], case["far"], device=DEV)
        else:
            s["bucket"], _ = _buckets(case)
            if case["train"]:
                flat = s["bucket"].reshape(-1)
                s["order"] = torch.argsort(flat, stable=True)
                s["ends"] = torch.cumsum(torch.bincount(flat, minlength=n), 0)
    if case["train"]:
        s["do"] = normal(b, lq, heads, d).bfloat16()
        for n in names:
            s[n].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_attention(state) if own else _plain_attention(state)


def _own_norm(s):
    from yolo_amd import tokens
    y = tokens.layer_norm(s["x"], s["weight"], s["bias"], s["eps"])
    if not s["case"]["train"]:
        return y
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _own_attention(s):
    from yolo_amd import tokens
    case = s["case"]
    given = {"scale": s["scale"], "key_mask": s["mask"]}
    if case["op"] == "biased":
        given["bias"] = tokens.relative_bias(s["table"], s["position"])
        given["position"] = s["position"]
    o = tokens.attention(s["q"], s["k"], s["v"], **given)
    if not case["train"]:
        return o
    names = ["q", "k", "v"] + (["table"] if case["op"] == "biased" else [])
    grads = torch.autograd.grad(o, [s[n] for n in names], s["do"])
    return {"o": o.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


@torch.no_grad()
def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
    unit = centred * rstd
    y = (unit * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * unit).sum(0), "db": dy.sum(0)}


@torch.no_grad()
def _plain_attention(s):
    case = s["case"]
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    b, heads, lq, d = q.shape
    kv, lk = k.shape[1], k.shape[2]
    group = heads // kv
    k, v = (t.repeat_interleave(group, 1).contiguous() for t in (k, v))
    p = torch.matmul(q * s["scale"], k.transpose(2, 3).contiguous())
    if case["op"] == "biased":
        p += s["table"].float().t()[:, s["bucket"]]
    if s["mask"] is not None:
        p.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    top = p.amax(3, keepdim=True)
    p = torch.exp_(p.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(3, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(s["q"].dtype).contiguous()
    if not case["train"]:
        return out
    do = s["do"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds -= (do * o).sum(3, keepdim=True)
    ds *= p
    del p
    res = {"o": out, "dq": torch.matmul(ds, k) * s["scale"]}
    res["dk"] = torch.matmul(ds.transpose(2, 3).contiguous(), q).view(b, kv, group, lk, d).sum(2) * s["scale"]
    res["dv"] = dv.view(b, kv, group, lk, d).sum(2)
    for n in ("dq", "dk", "dv"):
        res[n] = res[n].transpose(1, 2).to(s["q"].dtype).contiguous()
    if case["op"] == "biased":
        # sums over all pairs of a bucket: differences of a running sum in 64 bits, along the pairs in order of bucket
        run_sum = ds.sum(0).view(heads, -1)[:, s["order"]].double().cumsum_(1)
        at = run_sum[:, (s["ends"] - 1).clamp(min=0)] * (s["ends"] > 0)
        res["dtable"] = torch.diff(at, dim=1, prepend=at.new_zeros(heads, 1)).t().to(s["table"].dtype).contiguous()
    return res


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"] == "norm" else _exact_attention(s)


def _exact_norm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    n = x.shape[1]
    mu = x.sum(1) / n
    var = ((x - mu[:, None]) ** 2).sum(1) / n
    inv = 1 / torch.sqrt(var + s["eps"])
    xh = (x - mu[:, None]) * inv[:, None]
    y = xh * w + b
    if not s["case"]["train"]:
        return y
    dy = s["dy"].double()
    dxh = dy * w
    dvar = -0.5 * inv ** 3 * (dxh * (x - mu[:, None])).sum(1)
    dmu = -inv * dxh.sum(1)
    dx = dxh * inv[:, None] + (2 / n) * dvar[:, None] * (x - mu[:, None]) + dmu[:, None] / n
    return {"y": y, "dx": dx, "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _exact_attention(s):
    """One image and one head at a time."""
    case = s["case"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    o = torch.zeros_like(q)
    res = {"o": o}
    if case["train"]:
        do = s["do"].double()
        res.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    biased = case["op"] == "biased"
    if biased:
        bucket, rows = _buckets(case)
        order = torch.argsort(bucket.reshape(-1), stable=True)
        sizes = torch.bincount(bucket.reshape(-1), minlength=rows).tolist()
        if case["train"]:
            res["dtable"] = torch.zeros(s["table"].shape, dtype=torch.float64, device=DEV)
    group = q.shape[2] // k.shape[2]
    for i in range(case["b"]):
        seen = slice(None) if s["mask"] is None else s["mask"][i].nonzero()[:, 0]
        if s["mask"] is not None and seen.numel() == 0:
            continue
        for h in range(q.shape[2]):
            ki, vi = k[i, seen, h // group], v[i, seen, h // group]
            z = s["scale"] * (q[i, :, h] @ ki.t())
            if biased:
                z = z + s["table"][:, h].double()[bucket]
            z = torch.softmax(z, 1)
            o[i, :, h] = z @ vi
            if not case["train"]:
                continue
            g = do[i, :, h]
            res["dv"][i, seen, h // group] += z.t() @ g
            dz = g @ vi.t()
            dz = z * (dz - (z * dz).sum(1, keepdim=True))
            res["dq"][i, :, h] = s["scale"] * (dz @ ki)
            res["dk"][i, seen, h // group] += s["scale"] * (dz.t() @ q[i, :, h])
            if biased:
                parts = dz.reshape(-1)[order].split(sizes)
                res["dtable"][:, h] += torch.stack([t.sum() for t in parts])
    return res if case["train"] else o
