"""Cases for the row operators of a training or matching step: the root-mean-square norm with the residual's addition (and its 8-bit
form), log probabilities of given candidates with entropy and the best alternatives, and the clipped global gradient norm over many
tensors.  `own` chooses between the plain torch form and the calls into i2pnet_amd."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3_MAX = 448.0
EPS = 1e-6

# (elements, tensors) of the registration network's parameters: 254 tensors, 844 896 elements
NETWORK = [(64, 87), (128, 48), (32, 24), (16, 18), (8192, 12), (256, 5), (4096, 4), (9216, 4), (36864, 4), (32768, 4), (16384, 3), (8576, 3),
           (2304, 3), (1, 2), (384, 2), (640, 2), (12288, 2), (16384, 2), (1024, 2), (4, 2), (768, 2), (3, 2), (160, 1), (256, 1), (512, 1),
           (1120, 1), (1024, 1), (2048, 1), (4288, 1), (8192, 1), (16768, 1), (32768, 1), (432, 1), (4608, 1), (18432, 1), (73728, 1),
           (33536, 1), (17152, 1), (40960, 1)]


def listed():
    return [
        # one token of a served model: the whole call is latency
        {"name": "norm one token", "op": "norm", "mode": "fwd", "rows": 1, "d": 4096, "dtype": "bf16", "residual": True, "group": 0},
        # features of the first grouping level at batch 8 (3600 points each), 64 channels in 32 bits, forward and backward
        {"name": "norm train features", "op": "norm", "mode": "train", "rows": 28800, "d": 64, "dtype": "fp32", "residual": True, "group": 0},
        # a training step's rows, wide, forward and backward through the residual stream
        {"name": "norm train wide", "op": "norm", "mode": "train", "rows": 8192, "d": 4096, "dtype": "bf16", "residual": True, "group": 0},
        # a prompt whose rows go to an 8-bit product, one scale for 128 columns; the width is no multiple of the group
        {"name": "norm 8 bits", "op": "norm", "mode": "q8", "rows": 6001, "d": 5000, "dtype": "bf16", "residual": True, "group": 128},
        # one token over a large vocabulary, with the eight best alternatives: the whole call is latency
        {"name": "logp one token", "op": "logp", "mode": "fwd", "rows": 1, "v": 131072, "dtype": "fp32", "top": 8, "mask": "none"},
        # the coarse cost volume's pairs at batch 8: 228 points each against 468 pixels, some pixels masked out, with gradients
        {"name": "logp match train", "op": "logp", "mode": "train", "rows": 1824, "v": 468, "dtype": "fp32", "top": 0, "mask": "inf"},
        # scoring a batch of answers: odd width, a mask of the type's lowest value, five alternatives
        {"name": "logp score", "op": "logp", "mode": "fwd", "rows": 777, "v": 50001, "dtype": "fp16", "top": 5, "mask": "lowest"},
        # a training step's loss with its gradient, an ordinary and a large vocabulary
        {"name": "logp train", "op": "logp", "mode": "train", "rows": 4096, "v": 32000, "dtype": "bf16", "top": 0, "mask": "none"},
        {"name": "logp train large", "op": "logp", "mode": "train", "rows": 8192, "v": 131072, "dtype": "bf16", "top": 0, "mask": "none"},
        # the registration network's own gradients, in place; the ordinary step, whose norm is within the limit
        {"name": "clip network", "op": "clip", "mode": "place", "n": 254, "numel": 844896, "dtype": "fp32", "limit": 4.0},
        # a few odd tensors, gathered into the flat 32-bit gradient that is reduced and stepped; clipped
        {"name": "clip few", "op": "clip", "mode": "into", "n": 5, "numel": 70001, "dtype": "bf16", "limit": 0.1},
        # a large model's gradients in 16 bits, some of them in 32; clipped
        {"name": "clip large", "op": "clip", "mode": "into", "n": 291, "numel": 300000007, "dtype": "bf16", "limit": 0.1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "logp", "clip"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "norm":
        d = _log(rng, 16, 16384)
        if rng.random() < 0.5:
            d = (d + 7) // 8 * 8
        rows = _log(rng, 1, max(2, min(30000, (1 << 25) // d)))
        mode = rng.choice(["fwd", "train", "q8"])
        return {"op": op, "mode": mode, "rows": rows, "d": d, "dtype": dtype, "residual": rng.random() < 0.7,
                "group": rng.choice([0, 64, 128]) if mode == "q8" else 0}
    if op == "logp":
        v = _log(rng, 100, 200000)
        rows = _log(rng, 1, max(2, min(8192, (1 << 28) // v)))
        mode = rng.choice(["fwd", "train"])
        return {"op": op, "mode": mode, "rows": rows, "v": v, "dtype": dtype, "top": rng.choice([0, 1, 5, 8, 20]) if mode == "fwd" else 0,
                "mask": rng.choice(["none", "inf", "lowest"])}
    n = _log(rng, 1, 600)
    numel = _log(rng, n * 8, max(n * 16, 1 << 27))
    return {"op": op, "mode": rng.choice(["place", "into"]), "n": n, "numel": numel, "dtype": dtype, "limit": rng.choice([0.1, 4.0])}


def _sizes(case):
    """the tensors' sizes: the network's own, or `n` of them that add up to `numel`, spread over a factor of about a thousand"""
    if case["n"] == 254 and case["numel"] == 844896:
        return [k for k, times in NETWORK for _ in range(times)]
    rng = random.Random(case["n"] * 1000003 + case["numel"])
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["n"])]
    total = sum(share)
    sizes = [max(1, int(case["numel"] * s / total)) for s in share]
    big = max(range(len(sizes)), key=sizes.__getitem__)
    sizes[big] += case["numel"] - sum(sizes)
    return sizes


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        out = torch.empty(*shape, dtype=dtype, device=dev)
        return out.normal_(0.0, scale, generator=g)

    st = dict(case)
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        st["x"] = randn(rows, d)
        st["r"] = randn(rows, d, scale=2.0) if case["residual"] else None
        st["w"] = (1.0 + 0.1 * torch.randn(d, device=dev, generator=g)).contiguous()
        if case["mode"] == "train":
            st["gy"] = randn(rows, d)
            st["gs"] = randn(rows, d) if case["residual"] else None
            for k in ("x", "r", "w"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
    elif case["op"] == "logp":
        rows, v = case["rows"], case["v"]
        x = randn(rows, v, scale=2.0)
        ids = torch.randint(0, v, (rows,), device=dev, generator=g)
        # a trained model's rows: the given candidate is often likely
        x.scatter_add_(1, ids[:, None], (8.0 * torch.rand(rows, 1, device=dev, generator=g)).to(dt))
        if case["mask"] != "none":
            drop = torch.rand(v, device=dev, generator=g) < 0.25
            fill = -math.inf if case["mask"] == "inf" else torch.finfo(dt).min
            kept = x.gather(1, ids[:, None])
            x[:, drop] = fill
            x.scatter_(1, ids[:, None], kept)
        st["x"], st["ids"] = x, ids
        if case["mode"] == "train":
            # the gradients of a scaled sum over the rows, so that 16-bit gradients keep their small values
            st["glp"] = -torch.rand(rows, device=dev, generator=g)
            st["gh"] = 0.01 * torch.randn(rows, device=dev, generator=g)
            x.requires_grad_(True)
    else:
        sizes = _sizes(case)
        n = sum(sizes)
        scale = 1.0 / math.sqrt(n)                          # a norm near one
        if case["mode"] == "place":
            # views of one buffer, each on a boundary of four elements: the trainer's own layout
            at, total = [], 0
            for k in sizes:
                at.append(total)
                total += (k + 3) // 4 * 4
            st["flat"] = randn(total, scale=scale)
            st["grads"] = [st["flat"][a:a + k] for a, k in zip(at, sizes)]
        else:
            # every eighth tensor of a 16-bit list is kept in 32 bits
            st["grads"] = [randn(k, scale=scale, dtype=torch.float32 if i % 8 == 7 else dt) for i, k in enumerate(sizes)]
            st["out"] = torch.empty(n, dtype=torch.float32, device=dev)
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------------------
def _norm_plain(st):
    dt = st["x"].dtype
    x, w = st["x"].detach(), st["w"].detach()
    # the residual stream is kept in the inputs' type; the norm is of the stream
    s = x if st["r"] is None else (x.float() + st["r"].detach().float()).to(dt)
    sf = s.float()
    rstd = torch.rsqrt((sf * sf).mean(-1, keepdim=True) + EPS)
    y32 = sf * rstd * w
    if st["mode"] == "q8":
        q, scale = _quantise(y32, st["group"])
        return [q, scale] + ([] if st["r"] is None else [s])
    out = [y32.to(dt)] + ([] if st["r"] is None else [s])
    if st["mode"] == "train":
        gy = st["gy"].float()
        xhat = sf * rstd
        gw = (gy * xhat).sum(0)
        t = gy * w
        dx = rstd * (t - xhat * (t * xhat).mean(-1, keepdim=True))
        if st["gs"] is not None:
            dx = dx + st["gs"].float()
        out += [dx.to(dt), gw]
    return out


def _quantise(y, group):
    rows, d = y.shape
    group = group or d
    ng = (d + group - 1) // group
    pad = torch.nn.functional.pad(y, (0, ng * group - d)).view(rows, ng, group)
    scale = pad.abs().amax(-1) / E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = (pad / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, ng * group)[:, :d]
    return q.to(torch.float8_e4m3fn).contiguous(), scale


def _logp_plain(st):
    dt = st["x"].dtype
    x = st["x"].detach().float()
    ids = st["ids"][:, None]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    h = log_total - torch.where(e > 0, e * z, torch.zeros_like(e)).sum(-1, keepdim=True) / total
    lp = (z.gather(1, ids) - log_total).squeeze(1)
    out = [lp, h.squeeze(1)]
    if st["top"]:
        # equal values go to the lower index: the value's bits, ordered, above the index's complement
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        col = torch.arange(x.shape[1], device=x.device)
        key = order * (1 << 32) + ((1 << 32) - 1 - col)
        top = torch.topk(key, st["top"], dim=-1, sorted=True).values
        idx = (1 << 32) - 1 - (top & ((1 << 32) - 1))
        out += [z.gather(1, idx) - log_total, idx]
    if st["mode"] == "train":
        glp, gh = st["glp"][:, None], st["gh"][:, None]
        p = e / total
        logp = torch.where(p > 0, z - log_total, torch.zeros_like(z))
        dx = -p * (glp + gh * (logp + h))
        dx.scatter_add_(1, ids, glp)
        out.append(dx.to(dt))
    return out


def _clip_plain(st):
    grads, limit = st["grads"], st["limit"]
    flat = torch.cat([g.reshape(-1).float() for g in grads])
    total = flat.double().square().sum().sqrt().float()
    coef = torch.clamp(limit / (total + EPS), max=1.0)
    if st["mode"] == "place":
        st["grads"] = [g.copy_(g.float() * coef) for g in grads]
        return [total, st["flat"]]
    torch.mul(flat, coef, out=st["out"])
    return [total, st["out"]]


# ---- the framework's calls ------------------------------------------------------------------------------------------------------
def _norm_own(st):
    from i2pnet_amd import modules
    x, w, r = st["x"], st["w"], st["r"]
    if st["mode"] == "q8":
        return list(modules.rms_norm_q8(x, w, residual=r, eps=EPS, group=st["group"]))
    if r is None:
        y = modules.rms_norm(x, w, eps=EPS)
        if st["mode"] == "fwd":
            return [y]
        gx, gw = torch.autograd.grad(y, [x, w], st["gy"])
        return [y.detach(), gx, gw]
    y, s = modules.rms_norm(x, w, residual=r, eps=EPS)
    if st["mode"] == "fwd":
        return [y, s]
    gx, gw = torch.autograd.grad([y, s], [x, w], [st["gy"], st["gs"]])
    return [y.detach(), s.detach(), gx, gw]


def _logp_own(st):
    from i2pnet_amd import loss
    o = loss.token_logprobs(st["x"], st["ids"], top=st["top"])
    if st["mode"] == "train":
        (dx,) = torch.autograd.grad([o.logp, o.entropy], [st["x"]], [st["glp"], st["gh"]])
        return [o.logp.detach(), o.entropy.detach(), dx]
    return [o.logp, o.entropy] + ([o.top_logp, o.top_ids] if st["top"] else [])


def _clip_own(st):
    from i2pnet_amd import train
    if st["mode"] == "place":
        return [train.clip_grad_norm_(st["grads"], st["limit"]), st["flat"]]
    return [train.clip_grad_norm_(st["grads"], st["limit"], out=st["out"]), st["out"]]


def run(state):
    if own:
        return {"norm": _norm_own, "logp": _logp_own, "clip": _clip_own}[state["op"]](state)
    return {"norm": _norm_plain, "logp": _logp_plain, "clip": _clip_plain}[state["op"]](state)


def work(case):
    es = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, r = case["rows"] * case["d"], int(case["residual"])
        if case["mode"] == "q8":
            groups = case["rows"] * (math.ceil(case["d"] / case["group"]) if case["group"] else 1)
            return {"bytes": n * es * (1 + 2 * r) + n + 4 * groups + 4 * case["d"], "flops": 8 * n}
        tensors = 2 + 2 * r + (2 + r if case["mode"] == "train" else 0)
        return {"bytes": n * es * tensors + 4 * case["d"] * (2 if case["mode"] == "train" else 1), "flops": n * (16 if case["mode"] == "train" else 5)}
    if case["op"] == "logp":
        n, train = case["rows"] * case["v"], case["mode"] == "train"
        return {"bytes": n * es * (2 if train else 1) + case["rows"] * (16 + 12 * case["top"] + (8 if train else 0)), "flops": n * (14 if train else 6)}
    n = case["numel"]
    if case["mode"] == "place":                             # within the limit nothing has to be written
        return {"bytes": n * es * (1 if case["limit"] > 1 else 2) + 4, "flops": 2 * n}
    read = sum(k * (4 if i % 8 == 7 else es) for i, k in enumerate(_sizes(case)))
    return {"bytes": read + 4 * n + 4, "flops": 3 * n}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _norm_exact(case, st)
    if case["op"] == "logp":
        return _logp_exact(case, st)
    parts = [t.detach().to(torch.float64).flatten() for t in st["grads"]]
    norm = math.sqrt(math.fsum(float(torch.dot(p, p)) for p in parts))
    factor = min(1.0, case["limit"] / (norm + EPS))
    if case["mode"] == "place":
        buf = st["flat"].to(torch.float64)
        at = 0
        for p in parts:                                     # the padding between tensors is nobody's gradient
            buf[at:at + p.numel()] *= factor
            at += -(-p.numel() // 4) * 4
        return [torch.tensor(norm, dtype=torch.float64), buf]
    return [torch.tensor(norm, dtype=torch.float64), torch.cat(parts).mul_(factor)]


def _norm_exact(case, st):
    f64 = torch.float64
    a, w = st["x"].detach().to(f64), st["w"].detach().to(f64)
    if st["r"] is not None:
        a = (a + st["r"].detach().to(f64)).to(st["x"].dtype).to(f64)
    ms = torch.linalg.vector_norm(a, dim=-1, keepdim=True).square() / a.shape[-1]
    unit = a / torch.sqrt(ms + EPS)
    y = unit * w
    tail = [] if st["r"] is None else [a]
    if case["mode"] == "q8":
        width = case["group"] or case["d"]
        scales, vals = [], []
        for lo in range(0, case["d"], width):
            block = y[:, lo:lo + width]
            s = torch.linalg.vector_norm(block, ord=math.inf, dim=-1, keepdim=True) / E4M3_MAX
            s = torch.where(s == 0, 1.0, s)
            scales.append(s)
            vals.append(block / s)
        return [torch.cat(vals, 1), torch.cat(scales, 1)] + tail
    if case["mode"] == "fwd":
        return [y] + tail
    gy = st["gy"].to(f64)
    # d(unit)/d(a): the part of the weighted gradient along the row is taken out, but for what eps leaves of it
    gw = torch.einsum("rd,rd->d", gy, unit)
    v = gy * w
    along = torch.einsum("rd,rd->r", v, unit)[:, None] / a.shape[-1]
    dx = (v - unit * along) / torch.sqrt(ms + EPS)
    if st["gs"] is not None:
        dx = dx + st["gs"].to(f64)
    return [y] + tail + [dx, gw]


def _logp_exact(case, st):
    f64 = torch.float64
    x, ids = st["x"].detach(), st["ids"]
    rows, v = x.shape
    lp, ent, top_v, top_i, grads = [], [], [], [], []
    step = max(1, (1 << 26) // v)
    for lo in range(0, rows, step):
        a = x[lo:lo + step].to(f64)
        k = ids[lo:lo + step]
        lse = torch.logsumexp(a, dim=-1, keepdim=True)
        logs = a - lse
        probs = logs.exp()
        h = -torch.special.xlogy(probs, probs).sum(-1, keepdim=True)
        lp.append(logs[torch.arange(len(k), device=k.device), k])
        ent.append(h[:, 0])
        if case["top"]:
            vals, idx = [], []
            left = a.clone()
            for _ in range(case["top"]):                    # the first of the largest, then without it
                i = torch.argmax(left, dim=-1, keepdim=True)
                idx.append(i)
                vals.append(logs.gather(1, i))
                left.scatter_(1, i, -math.inf)
            top_v.append(torch.cat(vals, 1))
            top_i.append(torch.cat(idx, 1))
        if case["mode"] == "train":
            glp, gh = st["glp"][lo:lo + step, None].to(f64), st["gh"][lo:lo + step, None].to(f64)
            dx = -probs * glp - gh * (torch.special.xlogy(probs, probs) + probs * h)
            dx[torch.arange(len(k), device=k.device), k] += glp[:, 0]
            grads.append(dx)
    out = [torch.cat(lp), torch.cat(ent)]
    if case["top"]:
        out += [torch.cat(top_v), torch.cat(top_i)]
    if case["mode"] == "train":
        out.append(torch.cat(grads))
    return out
