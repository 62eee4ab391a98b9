"""Row operators of a training or matching step against their formulas in 64 bits: modules.rms_norm / rms_norm_q8, loss.token_logprobs,
train.clip_grad_norm_.

Tolerances: U is half a step of fp32, u half a step of the stored type.  A sum of n terms whose longest chain of additions is c terms long
(at most 64 in a thread's registers or n / 256 where a thread has more, and a tree of at most 24 levels above) is off by at most c U of
the sum of the terms' magnitudes; a product, quotient or root adds U, e^z adds (2 + 2 |z|) U, the store adds u of the value."""
import math

import pytest
import torch

from i2pnet_amd import loss, modules, ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else U


def chain(n):
    return max(64, n // 256) + 24


def tiny(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps if t != torch.float32 else 1.2e-38


def rnd(*shape, dtype=torch.float32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def within(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), what
    fine = torch.isfinite(want)
    over = ((got - want).abs() - tol.cpu().double().expand(want.shape))[fine]
    assert not over.numel() or float(over.max()) <= 0.0, (what, float((got - want).abs()[fine].max()), float(over.max()))


# ---- RMS norm --------------------------------------------------------------------------------------------------------------------
def norm64(x, r, w, eps, gy=None, gs=None):
    """-> s (stored), xh, y and, with gy, dx, dw and the magnitudes of their terms"""
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    a = s.double()
    rstd = 1 / (a.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = a * rstd
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    out = [s, xh * w]
    if gy is not None:
        g = gy.double()
        t = g * w
        m = (t * xh).mean(-1, keepdim=True)
        dx = rstd * (t - xh * m)
        mag = rstd * (t.abs() + xh.abs() * (t * xh).abs().mean(-1, keepdim=True))
        if gs is not None:
            dx, mag = dx + gs.double(), mag + gs.double().abs()
        out += [dx, mag, (g * xh).flatten(0, -2).sum(0), (g * xh).abs().flatten(0, -2).sum(0)]
    return out


NORM_SHAPES = [(1, 1), (1, 4096), (2, 7), (3, 64), (5, 65), (33, 257), (4, 512), (7, 1000), (2, 2049), (3, 5000), (2, 8191), (1, 16384), (2, 40001), (2, 70003),
               (1500, 64), (700, 130)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,d", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_forward_and_backward(dtype, rows, d, residual):
    x, r = rnd(rows, d, dtype=dtype, seed=1), rnd(rows, d, dtype=dtype, scale=2.0, seed=2) if residual else None
    wt = torch.float32 if (rows + d) % 2 else dtype
    w, gy, gs = (1 + 0.1 * rnd(d, seed=3)).to(wt), rnd(rows, d, dtype=dtype, seed=4), rnd(rows, d, dtype=dtype, seed=5) if residual else None
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w) + ((r,) if residual else ())]
    out = modules.rms_norm(leaves[0], leaves[1], residual=leaves[2] if residual else None, eps=1e-5)
    s, y64, dx64, mag, dw64, dwmag = norm64(x, r, w, 1e-5, gy, gs)
    u = half_step(dtype)
    y = out[0] if residual else out
    within(y, y64, (u + (chain(d) + 8) * U) * y64.abs() + tiny(dtype), "y")
    if residual:
        assert torch.equal(out[1].detach().cpu(), s)
    grads = torch.autograd.grad(out, leaves, [gy.to(DEV), gs.to(DEV)] if residual else [gy.to(DEV)])
    within(grads[0], dx64, u * dx64.abs() + (2 * chain(d) + 16) * U * mag + tiny(dtype), "dx")
    within(grads[1], dw64, half_step(wt) * dw64.abs() + (rows + chain(d) + 16) * U * dwmag + tiny(wt), "dw")
    assert grads[1].dtype == wt and grads[0].dtype == dtype
    if residual:
        assert torch.equal(grads[2], grads[0])


def test_rms_norm_gradient_against_differences():
    rows, d, h = 3, 12, 1e-3
    x, w, gy = rnd(rows, d, seed=1).double(), rnd(d, seed=2).double(), rnd(rows, d, seed=3).double()
    f = lambda a, b: (norm64(a, None, b, 1e-2)[1] * gy).sum()
    num = torch.zeros(rows, d, dtype=torch.float64)
    for i in range(rows):
        for j in range(d):
            e = torch.zeros_like(x); e[i, j] = h
            num[i, j] = (f(x + e, w) - f(x - e, w)) / (2 * h)
    a, b = x.float().to(DEV).requires_grad_(True), w.float().to(DEV)
    (dx,) = torch.autograd.grad(modules.rms_norm(a, b, eps=1e-2), a, gy.float().to(DEV))
    # central differences: h^2 / 6 times the third derivative, below 100 for these values; the inputs' rounding to fp32 adds 100 U at most
    assert float((dx.cpu().double() - num).abs().max()) < 1e-6 * 100 / 6 + 100 * U * 10


@pytest.mark.parametrize("need", ["x", "w", "r", "stream only", "y only", "none"])
def test_rms_norm_gradients_that_are_not_wanted(need):
    x, r, w = (rnd(*s, seed=i).to(DEV) for i, s in enumerate([(9, 40), (9, 40), (40,)]))
    gy, gs = rnd(9, 40, seed=5).to(DEV), rnd(9, 40, seed=6).to(DEV)
    full = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = modules.rms_norm(full[0], full[2], residual=full[1])
    want = torch.autograd.grad([y, s], full, [gy, gs], retain_graph=True)
    if need == "none":
        y, s = modules.rms_norm(x, w, residual=r)
        assert not y.requires_grad and not s.requires_grad
    elif need == "stream only":
        assert torch.equal(torch.autograd.grad(s, full[0], gs)[0], gs)
    elif need == "y only":
        a, b = torch.autograd.grad(y, full[:2], gy)
        assert torch.equal(a, b) and not torch.equal(a, want[0])
    else:
        k = "xrw".index(need)
        part = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, r, w))]
        y, s = modules.rms_norm(part[0], part[2], residual=part[1])
        outs, gs2 = ([y, s], [gy, gs]) if need != "w" else ([y], [gy])
        assert torch.equal(torch.autograd.grad(outs, part[k], gs2)[0], want[k])


def test_rms_norm_accumulates_into_leaves_used_twice():
    x = rnd(6, 33, seed=1).to(DEV).requires_grad_(True)
    w = rnd(33, seed=2).to(DEV).requires_grad_(True)
    y, s = modules.rms_norm(x, w, residual=x)                     # the same tensor on both sides
    (y.sum() + s.sum()).backward()
    _, _, dx, mag, dw, dwmag = norm64(x.detach().cpu(), x.detach().cpu(), w.detach().cpu(), 1e-6, torch.ones(6, 33), torch.ones(6, 33))
    within(x.grad, 2 * dx, 2 * (2 * chain(33) + 20) * U * mag, "dx")
    within(w.grad, dw, (6 + chain(33) + 16) * U * dwmag, "dw")


@pytest.mark.parametrize("layout", ["pitch", "column slice", "transposed", "expanded", "3d", "offset 1"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rms_norm_layouts(layout, dtype):
    rows, d = 6, 100
    base = rnd(rows, 3, 2 * d + 1, dtype=dtype, seed=7).to(DEV)
    x = {"pitch": base[:, 0, :d], "column slice": base[:, 1, 3:3 + d], "transposed": base[:, 2, :d].t().contiguous().t(),
         "expanded": base[:1, 0, :d].expand(rows, d), "3d": base[:, :, 1:1 + d], "offset 1": base.view(-1)[1:1 + rows * d].view(rows, d)}[layout]
    w = rnd(d, seed=8).to(DEV)
    x0 = x.detach()
    leaf = x0.clone().contiguous().requires_grad_(True)
    want = modules.rms_norm(leaf, w)
    gy = want.detach().sum(-1, keepdim=True).expand(want.shape)          # an expanded gradient
    got_leaf = x0.requires_grad_(True)
    got = modules.rms_norm(got_leaf, w)
    assert torch.equal(got, want) and got.is_contiguous()
    assert torch.equal(torch.autograd.grad(got, got_leaf, gy)[0], torch.autograd.grad(want, leaf, gy.contiguous())[0])
    y, s = modules.rms_norm(x0.detach(), w, residual=x0.detach())
    y2, s2 = modules.rms_norm(leaf.detach(), w, residual=leaf.detach())
    assert torch.equal(y, y2) and torch.equal(s, s2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,d,group", [(1, 1, 0), (3, 31, 32), (4, 64, 32), (2, 130, 64), (5, 1000, 128), (2, 1024, 512), (3, 5000, 256), (2, 70003, 128),
                                          (2, 4096, 0), (3, 40001, 0), (300, 96, 32), (7, 2056, 512)])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_q8(dtype, rows, d, group, residual):
    x, r, w = rnd(rows, d, dtype=dtype, seed=1), rnd(rows, d, dtype=dtype, seed=2) if residual else None, 1 + rnd(d, seed=3) * 0.1
    out = modules.rms_norm_q8(x.to(DEV), w.to(DEV), residual=r.to(DEV) if residual else None, eps=1e-5, group=group)
    s, y = norm64(x, r, w, 1e-5)
    q, scale = out[0].cpu(), out[1].cpu().double()
    g = group or d
    ng = -(-d // g)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, ng)
    pad = torch.nn.functional.pad(y.abs(), (0, ng * g - d)).view(rows, ng, g)
    want = pad.amax(-1) / 448
    rel = (chain(d) + 12) * U
    within(scale, want, rel * want, "scale")
    cols = scale.repeat_interleave(g, 1)[:, :d]
    # half a step of e4m3: 2^-4 of the value, 2^-10 below the smallest normal value 2^-6; the quotient before the rounding is off by rel
    err = (q.double() * cols - y).abs()
    assert float((err - (2.0 ** -4 * (1 + rel) * y.abs()).clamp_min(2.0 ** -10 * 1.01 * cols) - 2 * rel * y.abs()).max()) <= 0
    if residual:
        assert torch.equal(out[2].cpu(), s)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("group", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("d", [33, 64, 96, 100, 129, 200, 256, 257, 300, 500, 511, 513, 1000, 1030, 2100])
def test_rms_norm_q8_every_group_of_narrow_rows(dtype, group, d):
    x, w = rnd(37, d, dtype=dtype, seed=d), 1 + rnd(d, seed=3) * 0.1
    q, scale = modules.rms_norm_q8(x.to(DEV), w.to(DEV), eps=1e-5, group=group)
    _, y = norm64(x, None, w, 1e-5)
    ng = -(-d // group)
    want = torch.nn.functional.pad(y.abs(), (0, ng * group - d)).view(37, ng, group).amax(-1) / 448
    rel = (chain(d) + 12) * U
    within(scale, want, rel * want, "scale")
    cols = scale.cpu().double().repeat_interleave(group, 1)[:, :d]
    err = (q.cpu().double() * cols - y).abs()
    assert float((err - (2.0 ** -4 * (1 + rel) * y.abs()).clamp_min(2.0 ** -10 * 1.01 * cols) - 2 * rel * y.abs()).max()) <= 0


def test_rms_norm_q8_special_rows():
    x = rnd(6, 64, seed=1)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 40] = float("inf")
    x[4, :32] = 0
    q, scale = modules.rms_norm_q8(x.to(DEV), None, group=32)
    q, scale = q.float().cpu(), scale.cpu()
    assert torch.equal(scale[1], torch.ones(2)) and not q[1].any()
    assert scale[4, 0] == 1 and not q[4, :32].any() and q[4, 32:].abs().max() == 448
    assert torch.isinf(scale[2]).all() and torch.isnan(q[2] * scale[2].repeat_interleave(32)).all()
    assert torch.isinf(scale[3, 1]) and torch.isnan(q[3, 40])
    assert torch.isfinite(scale[[0, 1, 4, 5]]).all() and torch.isfinite(q[[0, 1, 4, 5]]).all()


def test_rms_norm_extremes():
    x = torch.zeros(4, 50)
    x[1] = 1e-20; x[2] = 1e10; x[3, 0] = float("nan")
    y = modules.rms_norm(x.to(DEV), None, eps=1e-6).cpu()
    assert not y[0].any() and torch.isnan(y[3]).all()
    assert float((y[2] - 1).abs().max()) < 100 * U and float((y[1] - 1e-17).abs().max()) < 1e-17 * 100 * U
    assert modules.rms_norm(torch.zeros(0, 8, device=DEV), torch.ones(8, device=DEV)).shape == (0, 8)
    leaf, w = torch.zeros(0, 8, device=DEV, requires_grad=True), torch.ones(8, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(modules.rms_norm(leaf, w).sum(), [leaf, w])
    assert gx.shape == (0, 8) and not gw.any()
    assert modules.rms_norm_q8(torch.zeros(0, 8, device=DEV), None)[1].shape == (0, 1)
    half = modules.rms_norm(torch.full((1, 8), 60000.0, dtype=torch.float16, device=DEV), None)       # squares past fp16
    assert torch.equal(half.cpu(), torch.ones(1, 8, dtype=torch.float16))


def test_more_rows_than_one_launch_takes():
    rows = (1 << 25) + 77                       # 16 rows a block, 2^21 blocks a launch
    x = torch.full((rows, 1), 3.0, dtype=torch.bfloat16, device=DEV)
    x[-1] = -3.0
    x[1 << 25] = 0.0
    y, s = modules.rms_norm(x, None, residual=x)
    assert s[-1] == -6 and y[-1] == -1 and y[1 << 25] == 0 and y[(1 << 25) - 1] == 1 and int(y.eq(1).sum()) == rows - 2
    q, scale = modules.rms_norm_q8(x, None)
    assert q[-1].float() == -448 and scale[-1] > 0 and scale[1 << 25] == 1
    ids = torch.zeros(rows, dtype=torch.long, device=DEV)
    ids[-1] = 5
    o = loss.token_logprobs(x, ids, top=1)      # 2^21 rows a launch
    assert torch.isnan(o.logp[-1]) and not o.logp[:-1].any() and not o.entropy.any() and not o.top_ids.any() and not o.top_logp.any()


# ---- log probabilities -----------------------------------------------------------------------------------------------------------
def logp64(x, ids, top, gl=None, gh=None):
    a = x.double()
    m = a.amax(-1, keepdim=True)
    z = a - torch.where(m.isfinite(), m, torch.zeros_like(m))             # (3e38 + 8 is 3e38 in 64 bits too)
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    p = lp.exp()
    plogp = torch.special.xlogy(p, p)
    H = -plogp.sum(-1, keepdim=True)
    keys, order = torch.sort(a, dim=-1, descending=True, stable=True)
    out = [lp.gather(1, ids[:, None])[:, 0], H[:, 0], lp.gather(1, order[:, :top]), order[:, :top]]
    if gl is not None:
        gl, gh = gl.double()[:, None], gh.double()[:, None]
        dx = -p * gl - gh * (plogp + p * H)
        dx.scatter_add_(1, ids[:, None], gl)
        mag = p * (gl.abs() + gh.abs() * (lp.clamp_min(-200).abs() + H))
        out += [dx, mag]
    return out


def logp_tol(v, lp, span):
    return (chain(v) + 64 + 2 * span) * U + 3 * U * lp.abs()


LOGP_SHAPES = [(1, 1), (3, 2), (1, 131072), (5, 33), (70, 100), (9, 468), (4, 1000), (2, 2047), (3, 2049), (6, 4100), (2, 8192), (3, 20001), (2, 32000),
               (2, 33333), (1, 70001), (2, 200003)]


def mask_some(x, kind, ids):
    if kind == "none":
        return x
    x = x.clone()
    drop = torch.rand(x.shape, generator=torch.Generator().manual_seed(9)) < 0.5
    drop.scatter_(1, ids[:, None], False)
    x[drop] = -math.inf if kind == "inf" else torch.finfo(x.dtype).min
    return x


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,v", LOGP_SHAPES)
@pytest.mark.parametrize("mask", ["none", "inf", "lowest"])
def test_token_logprobs(dtype, rows, v, mask):
    g = torch.Generator().manual_seed(v)
    ids = torch.randint(0, v, (rows,), generator=g)
    x = mask_some(rnd(rows, v, dtype=dtype, scale=3.0, seed=v + 1), mask, ids)
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    top = min(v, [1, 5, 8, 20, 32][(rows + v) % 5])
    leaf = x.to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV), top=top)
    lp, H, tl, ti, dx, mag = logp64(x, ids, top, gl, gh)
    within(o.logp, lp, logp_tol(v, lp, 16), "logp")
    within(o.entropy, H, (chain(v) + 64) * U * 33 * torch.ones_like(H), "entropy")
    assert torch.equal(o.top_ids.cpu(), ti)
    within(o.top_logp, tl, logp_tol(v, tl.clamp_min(-1e37), 16), "top_logp")
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl.to(DEV), gh.to(DEV)])
    tol = half_step(dtype) * dx.abs() + (8 * chain(v) + 2000) * U * mag + (1 + gl.abs() + gh.abs())[:, None] * 1e-36 + tiny(dtype)
    within(d, dx, tol, "dlogits")


@pytest.mark.parametrize("top", [0, 1, 2, 31, 32])
@pytest.mark.parametrize("v", [32, 64, 100, 300, 513, 3000, 17000, 40000, 150000])
@pytest.mark.parametrize("kind", ["ties", "equal", "sorted", "reversed", "clump", "inf", "zeros of both signs"])
def test_token_logprobs_alternatives(v, top, kind):
    """the k best of rows where many scores are equal or the best ones sit together"""
    rows = 3
    x = rnd(rows, v, seed=v)
    if kind == "ties":
        x = (x * 2).round()
    elif kind == "equal":
        x = torch.full((rows, v), 1.5)
    elif kind == "sorted":
        x = torch.arange(v).float().expand(rows, v) / v
    elif kind == "reversed":
        x = -torch.arange(v).float().expand(rows, v) / v
    elif kind == "clump":
        x[:, v // 2:v // 2 + 40] += 50
    elif kind == "inf":
        x[:, 5:] = -math.inf
    else:
        x = torch.where(x > 0, 0.0, -0.0)
    for dt in (torch.float32, torch.bfloat16):
        xs = x.to(dt).contiguous()
        o = loss.token_logprobs(xs.to(DEV), torch.zeros(rows, dtype=torch.long, device=DEV), top=top)
        _, _, tl, ti = logp64(xs, torch.zeros(rows, dtype=torch.long), top)
        assert torch.equal(o.top_ids.cpu(), ti)
        within(o.top_logp, tl, logp_tol(v, tl.clamp_min(-1e37), 16), "top_logp")


@pytest.mark.parametrize("v", [40, 700, 9000, 100001])
def test_token_logprobs_special_rows(v):
    x = rnd(9, v, seed=3)
    x[1] = -math.inf                                        # nothing left
    x[2, 7] = math.nan
    x[3, v - 1] = math.inf
    x[4] = math.nan                                         # padding: not read
    x[5] = torch.finfo(torch.float32).min                   # all at the lowest value: uniform
    x[6, :] = -math.inf; x[6, 11] = 3.0                     # one candidate
    ids = torch.tensor([0, 3, 7, 2, -100, 1, 11, v, -1])
    leaf = x.to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV), top=3)
    lp, H, tl, ti = (t.cpu() for t in o)
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [torch.ones(9, device=DEV), torch.ones(9, device=DEV)])
    d = d.cpu()
    assert lp[1] == -math.inf and H[1] == 0 and not d[1].any() and (tl[1] == -math.inf).all() and ti[1].tolist() == [0, 1, 2]
    assert torch.isnan(lp[[2, 3]]).all() and torch.isnan(H[[2, 3]]).all() and torch.isnan(d[[2, 3]]).all() and torch.isnan(tl[[2, 3]]).all()
    assert ti[2, 0] == 7 and ti[3, 0] == v - 1
    assert lp[4] == 0 and H[4] == 0 and not d[4].any() and (ti[4] == -1).all() and (tl[4] == -math.inf).all()
    assert abs(float(lp[5]) + math.log(v)) < (chain(v) + 64) * U * 16 and abs(float(H[5]) - math.log(v)) < (chain(v) + 64) * U * 33
    assert lp[6] == 0 and H[6] == 0 and not d[6].any() and ti[6].tolist() == [11, 0, 1] and tl[6].tolist() == [0, -math.inf, -math.inf]
    assert torch.isnan(lp[[7, 8]]).all() and torch.isnan(d[[7, 8]]).all() and torch.isfinite(H[[7, 8]]).all()
    ref = logp64(x[:1], ids[:1], 3)
    assert torch.equal(ti[:1], ref[3])


def test_token_logprobs_far_from_zero():
    """scores of a few thousand: the log of the sum must not lose its digits to the maximum"""
    x = rnd(4, 5000, seed=1) + 4096.0
    ids = torch.tensor([0, 1, 2, 3])
    gl, gh = torch.ones(4), torch.zeros(4)
    lp, _, _, _, dx, mag = logp64(x, ids, 0, gl, gh)
    leaf = x.to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV))
    within(o.logp, lp, logp_tol(5000, lp, 16), "logp")
    within(torch.autograd.grad(o.logp.sum(), leaf)[0], dx, U * dx.abs() + (8 * chain(5000) + 2000) * U * mag, "dlogits")


def test_token_logprobs_gradient_against_differences():
    x, ids = rnd(2, 9, seed=4).double(), torch.tensor([3, 8])
    gl, gh = torch.tensor([0.7, -1.1]), torch.tensor([0.4, 0.9])

    def f(a):
        lp, H, _, _ = logp64(a, ids, 0)
        return (lp * gl.double() + H * gh.double()).sum()
    num = torch.zeros_like(x)
    for i in range(2):
        for j in range(9):
            e = torch.zeros_like(x); e[i, j] = 1e-4
            num[i, j] = (f(x + e) - f(x - e)) / 2e-4
    leaf = x.float().to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV))
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl.to(DEV), gh.to(DEV)])
    # 1e-8 / 6 times a third derivative below 20; inputs and arithmetic in fp32: 400 U at most
    assert float((d.cpu().double() - num).abs().max()) < 1e-7 + 400 * U


@pytest.mark.parametrize("which", ["logp", "entropy"])
def test_token_logprobs_one_gradient(which):
    x, ids = rnd(5, 77, seed=4), torch.tensor([3, 8, 0, 76, 9])
    one, zero = torch.ones(5), torch.zeros(5)
    leaf = x.to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV), top=2)
    assert not o.top_logp.requires_grad and not o.top_ids.requires_grad
    (d,) = torch.autograd.grad(getattr(o, which).sum(), leaf)
    dx, mag = logp64(x, ids, 0, *((one, zero) if which == "logp" else (zero, one)))[4:]
    within(d, dx, U * dx.abs() + (8 * chain(77) + 2000) * U * mag + 1e-36, "dlogits")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_token_logprobs_layouts(dtype):
    """a padded vocabulary, a transposed one, leading axes, ids with strides"""
    base = rnd(3, 4, 1030, dtype=dtype, seed=2).to(DEV)
    ids = torch.randint(0, 1001, (3, 8), generator=torch.Generator().manual_seed(1)).to(DEV)[:, ::2]
    for x in (base[:, :, :1001], base[:, :, 5:1006], base[:, :, :1001].transpose(0, 1).contiguous().transpose(0, 1), base[:, :, :1001].expand(3, 4, 1001)):
        a, b = x.detach().requires_grad_(True), x.detach().contiguous().clone().requires_grad_(True)
        oa, ob = loss.token_logprobs(a, ids, top=4), loss.token_logprobs(b, ids.contiguous(), top=4)
        for p, q in zip(oa, ob):
            assert p.shape == q.shape and torch.equal(p, q)
        ga, gb = (torch.autograd.grad(o.logp.sum() + o.entropy.sum(), t)[0] for o, t in ((oa, a), (ob, b)))
        assert torch.equal(ga, gb) and ga.shape == x.shape
    assert loss.token_logprobs(base[:0], ids[:0], top=2).top_ids.shape == (0, 4, 2)
    one = loss.token_logprobs(base[0, 0], ids[0, 0], top=3)                        # a single row without leading axes
    assert one.logp.shape == () and torch.equal(one.top_ids, loss.token_logprobs(base[:1, 0], ids[:1, 0], top=3).top_ids[0])


def test_token_logprobs_beyond_32_bit_offsets():
    """rows whose elements lie past 2^32 in the buffer"""
    v, rows = 70000, 4
    pitch = (1 << 31) // 2
    x = torch.zeros(pitch * (rows + 1), dtype=torch.bfloat16, device=DEV)
    rowsv = x.as_strided((rows, v), (pitch + 7, 1))
    vals = rnd(rows, v, dtype=torch.bfloat16, seed=5)
    rowsv.copy_(vals.to(DEV))
    ids = torch.arange(rows) * 1000
    got = loss.token_logprobs(rowsv, ids.to(DEV), top=3)
    want = loss.token_logprobs(vals.to(DEV), ids.to(DEV), top=3)
    for p, q in zip(got, want):
        assert torch.equal(p, q)


# ---- gradient norm and clipping --------------------------------------------------------------------------------------------------
def clip64(gs, limit, kind):
    flat = torch.cat([g.double().reshape(-1) for g in gs]) if gs else torch.zeros(0, dtype=torch.float64)
    n = flat.square().sum().sqrt() if kind == 2 else flat.abs().max() if flat.numel() else torch.zeros((), dtype=torch.float64)
    return n, torch.clamp(limit / (n + 1e-6), max=1.0)


def grads_of(sizes, seed=0):
    return [rnd(k, dtype=TYPES[(i + seed) % 3], seed=i + seed) for i, k in enumerate(sizes)]


SIZES = [[1], [3, 1, 5], [16384], [16385, 16383, 2], [0, 7, 0], [100003, 64, 1, 33000], [17] * 400, [256 * k + 1 for k in range(200)]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)} tensors, {sum(s)}")
@pytest.mark.parametrize("kind", [2, math.inf])
@pytest.mark.parametrize("limit", [0.5, 1e9])
@pytest.mark.parametrize("into", [False, True])
def test_clip_grad_norm(sizes, kind, limit, into):
    gs = grads_of(sizes)
    dev = [g.to(DEV) for g in gs]
    n, c = clip64(gs, limit, kind)
    out = torch.full((sum(sizes),), 7.0, device=DEV) if into else None
    total = train.clip_grad_norm_(dev, limit, norm_type=kind, out=out)
    assert total.shape == () and total.dtype == torch.float32
    # the sum is in 64 bits; the total is rounded once, the factor and the product three times more
    within(total, n, 1.001 * U * n + 1e-45, "norm")
    assert torch.equal(train.grad_norm([g.to(DEV) for g in gs], norm_type=kind), total)
    if into:
        want = torch.cat([g.double().reshape(-1) for g in gs]) * c
        within(out, want, 5 * U * want.abs() + 1e-44, "out")
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, gs))
    else:
        for a, b in zip(dev, gs):
            want = b.double() * c
            within(a, want, (half_step(b.dtype) + 5 * U) * want.abs() + tiny(b.dtype), "gradient")
            assert limit < 1 or torch.equal(a.cpu(), b)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", [2, math.inf])
def test_clip_grad_norm_not_finite(bad, kind):
    gs = [torch.ones(50, device=DEV), torch.ones(20000, device=DEV), torch.ones(3, device=DEV)]
    gs[1][17000] = bad
    ref = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
    for p, g in zip(ref, gs):
        p.grad = g.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        train.clip_grad_norm_(gs, 1.0, norm_type=kind, error_if_nonfinite=True)
    assert gs[0].eq(1).all()
    got = train.clip_grad_norm_(gs, 1.0, norm_type=kind)
    want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm_type=kind)
    assert torch.equal(got, want) or (got.isnan() and want.isnan())
    for p, g in zip(ref, gs):
        assert torch.equal(torch.nan_to_num(p.grad, nan=5.0), torch.nan_to_num(g, nan=5.0))


def test_clip_grad_norm_large_values_and_parameters():
    """squares past fp32; parameters whose .grad is meant, some without one, one frozen, channels_last; extra dims"""
    g = torch.full((1000,), 1e30, device=DEV)
    n = train.clip_grad_norm_([g], 1.0)
    assert abs(float(n) / (1e30 * math.sqrt(1000.0)) - 1) < 4 * U and abs(float(g.double().norm()) - 1) < 8 * U
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 5, 3), torch.nn.Conv2d(5, 2, 1)).to(DEV).to(memory_format=torch.channels_last)
    net(torch.randn(2, 3, 8, 8, device=DEV).to(memory_format=torch.channels_last)).square().sum().backward()
    net[1].bias.grad = None
    net[1].bias.requires_grad_(False)
    kept = net[1].bias.detach().clone()
    net[0].weight.grad = net[0].weight.grad.to(memory_format=torch.channels_last)
    want = {k: p.grad.clone() for k, p in net.named_parameters() if p.grad is not None}
    n64 = torch.sqrt(sum(v.double().square().sum() for v in want.values()))
    version = net[0].weight.grad._version
    n = train.clip_grad_norm_(net.parameters(), 0.25)
    assert abs(float(n) / float(n64) - 1) < 2 * U and net[0].weight.grad._version > version
    for k, p in net.named_parameters():
        if k in want:
            within(p.grad, want[k].double() * (0.25 / (n64 + 1e-6)), 8 * U * want[k].abs(), k)
    assert torch.equal(net[1].bias, kept)
    assert float(train.clip_grad_norm_([torch.zeros(0, device=DEV)], 1.0)) == 0.0
    assert float(train.clip_grad_norm_([net[1].bias], 1.0)) == 0.0 and float(train.grad_norm([])) == 0.0
    single = torch.full((4,), 3.0, device=DEV)
    assert float(train.clip_grad_norm_(single, 7.0)) == 6.0 and single.eq(3).all()


def test_clip_grad_norm_views_at_odd_addresses():
    flat = rnd(5000, dtype=torch.bfloat16, seed=1).to(DEV)
    keep = flat.clone()
    views = [flat[1:1002], flat[1003:1004], flat[1005:3000], flat[3001:5000]]
    n, c = clip64([v.cpu() for v in views], 0.1, 2)
    train.clip_grad_norm_(views, 0.1)
    for lo, hi in ((1, 1002), (1003, 1004), (1005, 3000), (3001, 5000)):
        want = keep[lo:hi].cpu().double() * c
        within(flat[lo:hi], want, (2.0 ** -8 + 5 * U) * want.abs() + tiny(torch.bfloat16), "view")
    for i in (0, 1002, 1004, 3000):
        assert flat[i] == keep[i]                              # what lies between is nobody's


def test_clip_grad_norm_a_long_tensor():
    """more elements than one entry of the kernels' table covers"""
    n = (1 << 30) + 12345
    g = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    total = train.clip_grad_norm_([g, torch.ones(3, device=DEV)], 16.0)
    assert abs(float(total) / math.sqrt(n + 3) - 1) < 2 * U
    c = torch.tensor(16.0 / math.sqrt(n + 3)).to(torch.bfloat16)
    assert g[:5].eq(c.to(DEV)).all() and g[(1 << 30) - 5:(1 << 30) + 5].eq(c.to(DEV)).all() and g[-1] == c.to(DEV)


# ---- together, streams, graphs ---------------------------------------------------------------------------------------------------
def matching_step(params, feats, pixels, ids, limit):
    """features of points and pixels -> norm -> scores -> -log p + entropy term -> gradients, clipped"""
    f, w, g = params
    y, s = modules.rms_norm(feats, w, residual=f)
    logits = torch.nn.functional.linear(torch.nn.functional.linear(y, g), pixels)
    o = loss.token_logprobs(logits, ids, top=3)
    grads = list(torch.autograd.grad(-o.logp.mean() + 0.1 * o.entropy.mean() + 1e-3 * s.square().mean(), params))
    total = train.clip_grad_norm_(grads, limit)
    return o, grads, total


def matching_inputs(seed=0):
    f, w, g = rnd(90, 64, seed=seed), 1 + 0.1 * rnd(64, seed=seed + 1), rnd(48, 64, scale=0.2, seed=seed + 2)
    feats, pixels = rnd(90, 64, seed=seed + 3), rnd(117, 48, seed=seed + 4)
    return [f, w, g], feats, pixels, torch.randint(0, 117, (90,), generator=torch.Generator().manual_seed(seed))


def test_a_matching_step():
    params, feats, pixels, ids = matching_inputs()
    p64 = [p.double().requires_grad_(True) for p in params]
    s = feats.double() + p64[0]
    y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * p64[1]
    lp = torch.log_softmax(y @ p64[2].t() @ pixels.double().t(), -1)
    H = -(lp.exp() * lp).sum(-1)
    want = torch.autograd.grad(-lp.gather(1, ids[:, None]).mean() + 0.1 * H.mean() + 1e-3 * s.square().mean(), p64)
    n, c = clip64(want, 0.05, 2)
    dev = [p.to(DEV).requires_grad_(True) for p in params]
    o, grads, total = matching_step(dev, feats.to(DEV), pixels.to(DEV), ids.to(DEV), 0.05)
    assert torch.equal(o.top_ids.cpu(), lp.detach().topk(3).indices)
    # scores are sums of 48 products of sums of 64, magnitude below 200: off by at most (64 + 48) U 200, and that enters p as a factor
    rel = 3 * (64 + 48) * 200 * U
    assert abs(float(total) / float(n) - 1) < rel
    for a, b in zip(grads, want):
        assert float((a.cpu().double() - b * c).norm() / (b * c).norm()) < rel


def test_two_runs_are_bit_identical():
    for dtype in TYPES:
        x, r = rnd(3000, 1001, dtype=dtype, seed=1).to(DEV), rnd(3000, 1001, dtype=dtype, seed=2).to(DEV)
        w, ids = rnd(1001, seed=3).to(DEV), torch.randint(0, 1001, (3000,), generator=torch.Generator().manual_seed(1)).to(DEV)

        def once():
            a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            y, s = modules.rms_norm(a, b, residual=r)
            o = loss.token_logprobs(y, ids, top=5)
            ga, gb = torch.autograd.grad(o.logp.sum() + o.entropy.sum() + s.float().sum(), [a, b])
            n = train.clip_grad_norm_([ga, gb], 0.1)
            return [y, s, *o, ga, gb, n]
        for p, q in zip(once(), once()):
            assert torch.equal(p, q)


def test_side_stream():
    params, feats, pixels, ids = matching_inputs(5)
    dev = [p.to(DEV).requires_grad_(True) for p in params]
    a = [t.to(DEV) for t in (feats, pixels, ids)]
    want = matching_step(dev, *a, 0.05)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = matching_step(dev, *a, 0.05)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got[2], want[2]) and all(torch.equal(p, q) for p, q in zip(list(got[0]) + got[1], list(want[0]) + want[1]))


def test_captured_calls_replay_on_new_inputs():
    """two graphs of the same calls, replayed in turn with eager work between, each replay checked against the eager result"""
    x, r = torch.zeros(300, 520, device=DEV, dtype=torch.bfloat16), torch.zeros(300, 520, device=DEV, dtype=torch.bfloat16)
    w, ids = torch.ones(520, device=DEV), torch.zeros(300, dtype=torch.long, device=DEV)
    big, one = torch.zeros(3, 90001, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    gy, gl, gh = torch.zeros(300, 520, device=DEV, dtype=torch.bfloat16), torch.zeros(300, device=DEV), torch.zeros(300, device=DEV)
    be = ops.hip_backend()

    def calls():
        y, s, rstd = be.rms_norm_forward(x, w, r, 1e-6)
        dx, dw = be.rms_norm_backward(s, w, rstd, gy, gy, True)
        q, scale, _ = be.rms_norm_q8(x, w, r, 1e-6, 128)
        o = be.token_logprobs_forward(y, ids, 5, -100)
        dl = be.token_logprobs_backward(o[4], o[5], -100, o[6], o[1], gl, gh)
        b = be.token_logprobs_forward(big, one, 8, -100)
        flat = torch.empty(dx.numel() + dw.numel(), device=DEV)
        n = be.clip_grad_norm([dx, dw], 0, 0.5, flat)
        m = be.clip_grad_norm([dx, dw], 0, 0.5)
        return [y, s, dx, dw, q.view(torch.uint8), scale, *o[:4], dl, *b[:4], flat, n, m]

    def fill(seed):
        for i, t in enumerate((x, r, w, big, gy, gl, gh)):
            t.copy_(rnd(*t.shape, seed=seed * 10 + i))
        ids.copy_(torch.randint(0, 520, (300,), generator=torch.Generator().manual_seed(seed)))
        one.copy_(torch.randint(0, 90001, (3,), generator=torch.Generator().manual_seed(seed)))
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = calls()
        graphs.append((g, outs))
    for k in range(4):
        fill(k + 1)
        want = [t.clone() for t in calls()]
        for g, outs in (graphs if k % 2 else graphs[::-1]):
            g.replay()
            calls()                                            # eager work behind the replay must not disturb its results
            torch.cuda.synchronize()
            for i, (p, q) in enumerate(zip(outs, want)):
                assert torch.equal(p, q), (k, i)


def test_the_rows_behind_a_batch_stay_as_they_are():
    """outputs have the given rows only: a guard region behind the flat output and padding rows of the inputs stay untouched"""
    buf = torch.full((1000,), 9.0, device=DEV)
    g = [torch.ones(300, device=DEV, dtype=torch.bfloat16), torch.ones(77, device=DEV)]
    train.clip_grad_norm_(g, 1.0, out=buf[100:477])
    assert buf[:100].eq(9).all() and buf[477:].eq(9).all() and not buf[100:477].eq(9).any()


@pytest.mark.parametrize("far", [1e5, -1e5, 3e38, -3e38, 1e30])
def test_token_logprobs_maximum_far_from_zero(far):
    """a maximum beyond the range where its logarithm's rounding is carried along, up to the type's largest values"""
    v = 3000
    x = far + (rnd(4, v, seed=2) * (4.0 if abs(far) < 1e6 else 1e-3 * abs(far)))
    x[1] = far                                              # uniform
    x[2, 5:] = torch.finfo(torch.float32).min
    x[3, 5:] = -math.inf
    ids = torch.tensor([0, 1, 2, 3])
    gl, gh = torch.ones(4), 0.5 * torch.ones(4)
    lp, H, tl, ti, dx, mag = logp64(x, ids, 4, gl, gh)
    leaf = x.to(DEV).requires_grad_(True)
    o = loss.token_logprobs(leaf, ids.to(DEV), top=4)
    # z of the given candidate is one subtraction off: U of the larger operand, at most 2 U |far| where that is below 1e6
    near = 2 * U * abs(far) if abs(far) < 1e6 else 0.0
    lp, tl = (t.masked_fill(t < -3.4e38, -math.inf) for t in (lp, tl))
    big = lambda t: torch.where(t < -1e30, t.abs() * 4 * U, logp_tol(v, t.clamp_min(-1e37), 16) + near)
    within(o.logp, lp, big(lp.clamp_min(-3.5e38)), "logp")
    within(o.top_logp, tl, big(tl.clamp_min(-3.5e38)), "top_logp")
    assert torch.equal(o.top_ids.cpu(), ti)
    within(o.entropy, H, (chain(v) + 64) * U * 33 * torch.ones_like(H) + 32 * near, "entropy")
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl.to(DEV), gh.to(DEV)])
    within(d, dx, U * dx.abs() + (8 * chain(v) + 2000) * U * mag + 64 * near * mag + 1e-36, "dlogits")


def test_double_backward_is_refused():
    for f in (lambda a: modules.rms_norm(a, None), lambda a: loss.token_logprobs(a, torch.zeros(3, dtype=torch.long, device=DEV)).logp):
        a = rnd(3, 9, seed=1).to(DEV).requires_grad_(True)
        (g,) = torch.autograd.grad(f(a).sum(), a, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.square().sum().backward()


def test_what_a_backward_pass_needs_may_not_be_changed():
    a, w = rnd(3, 9, seed=1).to(DEV).requires_grad_(True), rnd(9, seed=2).to(DEV).requires_grad_(True)
    y, s = modules.rms_norm(a, w, residual=a)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    b = torch.zeros(9, device=DEV, requires_grad=True)
    y = (b * b).sum()
    train.clip_grad_norm_([b.detach()], 1.0)                # clipping counts as a change too
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_captured_training_pass():
    """forward and backward through autograd in a graph, replayed on new inputs with eager passes between"""
    x, w = torch.zeros(64, 130, device=DEV, requires_grad=True), torch.ones(130, device=DEV, requires_grad=True)
    ids = torch.zeros(64, dtype=torch.long, device=DEV)

    def one():
        y, s = modules.rms_norm(x, w, residual=x)
        o = loss.token_logprobs(y, ids, top=2)
        g = list(torch.autograd.grad(-o.logp.mean() + 0.1 * o.entropy.mean() + s.square().mean(), [x, w]))
        return g + [train.clip_grad_norm_(g, 1e-3), o.logp.detach(), o.top_ids]

    def fill(seed):
        with torch.no_grad():
            x.copy_(rnd(64, 130, seed=seed))
        ids.copy_(torch.randint(0, 130, (64,), generator=torch.Generator().manual_seed(seed)))
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = one()
    for k in range(3):
        fill(k + 1)
        want = [t.clone() for t in one()]
        graph.replay()
        one()
        torch.cuda.synchronize()
        for p, q in zip(outs, want):
            assert torch.equal(p, q)


def test_gradients_that_carry_a_graph_can_be_clipped():
    a = rnd(40, seed=1).to(DEV).requires_grad_(True)
    (g,) = torch.autograd.grad((a ** 3).sum(), a, create_graph=True)
    b = torch.nn.Parameter(torch.zeros(40, device=DEV))
    b.grad = g
    want = g.detach().clone()
    n = train.clip_grad_norm_([b], 1.0, error_if_nonfinite=True)
    assert abs(float(n) / float(want.double().norm()) - 1) < 2 * U
    within(b.grad, want.double() / (want.double().norm() + 1e-6), 8 * U * want.abs(), "clipped")


def test_reads_and_writes_between_guards():
    """every operator on views in the middle of larger buffers: what lies around them keeps its bits, at each width's last vector"""
    for dtype in TYPES:
        for d in (1, 5, 8, 63, 65, 519, 2049, 4103):
            pad = 24
            buf = torch.full((3, d + 2 * pad), 1.0, dtype=dtype, device=DEV)
            x = buf[:, pad:pad + d]
            x.copy_(rnd(3, d, dtype=dtype, seed=d))
            keep = buf.clone()
            ids = torch.zeros(3, dtype=torch.long, device=DEV)
            leaf = x.detach().requires_grad_(True)
            y, s = modules.rms_norm(leaf, None, residual=leaf)
            o = loss.token_logprobs(leaf, ids, top=min(d, 4))
            torch.autograd.grad(y.float().sum() + s.float().sum() + o.logp.sum(), leaf)
            modules.rms_norm_q8(x, None, group=32)
            assert torch.equal(buf, keep)
            flat = buf.view(-1)
            views = [flat[k * (d + 2 * pad) + pad:k * (d + 2 * pad) + pad + d] for k in range(3)]
            train.clip_grad_norm_(views, 1e-2)
            mask = torch.ones_like(buf, dtype=torch.bool)
            mask[:, pad:pad + d] = False
            assert torch.equal(buf[mask], keep[mask])


@pytest.mark.parametrize("rows,v,dtype", [(2100, 16384, torch.bfloat16), (1100, 16388, torch.float32), (1100, 16389, torch.float32)])
def test_token_logprobs_gradient_past_the_caches(rows, v, dtype):
    """gradients of 64 MB and more, which are written past the caches where rows start on 16 bytes"""
    x = torch.randn(rows, v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    ids = torch.randint(0, v, (rows,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    ids[5] = -100
    ids[rows - 1] = v
    leaf = x.clone().requires_grad_(True)
    o = loss.token_logprobs(leaf, ids)
    (d,) = torch.autograd.grad(o.logp.sum() + o.entropy.sum(), leaf)
    assert not d[5].any() and torch.isnan(d[rows - 1]).all()
    some = torch.tensor([0, 1, 2, 3, 4, 6, rows // 2, rows - 4, rows - 3, rows - 2])
    one = torch.ones(len(some))
    dx, mag = logp64(x[some.to(DEV)].cpu(), ids.cpu()[some], 0, one, one)[4:]
    within(d[some.to(DEV)], dx, half_step(dtype) * dx.abs() + (8 * chain(v) + 2000) * U * mag + 1e-36, "dlogits")
    # every row's gradient sums to 0 but for those errors; |dx| adds up to 2.2 over such a row and the terms' magnitudes to 20.5
    assert float(d[6:rows - 1].double().sum(-1).abs().max()) < 40 * (half_step(dtype) + (8 * chain(v) + 2000) * U)


def test_negated_views():
    """views whose sign is a flag that torch keeps beside them (the imaginary part of a conjugate) stand for the negated memory"""
    for d in (1, 40):
        z = torch.complex(rnd(6, d, seed=1), rnd(6, d, seed=2)).to(DEV)
        flat = rnd(6, d, seed=3).to(DEV)
        for a in (z.conj().imag, torch._neg_view(flat)):
            assert a.is_neg()
            b = a.clone(memory_format=torch.contiguous_format).resolve_neg().clone()
            b.copy_(-(z.imag if a.stride() != flat.stride() else flat))
            w, gy, one = torch._neg_view(rnd(d, seed=4).to(DEV)), torch._neg_view(rnd(6, d, seed=5).to(DEV)), torch._neg_view(rnd(6, seed=6).to(DEV))
            ids = torch._neg_view(-torch.tensor([0] * 5 + [d - 1], device=DEV))
            sides = []
            for x, real in ((a, lambda t: t), (b, lambda t: 0 + t)):
                x, p = x.detach().requires_grad_(True), real(w).detach().requires_grad_(True)
                y, s = modules.rms_norm(x, p, residual=x)
                alone = modules.rms_norm(x, p)
                o = loss.token_logprobs(x, real(ids), top=1)
                q = modules.rms_norm_q8(x.detach(), p.detach(), residual=x.detach(), group=32)
                gx, gp = torch.autograd.grad([y, s], [x, p], [real(gy), real(gy)])
                (gl,) = torch.autograd.grad([o.logp, o.entropy], [x], [real(one), real(one)])
                out = torch.empty(6 * d, device=DEV)
                n = train.clip_grad_norm_([real(gy)], 0.5, out=out)
                sides.append([y, s, alone, gx, gp, gl, out, n, *o, q[0].view(torch.uint8), *q[1:]])
            for i, (p, q) in enumerate(zip(*sides)):
                assert torch.equal(p, q), (d, i)
    base = torch.full((4,), -3.0, device=DEV)
    assert float(train.clip_grad_norm_([torch._neg_view(base)], 3.0)) == 6.0 and float((base + 1.5).abs().max()) < 1e-6
    with pytest.raises(RuntimeError, match="out must"):
        train.clip_grad_norm_([base], 1.0, out=torch._neg_view(torch.empty(4, device=DEV)))


@pytest.mark.parametrize("count", [1800, 2048])
def test_the_norm_does_not_depend_on_the_call(count):
    """squares whose sum lies a few last places of fp64 above a tie of fp32: the order of the additions shows in the rounded norm.  2^24, 4096,
    4096 and 1 have (2^24 + 1)^2 as their sum; 0.15^2 = 0.0225 is lost beside it alone (half a last place: 2^-5) and kept in pairs"""
    vals = torch.zeros(count)
    vals[0], vals[1], vals[2], vals[3] = 2.0 ** 24, 4096.0, 4096.0, 1.0
    vals[256::256] = 0.15
    gs = [vals[i:i + 1].to(DEV) for i in range(count)]
    n = train.grad_norm(gs)
    out = torch.empty(count, device=DEV)
    for limit in (1e9, 1.0):
        assert torch.equal(train.clip_grad_norm_(gs, limit, out=out), n)
    assert torch.equal(train.clip_grad_norm_([g.clone() for g in gs], 1e9), n)
    assert abs(float(n) - 16777217.0) <= 1.0


def far_rows(d, dtype, seed=0):
    """an ordinary row; rows whose squares, or only their sum, pass fp32; a row near the type's largest values; one with an inf"""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(6, d, generator=g) * 2 - 1
    x[:, 0] = 0.75
    return (x * torch.tensor([1.0, 1.5e19, 1e30, 3.3e38, 1e25, 1.0])[:, None]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [1, 3, 7, 64, 120, 250, 520, 1000, 2050, 4100, 8200, 16000, 30000, 40001])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_squares_past_fp32(dtype, d, residual):
    base = far_rows(d, dtype, d)
    x, r = ((base.double() * 0.6).to(dtype), (base.double() * 0.4).to(dtype)) if residual else (base, None)
    x[5, d // 2] = math.inf
    w, gy, gs = 1 + 0.1 * rnd(d, seed=3), rnd(6, d, dtype=dtype, seed=4), rnd(6, d, dtype=dtype, scale=0.1, seed=5) if residual else None
    s, y64, dx64, mag, _, _ = norm64(x, r, w, 1e-6, gy, gs)
    rstd = 1 / (s.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    # rstd below the smallest normal number is off by half a step of 2^-149
    rel = (chain(d) + 8) * U + torch.where(rstd > 0, 2.0 ** -150 / rstd, torch.zeros_like(rstd))
    leaf, weight = x.to(DEV).requires_grad_(True), w.to(DEV)
    out = modules.rms_norm(leaf, weight, residual=r.to(DEV) if residual else None)
    y = out[0] if residual else out
    u = half_step(dtype)
    within(y, y64, u * y64.abs() + rel * y64.abs() + tiny(dtype), "y")
    (dx,) = torch.autograd.grad(out, leaf, [gy.to(DEV), gs.to(DEV)] if residual else [gy.to(DEV)])
    within(dx[:5], dx64[:5], u * dx64[:5].abs() + (2 * rel[:5] + (chain(d) + 16) * U) * mag[:5] + tiny(dtype), "dx")
    weight = weight.requires_grad_(True)
    z = modules.rms_norm(x[:5].to(DEV), weight, residual=r[:5].to(DEV) if residual else None)
    (dw,) = torch.autograd.grad(z[0] if residual else z, weight, gy[:5].to(DEV))
    *_, dw64, dwmag = norm64(x[:5], r[:5] if residual else None, w, 1e-6, gy[:5])
    within(dw, dw64, U * dw64.abs() + (float(rel[:5].max()) + 16 * U) * dwmag, "dw")
    for group in (0, 32, 512):
        q, scale = modules.rms_norm_q8(x[:5].to(DEV), w.to(DEV), residual=r[:5].to(DEV) if residual else None, group=group)[:2]
        g = group or d
        ng = -(-d // g)
        want = torch.nn.functional.pad(y64[:5].abs(), (0, ng * g - d)).view(5, ng, g).amax(-1) / 448
        off = rel[:5] + 4 * U
        within(scale, want, off * want, "scale")
        cols = scale.cpu().double().repeat_interleave(g, 1)[:, :d]
        err = (q.cpu().double() * cols - y64[:5]).abs()
        assert float((err - (2.0 ** -4 * (1 + off) * y64[:5].abs()).clamp_min(2.0 ** -10 * 1.01 * cols) - 2 * off * y64[:5].abs()).max()) <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d,group", [(5, 32), (64, 0), (300, 64), (1000, 512), (4096, 128), (40001, 0), (40001, 128)])
@pytest.mark.parametrize("weight", [1e-35, 1e-36, 1e-38, 1e-40, 1e-42, 1e-45])
def test_rms_norm_q8_of_tiny_outputs(dtype, d, group, weight):
    """scales below the smallest normal number are kept: 1 stands for a quotient that is 0, and for nothing else"""
    x, w = rnd(3, d, dtype=dtype, seed=1), (torch.full((d,), weight, dtype=torch.float64) * (1 + 0.1 * rnd(d, seed=2).double())).float()
    x[1] = 0
    q, scale = modules.rms_norm_q8(x.to(DEV), w.to(DEV), group=group)
    _, y = norm64(x, None, w, 1e-6)
    g = group or d
    ng = -(-d // g)
    want = torch.nn.functional.pad(y.abs(), (0, ng * g - d)).view(3, ng, g).amax(-1) / 448
    rel, step = (chain(d) + 12) * U, 2.0 ** -149
    scale = scale.cpu().double()
    # the largest value is off by half a step of 2^-149 at most, the quotient by another half
    zero = scale == 1
    assert (want[zero] <= 0.51 * step).all() and zero[1].all() and (want[~zero] >= 0.49 * step).all()
    within(scale[~zero], want[~zero], rel * want[~zero] + 0.51 * step, "scale")
    cols = scale.repeat_interleave(g, 1)[:, :d]
    dead = zero.repeat_interleave(g, 1)[:, :d]
    assert not q.cpu().double()[dead].any()
    # a scale rounded down by half a step saturates its largest values: 448 half steps; the value itself is off by half a step
    err = (q.cpu().double() * cols - y).abs()
    bound = (2.0 ** -4 * (1 + rel) * y.abs()).clamp_min(2.0 ** -10 * 1.01 * cols) + 2 * rel * y.abs() + (448 * 0.51 + 1) * step
    assert float((err - bound).masked_fill(dead, -1.0).max()) <= 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [1, 7, 64, 250, 520, 4100, 16000, 30000, 40001])
@pytest.mark.parametrize("eps", [0.0, 1e-37])
def test_rms_norm_squares_below_fp32(dtype, d, eps):
    """rows whose squares are too small for fp32, next to ordinary ones, where eps does not cover them"""
    x = (far_rows(d, torch.float64, d) / far_rows(d, torch.float64, d).abs().amax(-1, keepdim=True) *
         torch.tensor([1.0, 1e-12, 1e-18, 1e-22, 1e-30, 1e-37], dtype=torch.float64)[:, None]).to(dtype)
    w, gy = 1 + 0.1 * rnd(d, seed=3), rnd(6, d, dtype=dtype, seed=4)
    s, y64, dx64, mag, dw64, dwmag = norm64(x, None, w, eps, gy)
    rel = (chain(d) + 10) * U
    leaf, weight = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = modules.rms_norm(leaf, weight, eps=eps)
    within(y, y64, half_step(dtype) * y64.abs() + rel * y64.abs() + tiny(dtype), "y")
    dx, dw = torch.autograd.grad(y, [leaf, weight], gy.to(DEV))
    # rows of 1e-37 have gradients up to 1e37 times a few: within the types' range
    within(dx, dx64, half_step(dtype) * dx64.abs() + (2 * rel + (chain(d) + 16) * U) * mag + tiny(dtype), "dx")
    within(dw, dw64, U * dw64.abs() + (rel + 16 * U) * dwmag, "dw")
    q, scale = modules.rms_norm_q8(x.to(DEV), w.to(DEV), eps=eps)
    want = y64.abs().amax(-1, keepdim=True) / 448
    within(scale, want, (rel + 4 * U) * want, "scale")
    err = (q.cpu().double() * scale.cpu().double() - y64).abs()
    assert float((err - (2.0 ** -4 * (1 + rel) * y64.abs()).clamp_min(2.0 ** -10 * 1.01 * scale.cpu().double()) - 2 * rel * y64.abs()).max()) <= 0


def test_rms_norm_of_zeros_without_eps():
    y = modules.rms_norm(torch.zeros(2, 40, device=DEV), None, eps=0.0)
    assert torch.isnan(y).all()                             # 0 / 0, as the formula has it
    assert not modules.rms_norm(torch.zeros(2, 40, device=DEV), None, eps=1e-38).any()


def twice_cases():
    w, ids, r = rnd(9, seed=2).to(DEV), torch.zeros(3, dtype=torch.long, device=DEV), rnd(3, 9, seed=3).to(DEV)
    return {"norm": lambda a: modules.rms_norm(a, w), "norm, rows apart": lambda a: modules.rms_norm(a.t().contiguous().t(), w),
            "norm, residual": lambda a: modules.rms_norm(a, w, residual=r)[0], "stream": lambda a: modules.rms_norm(r, w, residual=a)[1],
            "norm of the stream": lambda a: modules.rms_norm(modules.rms_norm(r, w, residual=a)[1], None),
            "logp": lambda a: loss.token_logprobs(a, ids).logp, "entropy": lambda a: loss.token_logprobs(a, ids).entropy}


@pytest.mark.parametrize("name", ["norm", "norm, rows apart", "norm, residual", "stream", "norm of the stream", "logp", "entropy"])
def test_second_derivatives_are_refused_by_every_way(name):
    """and are not taken for zero: with respect to the input, the weight and the gradient that came in, by autograd.grad and torch.autograd.functional"""
    f, a = twice_cases()[name], rnd(3, 9, seed=1).to(DEV).requires_grad_(True)
    refused = lambda: pytest.raises(RuntimeError, match="once_differentiable")
    y = f(a)
    gy = torch.ones_like(y).requires_grad_(True)
    (g,) = torch.autograd.grad(y, a, gy, create_graph=True)
    for what in (a, gy):
        for unused in (False, True):
            with refused():
                torch.autograd.grad(g.square().sum(), what, retain_graph=True, allow_unused=unused)
    with refused():
        torch.autograd.functional.hessian(lambda b: f(b).sum(), a.detach())
    with refused():
        torch.autograd.functional.vhp(lambda b: f(b).square().sum(), a.detach(), torch.ones_like(a))
    with refused():
        torch.autograd.functional.jvp(f, a.detach(), torch.ones_like(a))
    # the first derivatives that carry that refusal are the ordinary ones
    (plain,) = torch.autograd.grad(f(a), a, gy.detach())
    assert torch.equal(g, plain) and not plain.requires_grad
    assert torch.autograd.functional.jacobian(lambda b: f(b).sum(0), a.detach()).shape[-2:] == a.shape


def test_second_derivatives_of_the_weight_are_refused():
    x, w = rnd(3, 9, seed=1).to(DEV), rnd(9, seed=2).to(DEV).requires_grad_(True)
    (g,) = torch.autograd.grad(modules.rms_norm(x, w).square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(g.sum(), w, allow_unused=True)
