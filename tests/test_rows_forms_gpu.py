"""Row operators: every form that the rules on sizes and types choose, against the formulas in 64 bits, and every output and workspace between
guards.  Tolerances as in test_rows_gpu.py, unless a test says otherwise."""
import ctypes as C
import math

import pytest
import torch

from i2pnet_amd import _lib, loss, modules, train
from test_rows_gpu import DEV, TYPES, U, chain, half_step, logp64, logp_tol, norm64, rnd, tiny, within

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


# ---- RMS norm --------------------------------------------------------------------------------------------------------------------
# rows of one to four vectors for each of 8 .. 1024 threads, in whole vectors and with a partial last one
WIDTHS = {4: [24, 57, 100, 200, 400, 700, 1100, 1999, 3001, 4090, 6000, 12001, 16384],
          2: [40, 100, 201, 500, 1000, 2000, 2500, 3900, 6003, 8192, 12000, 16385, 20000, 24577, 32768]}


@pytest.mark.parametrize("dtype,d", [(t, d) for t in TYPES for d in WIDTHS[torch.finfo(t).bits // 8]], ids=str)
def test_rms_norm_at_every_width(dtype, d):
    rows = 7
    x, r, w = rnd(rows, d, dtype=dtype, seed=1), rnd(rows, d, dtype=dtype, scale=2.0, seed=2), 1 + 0.1 * rnd(d, seed=3)
    gy, gs = rnd(rows, d, dtype=dtype, seed=4), rnd(rows, d, dtype=dtype, seed=5)
    leaf, weight = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y, s = modules.rms_norm(leaf, weight, residual=r.to(DEV), eps=1e-5)
    s64, y64, dx64, mag, dw64, dwmag = norm64(x, r, w, 1e-5, gy, gs)
    assert torch.equal(s.detach().cpu(), s64)
    within(y, y64, (half_step(dtype) + (chain(d) + 8) * U) * y64.abs() + tiny(dtype), "y")
    dx, dw = torch.autograd.grad([y, s], [leaf, weight], [gy.to(DEV), gs.to(DEV)])
    within(dx, dx64, half_step(dtype) * dx64.abs() + (2 * chain(d) + 16) * U * mag + tiny(dtype), "dx")
    within(dw, dw64, U * dw64.abs() + (rows + chain(d) + 16) * U * dwmag, "dw")


@pytest.mark.parametrize("dtype,d", [(torch.float32, 1999), (torch.bfloat16, 2500), (torch.float16, 3900), (torch.bfloat16, 20001), (torch.float32, 16390)], ids=str)
def test_rms_norm_backward_of_more_rows_than_blocks(dtype, d):
    """a block walks several rows and sums their weight gradients: 1100 rows on at most 1024 blocks (256 and fewer of the wide ones)"""
    rows = 1100
    x, w, gy = rnd(rows, d, dtype=dtype, seed=1), 1 + 0.1 * rnd(d, seed=3), rnd(rows, d, dtype=dtype, seed=4)
    leaf, weight = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    dx, dw = torch.autograd.grad(modules.rms_norm(leaf, weight, eps=1e-5), [leaf, weight], gy.to(DEV))
    _, _, dx64, mag, dw64, dwmag = norm64(x, None, w, 1e-5, gy)
    within(dx, dx64, half_step(dtype) * dx64.abs() + (2 * chain(d) + 16) * U * mag + tiny(dtype), "dx")
    within(dw, dw64, U * dw64.abs() + (rows + chain(d) + 16) * U * dwmag, "dw")


def test_rms_norm_module():
    m = modules.RMSNorm(48, eps=1e-3).to(DEV)
    assert list(m.state_dict()) == ["weight"] and m.weight.eq(1).all() and m.weight.dtype == torch.float32
    with torch.no_grad():
        m.weight.copy_(1 + 0.1 * rnd(48, seed=1))
    for dtype in TYPES:
        x, r = rnd(3, 5, 48, dtype=dtype, seed=2).to(DEV), rnd(3, 5, 48, dtype=dtype, seed=3).to(DEV)
        assert torch.equal(m(x), modules.rms_norm(x, m.weight, eps=1e-3))
        y, s = m(x, residual=r)
        y2, s2 = modules.rms_norm(x, m.weight, residual=r, eps=1e-3)
        assert torch.equal(y, y2) and torch.equal(s, s2) and y.shape == x.shape
        m.zero_grad()
        y.float().square().sum().backward()
        _, y64, _, _, dw64, dwmag = norm64(x.cpu(), r.cpu(), m.weight.detach().cpu(), 1e-3, 2 * y.detach().float().cpu())
        within(m.weight.grad, dw64, U * dw64.abs() + (15 + chain(48) + 16) * U * dwmag + half_step(dtype) * dwmag, "dw")
    h = modules.RMSNorm(48).to(DEV).bfloat16()
    x = rnd(2, 48, dtype=torch.bfloat16, seed=2).to(DEV)
    (g,) = torch.autograd.grad(h(x).sum(), h.weight)
    assert g.dtype == torch.bfloat16


# ---- log probabilities -----------------------------------------------------------------------------------------------------------
def many_rows(rows, v, dtype, mask, seed=1):
    """scores of many rows on the device, with rows of every special kind -> scores, ids, rows to look at"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.empty(rows, v, dtype=dtype, device=DEV).normal_(0.0, 3.0, generator=g)
    ids = torch.randint(0, v, (rows,), device=DEV, generator=g)
    if mask is not None:
        drop = torch.rand(v, device=DEV, generator=g) < 0.25
        kept = x.gather(1, ids[:, None])
        x[:, drop] = mask if math.isinf(mask) else torch.finfo(dtype).min
        x.scatter_(1, ids[:, None], kept)
    x[3] = 1.5                                              # all equal
    x[4] = (x[4] * 0.5).round()                             # many ties
    x[5, v // 2:v // 2 + 50] = 20.0                         # the best sit together
    x[7, :-3] = -math.inf                                   # fewer candidates than alternatives
    ids[7] = v - 2
    some = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 8, rows // 2, rows // 2 + 1, rows - 3, rows - 2, rows - 1])
    return x, ids, some


def check_some(x, ids, some, top, o, grads=None, gl=None, gh=None):
    v, dtype = x.shape[1], x.dtype
    xs, k, at = x.detach()[some.to(DEV)].cpu(), ids[some.to(DEV)].cpu(), some.to(DEV)
    ref = logp64(xs, k, top, *(() if grads is None else (gl[at].cpu(), gh[at].cpu())))
    lp, H, tl, ti = ref[:4]
    within(o.logp[at], lp, logp_tol(v, lp, 16), "logp")
    within(o.entropy[at], H, (chain(v) + 64) * U * 33 * torch.ones_like(H), "entropy")
    assert torch.equal(o.top_ids[at].cpu(), ti)
    within(o.top_logp[at], tl, logp_tol(v, tl.clamp_min(-1e37), 16), "top_logp")
    if grads is not None:
        dx, mag = ref[4:]
        g = 1 + gl[at].cpu().abs() + gh[at].cpu().abs()
        within(grads[at], dx, half_step(dtype) * dx.abs() + (8 * chain(v) + 2000) * U * mag + g[:, None] * 1e-36 + tiny(dtype), "dlogits")


@pytest.mark.parametrize("dtype", HALVES, ids=str)
@pytest.mark.parametrize("rows,v", [(16400, 8201), (8200, 40001)])
@pytest.mark.parametrize("top,mask", [(0, None), (8, -math.inf), (32, 0.0), (1, None)])
def test_token_logprobs_64_scores_a_thread(dtype, rows, v, top, mask):
    """whole rows and slices of 8193 .. 16384 scores of the 16-bit types, as many rows take them"""
    x, ids, some = many_rows(rows, v, dtype, mask)
    x[10] = -math.inf
    x[11, 77] = math.nan
    x[12, v - 1] = math.inf
    x[13] = math.nan                                        # padding: not read
    ids[13], ids[14] = -100, v
    leaf = x.requires_grad_(True)
    o = loss.token_logprobs(leaf, ids, top=top)
    gl, gh = torch.randn(rows, device=DEV), torch.randn(rows, device=DEV)
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl, gh])
    check_some(x, ids, some, top, o, d, gl, gh)
    assert o.logp[10] == -math.inf and o.entropy[10] == 0 and not d[10].any()
    assert torch.isnan(o.logp[11:13]).all() and torch.isnan(o.entropy[11:13]).all() and torch.isnan(d[11:13]).all() and torch.isnan(o.logp[14])
    assert o.logp[13] == 0 and o.entropy[13] == 0 and not d[13].any() and torch.isfinite(o.entropy[14])
    if top:
        assert o.top_ids[10].tolist() == list(range(top)) and o.top_ids[11, 0] == 77 and o.top_ids[12, 0] == v - 1 and o.top_ids[13].eq(-1).all()
    # every row against the form that few rows take
    with torch.no_grad():
        for lo in range(0, rows, 512):
            p = loss.token_logprobs(x[lo:lo + 512], ids[lo:lo + 512], top=top)
            assert torch.equal(p.top_ids, o.top_ids[lo:lo + 512])
            a, b = torch.nan_to_num(p.logp), torch.nan_to_num(o.logp[lo:lo + 512])
            assert float((a - b).abs().sub(2 * logp_tol(v, a.clamp_min(-1e30), 16)).max()) <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,v,top,mask", [(600, 40001, 8, -math.inf), (600, 40000, 32, None), (700, 20003, 5, 0.0), (520, 8200, 32, None)])
def test_token_logprobs_slices_of_many_rows(dtype, rows, v, top, mask):
    """slices of up to 8192 scores with alternatives, joined"""
    x, ids, some = many_rows(rows, v, dtype, mask)
    check_some(x, ids, some, top, loss.token_logprobs(x, ids, top=top))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,v,top", [(1, 1 << 21, 32), (1, (1 << 20) + 5, 8), (2, (1 << 21) - 7, 0), (3, (1 << 20) + 12345, 32)])
def test_token_logprobs_the_widest_rows(dtype, rows, v, top):
    """up to 256 slices of a row"""
    x, ids = rnd(rows, v, dtype=dtype, scale=3.0, seed=1).to(DEV), torch.arange(rows, device=DEV) * 1000003 % v
    leaf = x.requires_grad_(True)
    o = loss.token_logprobs(leaf, ids, top=top)
    gl, gh = torch.ones(rows, device=DEV), 0.5 * torch.ones(rows, device=DEV)
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl, gh])
    check_some(x, ids, torch.arange(rows), top, o, d, gl, gh)


def test_token_logprobs_more_slices_than_one_launch_takes():
    """2^21 blocks a launch: 2^20 rows of two slices, and some more"""
    rows, v, top = (1 << 20) + 77, 8193, 2
    x, ids, some = many_rows(rows, v, torch.float32, None)
    some = torch.cat([some, torch.tensor([(1 << 20) - 1, 1 << 20, (1 << 20) + 1])])
    ids[(1 << 20) + 1] = -100
    leaf = x.requires_grad_(True)
    o = loss.token_logprobs(leaf, ids, top=top)
    gl, gh = torch.ones(rows, device=DEV), 0.5 * torch.ones(rows, device=DEV)
    (d,) = torch.autograd.grad([o.logp, o.entropy], leaf, [gl, gh])
    check_some(x, ids, some[:-1], top, o, d, gl, gh)
    assert o.logp[some[-1]] == 0 and o.top_ids[some[-1]].eq(-1).all() and not d[some[-1]].any()
    assert int(o.logp.ge(0).sum()) == 1 and torch.isfinite(o.entropy).all()
    del x, leaf, d, o
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,v", [(40, 32), (30, 100), (20, 468), (9, 5000), (4, 32000), (2, 131072)])
def test_token_logprobs_gradient_keeps_its_digits(rows, v):
    """fp32, the log probability's gradient alone: p is off by the sum's error and its own.  A sum's chain is at most 64 scores of a thread, 10
    steps over its lanes and slices and 16 waves: 90 U; its terms e^z by (2 + 1.3 |z|) U each, on the average over p; the logarithm and the
    three steps to log p by U |log p| each; e^z again by (2 + 1.3 |log p|) U"""
    x, ids = rnd(rows, v, scale=3.0, seed=v), torch.arange(rows) % v
    gl = rnd(rows, seed=2)
    leaf = x.to(DEV).requires_grad_(True)
    (d,) = torch.autograd.grad(loss.token_logprobs(leaf, ids.to(DEV)).logp, leaf, gl.to(DEV))
    lp = torch.log_softmax(x.double(), -1)
    p, z = lp.exp(), x.double() - x.double().amax(-1, keepdim=True)
    rel = (90 + 2 + 1.3 * (p * z.abs()).sum(-1, keepdim=True) + 3 * lp.abs() + 2 + 1.3 * lp.abs() + z.abs() + 4) * U
    want = -p * gl.double()[:, None]
    want.scatter_add_(1, ids[:, None], gl.double()[:, None])
    within(d, want, rel * p * gl.double().abs()[:, None] + U * want.abs() + 1e-36, "dlogits")


# ---- outputs and workspaces between guards ---------------------------------------------------------------------------------------
class Guarded:
    """buffers in the middle of larger ones, all of whose bytes are the same before a call"""
    PAD, FILL = 4096, 0xA5

    def __init__(self):
        self.all = []

    def __call__(self, nbytes, shift=0):
        t = torch.full((2 * self.PAD + nbytes + 16,), self.FILL, dtype=torch.uint8, device=DEV)
        lo = self.PAD + shift
        self.all.append((t, lo, lo + nbytes))
        return C.c_void_p(t.data_ptr() + lo)

    def get(self, i, dtype, *shape):
        t, lo, hi = self.all[i]
        return t[lo:hi].clone().view(dtype).view(shape)

    def check(self, what):
        for i, (t, lo, hi) in enumerate(self.all):
            assert t[:lo].eq(self.FILL).all() and t[hi:].eq(self.FILL).all(), (what, i)


def p(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 3), (5, 7), (3, 65), (19, 129), (4, 257), (3, 2051), (2, 4103), (2, 9001), (2, 17001), (2, 40001), (300, 96)])
def test_rms_norm_writes_between_guards(dtype, rows, d):
    es, dt, st = torch.finfo(dtype).bits // 8, CODE[dtype], torch.cuda.current_stream().cuda_stream
    x, r, w = (t.to(DEV) for t in (rnd(rows, d, dtype=dtype, seed=1), rnd(rows, d, dtype=dtype, seed=2), 1 + 0.1 * rnd(d, seed=3)))
    gy, gs = rnd(rows, d, dtype=dtype, seed=4).to(DEV), rnd(rows, d, dtype=dtype, seed=5).to(DEV)
    g = Guarded()
    s, y, rstd = g(rows * d * es, es), g(rows * d * es, 3 * es), g(rows * 4, 4)
    _lib.call("i2p_rms_norm_fwd", rows, d, dt, 0, p(x), d, p(r), d, p(w), 1e-6, s, y, rstd, stream=st)
    leaf, weight = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = modules.rms_norm(leaf, weight, residual=r)
    dx, dw, scratch = g(rows * d * es, es), g(d * 4, 4), g(_lib.helper("i2p_rms_norm_bwd_scratch", rows, d))
    _lib.call("i2p_rms_norm_bwd", rows, d, dt, 0, s, d, p(gy), d, p(gs), d, p(w), rstd, dx, dw, scratch, stream=st)
    grads = torch.autograd.grad(want, [leaf, weight], [gy, gs])
    for group in (0, 32, 256, 512):
        ng = -(-d // group) if group else 1
        s2, q, scale = g(rows * d * es, es), g(rows * d, 1), g(rows * ng * 4, 4)
        _lib.call("i2p_rms_norm_q8", rows, d, dt, 0, p(x), d, p(r), d, p(w), 1e-6, group, s2, q, scale, stream=st)
    g.check((rows, d))
    assert torch.equal(g.get(0, dtype, rows, d), want[1]) and torch.equal(g.get(1, dtype, rows, d), want[0])
    assert torch.equal(g.get(3, dtype, rows, d), grads[0]) and torch.equal(g.get(4, torch.float32, d), grads[1])
    for i, group in enumerate((0, 32, 256, 512)):
        ng = -(-d // group) if group else 1
        q, scale, s2 = modules.rms_norm_q8(x, w, residual=r, group=group)
        assert torch.equal(g.get(6 + 3 * i, dtype, rows, d), s2) and torch.equal(g.get(7 + 3 * i, torch.uint8, rows, d), q.view(torch.uint8))
        assert torch.equal(g.get(8 + 3 * i, torch.float32, rows, ng), scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (3, 5, 5), (37, 33, 4), (3, 130, 32), (5, 513, 0), (3, 2049, 3), (2, 9001, 32), (600, 9001, 3), (2, 40001, 7), (1, 131073, 32)])
def test_token_logprobs_writes_between_guards(dtype, rows, v, top):
    es, dt, st = torch.finfo(dtype).bits // 8, CODE[dtype], torch.cuda.current_stream().cuda_stream
    x, ids = rnd(rows, v, dtype=dtype, seed=1).to(DEV), (torch.arange(rows) * 7 % v).to(DEV)
    ids[rows - 1] = -100 if rows > 2 else ids[rows - 1]
    leaf = x.clone().requires_grad_(True)
    want = loss.token_logprobs(leaf, ids, top=top)
    g = Guarded()
    logp, H, stat, tl, ti = g(rows * 4, 4), g(rows * 4, 4), g(rows * 8, 4), g(rows * top * 4, 4), g(rows * top * 8, 8)
    scratch = g(_lib.helper("i2p_token_logprobs_scratch", rows, v, dt, top))
    _lib.call("i2p_token_logprobs_fwd", rows, v, dt, p(x), v, p(ids), -100, top, logp, H, stat, tl, ti, scratch, stream=st)
    dx, gl, gh = g(rows * v * es, es), torch.ones(rows, device=DEV), torch.ones(rows, device=DEV)
    _lib.call("i2p_token_logprobs_bwd", rows, v, dt, p(x), v, p(ids), -100, stat, H, p(gl), p(gh), dx, stream=st)
    (grad,) = torch.autograd.grad([want.logp, want.entropy], leaf, [gl, gh])
    g.check((rows, v, top))
    assert torch.equal(g.get(0, torch.float32, rows), want.logp) and torch.equal(g.get(1, torch.float32, rows), want.entropy)
    assert torch.equal(g.get(3, torch.float32, rows, top), want.top_logp) and torch.equal(g.get(4, torch.int64, rows, top), want.top_ids)
    assert torch.equal(g.get(6, dtype, rows, v), grad)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 7, 1], [4095, 4097, 1], [16385] * 3, [5] * 700, [6000000, 9]], ids=lambda s: f"{len(s)}, {sum(s)}")
def test_clipping_writes_between_guards(sizes, into):
    st = torch.cuda.current_stream().cuda_stream
    types = [TYPES[i % 3] for i in range(len(sizes))]
    vals = [rnd(k, dtype=t, seed=i).to(DEV) for i, (k, t) in enumerate(zip(sizes, types))]
    g = Guarded()
    ptrs = [g(k * (torch.finfo(t).bits // 8), torch.finfo(t).bits // 8) for k, t in zip(sizes, types)]
    for (t, lo, hi), v in zip(g.all, vals):
        t[lo:hi] = v.view(torch.uint8)
    n = len(sizes)
    a, b, c = (C.c_void_p * n)(*[q.value for q in ptrs]), (C.c_longlong * n)(*sizes), (C.c_int * n)(*[CODE[t] for t in types])
    out = g(4 * sum(sizes), 4) if into else None
    total, scratch = g(4, 4), g(_lib.helper("i2p_grad_norm_scratch", n, C.cast(b, C.c_void_p)))
    _lib.call("i2p_clip_grad_norm", n, C.cast(a, C.c_void_p), C.cast(b, C.c_void_p), C.cast(c, C.c_void_p), 0, 1, 0.25, out, scratch, total, stream=st)
    keep = [v.clone() for v in vals]
    flat = torch.empty(sum(sizes), device=DEV) if into else None
    norm = train.clip_grad_norm_(keep, 0.25, out=flat)
    g.check(len(sizes))
    for i, (k, t) in enumerate(zip(sizes, types)):
        assert torch.equal(g.get(i, t, k), keep[i])
    assert torch.equal(g.get(n + into, torch.float32), norm.view(())) and (not into or torch.equal(g.get(n, torch.float32, sum(sizes)), flat))
