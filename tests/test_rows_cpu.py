"""Row operators without a GPU: what is refused before any launch."""
import ctypes as C
import math
from pathlib import Path

import pytest
import torch

from i2pnet_amd import _lib, loss, modules, ops, train

BAD, OVERLAP = "bad argument", "share memory"


def call(name, *args):
    _lib.call(name, *args)


P = 4096        # stands for a device pointer: every call here is refused before anything is launched


@pytest.mark.parametrize("change", [dict(rows=-1), dict(d=0), dict(d=-4), dict(dtype=3), dict(dtype=-1), dict(wdtype=2), dict(ldx=7), dict(ldr=7), dict(x=None),
                                    dict(y=None), dict(s=None), dict(res=None)])
def test_rms_norm_forward_refusals(change):
    a = dict(rows=2, d=8, dtype=1, wdtype=0, x=P, ldx=8, res=P, ldr=8, w=P, eps=1e-6, s=P, y=P, rstd=P) | change
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_rms_norm_fwd", *a.values())


@pytest.mark.parametrize("change", [dict(group=16), dict(group=48), dict(group=1024), dict(group=-32), dict(q=None), dict(scale=None), dict(d=0), dict(dtype=9),
                                    dict(wdtype=1, dtype=2)])
def test_rms_norm_q8_refusals(change):
    a = dict(rows=2, d=8, dtype=1, wdtype=0, x=P, ldx=8, res=None, ldr=0, w=P, eps=1e-6, group=32, s=None, q=P, scale=P) | change
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_rms_norm_q8", *a.values())


@pytest.mark.parametrize("change", [dict(rows=0), dict(d=0), dict(dtype=3), dict(lds=3), dict(ldgy=3), dict(ldgs=3), dict(s=None), dict(gy=None), dict(rstd=None),
                                    dict(dx=None), dict(scratch=None)])
def test_rms_norm_backward_refusals(change):
    a = dict(rows=2, d=8, dtype=1, wdtype=0, s=P, lds=8, gy=P, ldgy=8, gs=P, ldgs=8, w=P, rstd=P, dx=P, dw=P, scratch=P) | change
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_rms_norm_bwd", *a.values())


@pytest.mark.parametrize("change", [dict(rows=-1), dict(v=0), dict(v=(1 << 21) + 1, ldx=1 << 22), dict(dtype=3), dict(ldx=3), dict(top=-1), dict(top=9), dict(v=100, ldx=100, top=33),
                                    dict(x=None), dict(ids=None), dict(logp=None), dict(entropy=None), dict(top_logp=None), dict(top_ids=None)])
def test_token_logprobs_refusals(change):
    a = dict(rows=2, v=8, dtype=1, x=P, ldx=8, ids=P, ignore=-100, top=2, logp=P, entropy=P, stat=P, top_logp=P, top_ids=P, scratch=P) | change
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_token_logprobs_fwd", *a.values())


def test_token_logprobs_needs_its_scratch():
    assert _lib.helper("i2p_token_logprobs_scratch", 1, 1 << 20, 0, 0) > 0 and _lib.helper("i2p_token_logprobs_scratch", 1, 1000, 0, 32) == 0
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_token_logprobs_fwd", 1, 1 << 20, 0, P, 1 << 20, P, -100, 0, P, P, P, P, P, None)


@pytest.mark.parametrize("change", [dict(v=0), dict(dtype=3), dict(ldx=3), dict(x=None), dict(ids=None), dict(stat=None), dict(entropy=None), dict(dx=None)])
def test_token_logprobs_backward_refusals(change):
    a = dict(rows=2, v=8, dtype=1, x=P, ldx=8, ids=P, ignore=-100, stat=P, entropy=P, gl=None, gh=None, dx=P) | change
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_token_logprobs_bwd", *a.values())


def clip(ptrs, sizes, dtypes, kind=0, do=1, limit=1.0, out=None, scratch=P, total=P, n=None):
    a = (C.c_void_p * max(1, len(ptrs)))(*ptrs)
    b = (C.c_longlong * max(1, len(sizes)))(*sizes)
    c = (C.c_int * max(1, len(dtypes)))(*dtypes)
    call("i2p_clip_grad_norm", len(ptrs) if n is None else n, C.cast(a, C.c_void_p), C.cast(b, C.c_void_p), C.cast(c, C.c_void_p), kind, do, limit, out, scratch, total)


@pytest.mark.parametrize("args,what", [
    (([P], [-1], [0]), BAD), (([P], [4], [3]), BAD), (([None], [4], [0]), BAD), (([P + 2], [4], [0]), BAD), (([P + 1], [4], [1]), BAD), (([1 << 50], [4], [0]), BAD),
    (([P, P], [1 << 44, 1], [0, 0]), BAD),
    (([P, P], [4, 4], [0, 0]), OVERLAP), (([P, P + 12], [4, 4], [0, 0]), OVERLAP), (([P + 14, P], [4, 8], [1, 1]), OVERLAP)])
def test_clip_grad_norm_refusals(args, what):
    with pytest.raises(_lib.I2POpsError, match=what):
        clip(*args)


@pytest.mark.parametrize("change", [dict(kind=2), dict(kind=-1), dict(limit=-1.0), dict(limit=math.nan), dict(scratch=None), dict(scratch=P + 8), dict(total=None), dict(n=-1)])
def test_clip_grad_norm_argument_refusals(change):
    with pytest.raises(_lib.I2POpsError, match=BAD):
        clip([P], [4], [0], **change)


def test_clip_grad_norm_output_must_not_overlap():
    for out in (P, P + 12, P - 28):
        with pytest.raises(_lib.I2POpsError, match=OVERLAP):
            clip([P, P + 1024], [4, 4], [0, 0], out=out)


def test_rows_too_long():
    d = (1 << 30) + 1
    for name, args in (("i2p_rms_norm_fwd", (1, d, 1, 0, P, d, None, 0, None, 1e-6, None, P, None)),
                       ("i2p_rms_norm_q8", (1, d, 1, 0, P, d, None, 0, None, 1e-6, 0, None, P, P)),
                       ("i2p_rms_norm_bwd", (1, d, 1, 0, P, d, P, d, None, 0, None, P, P, None, None))):
        with pytest.raises(_lib.I2POpsError, match=BAD):
            call(name, *args)


def test_scratch_sizes():
    n = (C.c_longlong * 3)(1, 0, (1 << 31) + 5)
    assert _lib.helper("i2p_grad_norm_scratch", 3, C.cast(n, C.c_void_p)) >= 8
    assert _lib.helper("i2p_grad_norm_scratch", 0, None) >= 8
    assert _lib.helper("i2p_rms_norm_bwd_scratch", 0, 8) == 0 and _lib.helper("i2p_rms_norm_bwd_scratch", 1000000, 4096) >= 4096 * 4


def test_host_tensors_and_types_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for f in (lambda: modules.rms_norm(x, w), lambda: modules.rms_norm_q8(x, w), lambda: loss.token_logprobs(x, torch.zeros(2, dtype=torch.long)),
              lambda: train.clip_grad_norm_([x], 1.0), lambda: train.grad_norm([x])):
        with pytest.raises(RuntimeError, match="cuda"):
            f()
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        train.clip_grad_norm_([x.double()], 1.0)
    with pytest.raises(RuntimeError, match="no gradient"):
        modules.rms_norm_q8(x.clone().requires_grad_(True), w)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            train.clip_grad_norm_([x], bad)
    with pytest.raises(ValueError, match="norm_type"):
        train.clip_grad_norm_([x], 1.0, norm_type=1)
    with pytest.raises(RuntimeError, match="leaves"):
        train.clip_grad_norm_([(x.clone().requires_grad_(True) * 2)], 1.0)
    with pytest.raises(RuntimeError, match="leaves"):
        train.clip_grad_norm_([3.0], 1.0)


def test_other_tensor_classes_are_refused_as_gradients():
    class Other(torch.Tensor):
        pass
    with pytest.raises(RuntimeError, match="wanted"):
        train._grad_list([torch.zeros(3).as_subclass(Other)])
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.rows().clip_grad_norm([], 0, 1.0, None)
    with pytest.raises(RuntimeError, match="cuda"):
        ops.rows().rms_norm_backward(torch.zeros(2, 3), None, torch.zeros(2), torch.zeros(2, 3), None, True)


def test_lists_of_parameters():
    a, b, c = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    a.grad = torch.ones(3)
    c.requires_grad_(False)
    raw = torch.zeros(2)
    assert train._grad_list([a, b, c, raw])[0] is a.grad and len(train._grad_list([a, b, c, raw])) == 2
    assert train._grad_list(raw)[0] is raw and train._grad_list(x for x in ()) == []
    assert isinstance(ops.MAX_TOP, int)


def rows_calls(x, r, w, ids):
    """every public row operator on the given tensors"""
    return {"rms_norm": lambda: modules.rms_norm(x, w), "rms_norm residual": lambda: modules.rms_norm(x, w, residual=r)[0],
            "rms_norm_q8": lambda: modules.rms_norm_q8(x, w, residual=r)[0], "token_logprobs": lambda: loss.token_logprobs(x, ids).logp,
            "grad_norm": lambda: train.grad_norm([x]), "clip_grad_norm_": lambda: train.clip_grad_norm_([x], 1.0),
            "clip_grad_norm_ out": lambda: train.clip_grad_norm_([x], 1.0, out=r.reshape(-1))}


@pytest.mark.parametrize("name", sorted(rows_calls(*[torch.zeros(1)] * 4)))
@pytest.mark.parametrize("which", ["x", "r", "w"])
def test_forward_mode_is_refused(name, which):
    """a tangent would be lost without a word: the outputs carry none"""
    t = {"x": torch.ones(2, 8), "r": torch.ones(2, 8), "w": torch.ones(8)}
    with torch.autograd.forward_ad.dual_level():
        t[which] = torch.autograd.forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        uses = {"x": True, "r": name in ("rms_norm residual", "rms_norm_q8", "clip_grad_norm_ out"),
                "w": name.startswith("rms_norm")}[which]
        if uses:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                rows_calls(t["x"], t["r"], t["w"], torch.zeros(2, dtype=torch.long))[name]()


def test_forward_mode_through_a_backward_pass_is_refused():
    s, g, one = torch.ones(2, 8), torch.ones(2, 8), torch.ones(2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual
        for a, b, c in ((dual(s, g), g, None), (s, dual(g, g), None), (s, g, dual(g, g))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.rows().rms_norm_backward(a, None, one, b, c, False)
        ids, stat = torch.zeros(2, dtype=torch.long), torch.zeros(2, 2)
        for a, b, c in ((dual(s, g), one, one), (s, dual(one, one), None), (s, None, dual(one, one))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.rows().token_logprobs_backward(a, ids, -100, stat, one, b, c)


@pytest.mark.parametrize("name", sorted(rows_calls(*[torch.zeros(1)] * 4)))
def test_a_call_that_is_being_traced_is_refused(name):
    """a trace would hold the allocation of the outputs and not the launch: replayed, it would return what memory held"""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, r, w, ids = torch.ones(2, 8), torch.ones(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.long)
    f = lambda a, b, c: rows_calls(a, b, c, ids)[name]() + 0
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(f, (x, r, w), check_trace=False)
    for pre in (False, True):
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f, pre_dispatch=pre)(x, r, w)


def test_a_backward_pass_that_is_being_traced_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    s, one, ids = torch.ones(2, 8), torch.ones(2), torch.zeros(2, dtype=torch.long)
    for f in (lambda a: ops.rows().rms_norm_backward(a, None, one, a, None, False)[0],
              lambda a: ops.rows().token_logprobs_backward(a, ids, -100, torch.zeros(2, 2), one, one, None)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (s,), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(s)


def test_parameters_without_gradients_have_a_norm_of_zero_on_their_device():
    p = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(2), requires_grad=False)]
    for f in (lambda a: train.grad_norm(a), lambda a: train.clip_grad_norm_(a, 1.0), lambda a: train.clip_grad_norm_(a, 1.0, error_if_nonfinite=True),
              lambda a: train.clip_grad_norm_(a, 1.0, out=torch.zeros(0))):
        for a in (p, p[0], iter(p), p[1:]):
            n = f(a)
            assert n.device.type == "cpu" and n.dtype == torch.float32 and n.shape == () and float(n) == 0.0
    with pytest.raises(RuntimeError, match="out must be empty"):
        train.clip_grad_norm_(p, 1.0, out=torch.zeros(1))


def test_the_longest_row():
    """I2P_MAX_ROW itself: the row after it is refused, and by the tensor checks too"""
    for d, ok in ((1 << 26, True), ((1 << 26) + 1, False)):
        for name, args in (("i2p_rms_norm_fwd", (0, d, 1, 0, None, d, None, 0, None, 1e-6, None, None, None)),
                           ("i2p_rms_norm_q8", (0, d, 1, 0, None, d, None, 0, None, 1e-6, 0, None, None, None))):
            if ok:
                call(name, *args)                           # (no rows is no work)
            else:
                with pytest.raises(_lib.I2POpsError, match=BAD):
                    call(name, *args)
    with pytest.raises(_lib.I2POpsError, match=BAD):
        call("i2p_rms_norm_bwd", 1, (1 << 26) + 1, 1, 0, P, (1 << 26) + 1, P, (1 << 26) + 1, None, 0, None, P, P, None, None)
    assert _lib.helper("i2p_rms_norm_bwd_scratch", 1, 1 << 26) == 4 << 26


def test_limits_are_the_header_s():
    text = (Path(__file__).resolve().parent.parent / "include" / "i2p_ops.h").read_text()
    assert f"#define I2P_MAX_TOP {ops.MAX_TOP}\n" in text and "#define I2P_MAX_CANDIDATES (1 << 21)\n" in text and "#define I2P_MAX_ROW (1 << 26)\n" in text
    a = dict(rows=0, v=100, dtype=1, x=None, ldx=1 << 22, ids=None, ignore=-100, top=ops.MAX_TOP, logp=None, entropy=None, stat=None, top_logp=None, top_ids=None,
             scratch=None)
    call("i2p_token_logprobs_fwd", *a.values())
    call("i2p_token_logprobs_fwd", *(a | dict(v=1 << 21)).values())
    for change in (dict(top=ops.MAX_TOP + 1), dict(v=(1 << 21) + 1)):
        with pytest.raises(_lib.I2POpsError, match=BAD):
            call("i2p_token_logprobs_fwd", *(a | change).values())
