"""The serving calls have no derivatives: tensors that carry a gradient or a
forward-mode tangent, which a call would lose without a word, are refused."""
import pytest
import torch
from torch.autograd import forward_ad

import htree_amd
from htree_amd.cache import no_derivatives


def test_no_derivatives():
    x = torch.zeros(3)
    w = torch.zeros(3, requires_grad=True)
    no_derivatives("f", x, None)
    with pytest.raises(AssertionError, match="f has no backward"):
        no_derivatives("f", x, None, w)
    with torch.no_grad():
        no_derivatives("f", w)
    with forward_ad.dual_level():
        no_derivatives("f", x, None)
        d = forward_ad.make_dual(x, torch.ones(3))
        for t in (d, d[1:], d.view(3, 1)):
            with pytest.raises(AssertionError, match="f has no forward-mode derivative"), torch.no_grad():
                no_derivatives("f", None, t)


def tensors(dtype=torch.float32):
    f = lambda *n: torch.zeros(n, dtype=dtype, device="cuda:0")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    attend = dict(q=f(2, 8, 64), k_cache=f(4, 16, 2, 64), v_cache=f(4, 16, 2, 64), block_table=i32([[0, 1, 2]]),
                  lens=i32([40]), starts=i32([0, 2]), out=f(2, 8, 64))
    append = dict(k=f(2, 2, 64), v=f(2, 2, 64), k_cache=f(4, 16, 2, 64), v_cache=f(4, 16, 2, 64),
                  slots=torch.tensor([1, 2], device="cuda:0"), q=f(2, 8, 64), positions=i32([0, 1]),
                  cos=f(4, 32), sin=f(4, 32))
    return {"draft_attention": attend, "cache_append": append}


NAMES = [("draft_attention", n) for n in ("q", "k_cache", "v_cache", "out")] + \
    [("cache_append", n) for n in ("k", "v", "q", "k_cache", "v_cache", "cos", "sin")]


@pytest.mark.gpu
@pytest.mark.parametrize("call,name", NAMES)
def test_calls_refuse(call, name):
    f, args = getattr(htree_amd, call), tensors()[call]
    f(**args)
    with pytest.raises(AssertionError, match="no backward"):
        f(**dict(args, **{name: args[name].clone().requires_grad_()}))
    with forward_ad.dual_level():
        f(**args)
        dual = forward_ad.make_dual(args[name].clone(), torch.ones_like(args[name]))
        with pytest.raises(AssertionError, match="no forward-mode derivative"):
            f(**dict(args, **{name: dual}))
    with torch.no_grad():
        f(**dict(args, **{name: args[name].clone().requires_grad_()}))


@pytest.mark.gpu
@pytest.mark.parametrize("call,name", [n for n in NAMES if n[1] in ("q", "k")])
def test_transforms_do_not_pass(call, name):
    """Function transforms hand over tensors without storage: an error, and
    no result without its derivative."""
    f, args = getattr(htree_amd, call), tensors()[call]
    x = args[name]
    with pytest.raises((AssertionError, RuntimeError)):
        torch.func.jvp(lambda t: f(**dict(args, **{name: t})), (x,), (torch.ones_like(x),))
