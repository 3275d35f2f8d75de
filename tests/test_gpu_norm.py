"""GPU tests of head_norm and its gradients against the formulas in 64 bits,
and of the gradients against differences.

Bounds, with u = 2^-24: the sum of D <= 256 squares is added up in at most 16
steps a lane and 6 between lanes, each square rounded: 23 u of it, half of
that in its root, 2 u in the reciprocal root, so r is within 14 u.  A normed
element takes two more roundings, a rotated one two more: 18 u of
|n1 c| + |n2 s|; 32 u below.  Then one rounding to the type, half a step.
A gradient's dot product has the same sums (of products of three roundings),
so r^2 mean(g x) is within 60 u of its terms' absolute sum; 128 u below.  The
weights' gradient adds up to `items` terms one after another: items u."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).tiny * torch.finfo(t).eps / 2 if t is torch.float16 else 1e-40


def turn(x, cos, sin):
    if cos is None:
        return x
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def size_of_turn(x, cos, sin):
    if cos is None:
        return x.abs()
    a, b = x.abs().chunk(2, -1)
    return torch.cat([a * cos.abs() + b * sin.abs(), b * cos.abs() + a * sin.abs()], -1)


def reference(x, w, eps, cos, sin, dy=None):
    """y and its bound; with dy also dx, dw and theirs (without the rounding to the type)."""
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    D = x.shape[-1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r * w
    out = [turn(n, cos, sin), 32 * U * size_of_turn(n, cos, sin)]
    if dy is not None:
        h = turn(dy.double(), cos, None if sin is None else -sin)
        h_abs = size_of_turn(dy.double(), cos, sin)
        g, g_abs = h * w, h_abs * w.abs()
        dx = r * (g - x * r.square() * (g * x).mean(-1, keepdim=True))
        out += [dx, 128 * U * r * (g_abs + x.abs() * r.square() * (g_abs * x.abs()).mean(-1, keepdim=True))]
        terms = h_abs * x.abs() * r
        out += [(h * x * r).flatten(0, -2).sum(0), (64 + terms[..., 0].numel()) * U * terms.flatten(0, -2).sum(0)]
    return out


def close(got, want, bar, dtype, what):
    half, least = half_step(dtype)
    bar = bar + half * (want.abs() + bar) + least
    off = (got.double() - want).abs()
    assert got.dtype is dtype and bool((off <= bar).all()), (what, float((off / bar).max()))


def data(lead, H, Hkv, D, dtype, w_dtype, rope, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = DT[dtype]
    rand = lambda *n: torch.randn(*n, generator=g, device=DEV)
    q, k = (rand(*lead, H, D) * scale).to(t), (rand(*lead, Hkv, D) * scale).to(t)
    w = [None, None] if w_dtype is None else [(1 + 0.3 * rand(D)).to(DT[w_dtype]) for _ in range(2)]
    pos = cos = sin = None
    if rope:
        cos, sin = htree_amd.rope_cache(D, 500, 10000.0, DEV)
        pos = torch.randint(500, lead, generator=g, device=DEV).to(torch.int32)
    return q, k, w, pos, cos, sin, rand(*lead, H, D).to(t), rand(*lead, Hkv, D).to(t)


def check(q, k, w, pos, cos, sin, gq, gk, eps=1e-6):
    c = s = None
    if cos is not None:
        at = pos.long()
        c, s = cos.double()[at][..., None, :], sin.double()[at][..., None, :]
    plain = htree_amd.head_norm(q, k, *w, eps=eps, positions=pos, cos=cos, sin=sin)
    leaves = [x.detach().requires_grad_() for x in (q, k)]
    ws = [None if x is None else x.detach().clone().requires_grad_() for x in w]
    out = htree_amd.head_norm(*leaves, *ws, eps=eps, positions=pos, cos=cos, sin=sin)
    grads = torch.autograd.grad(out, [x for x in leaves + ws if x is not None], (gq, gk))
    for i, (x, dy, name) in enumerate(((q, gq, "q"), (k, gk, "k"))):
        y, y_bar, dx, dx_bar, dw, dw_bar = reference(x, w[i], eps, c, s, dy)
        assert torch.equal(plain[i], out[i]) and plain[i].is_contiguous() and plain[i].shape == x.shape
        close(out[i], y, y_bar, x.dtype, name)
        close(grads[i], dx, dx_bar, x.dtype, "d" + name)
        if w[i] is not None:
            at = 2 + sum(v is not None for v in w[:i])
            close(grads[at], dw, dw_bar, w[i].dtype, "dw" + name)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("dtype,D", [("float32", 4), ("float32", 32), ("float32", 36), ("float32", 128), ("float32", 252),
                                     ("float32", 256), ("bfloat16", 8), ("bfloat16", 24), ("bfloat16", 64),
                                     ("bfloat16", 96), ("bfloat16", 128), ("bfloat16", 248), ("bfloat16", 256),
                                     ("float16", 16), ("float16", 72), ("float16", 128), ("float16", 256)])
def test_types_and_head_dims(dtype, D, rope):
    for seed, (lead, H, Hkv) in enumerate([((1,), 1, 1), ((7,), 6, 2), ((2, 19), 33, 3)]):
        check(*data(lead, H, Hkv, D, dtype, dtype if seed else "float32", rope, seed))


@pytest.mark.parametrize("rows,H,Hkv,D,dtype", [(1, 64, 8, 128, "bfloat16"), (3000, 32, 2, 128, "bfloat16"),
                                                (4097, 8, 8, 64, "float32"), (20000, 5, 1, 32, "float16"),
                                                (2049, 64, 4, 256, "bfloat16")])
def test_many_rows(rows, H, Hkv, D, dtype):
    check(*data((rows,), H, Hkv, D, dtype, None, True, 3))
    check(*data((rows,), H, Hkv, D, dtype, "float32", False, 4))


@pytest.mark.parametrize("scale,eps", [(1e-3, 1e-6), (1e-4, 1e-5), (100.0, 1e-6), (0.0, 1e-6), (1.0, 0.0), (1.0, 10.0)])
def test_sizes_and_eps(scale, eps):
    check(*data((40,), 6, 2, 64, "float32", "float32", True, 5, scale), eps=eps)


def test_large_and_uneven_values():
    q, k, w, pos, cos, sin, gq, gk = data((30,), 6, 2, 128, "bfloat16", "bfloat16", True, 6)
    q[::3] *= 1e15
    q[1::3] *= 1e-8
    k[:, :, 5] = 1000.0
    check(q, k, w, pos, cos, sin, gq, gk)


def test_views_and_other_orders():
    """A fused projection's rows, heads before tokens, unaligned and expanded
    inputs and gradients."""
    g = torch.Generator(device=DEV).manual_seed(7)
    qkv = torch.randn(2, 33, 12, 64, generator=g, device=DEV).bfloat16()
    _, _, w, pos, cos, sin, gq, gk = data((2, 33), 8, 2, 64, "bfloat16", "bfloat16", True, 7)
    check(qkv[:, :, :8], qkv[:, :, 8:10], w, pos, cos, sin, gq, gk)
    bhtd = torch.randn(2, 10, 33, 64, generator=g, device=DEV).bfloat16()
    check(bhtd[:, :8].transpose(1, 2), bhtd[:, 8:].transpose(1, 2), w, pos, cos, sin, gq.transpose(1, 2).contiguous().transpose(1, 2), gk)
    odd = torch.randn(2, 33, 10 * 64 + 3, generator=g, device=DEV).bfloat16()
    check(odd[..., 3:3 + 512].view(2, 33, 8, 64), odd[..., 3 + 512:].view(2, 33, 2, 64), w, pos, cos, sin, gq, gk)
    check(qkv[:, :1, :8].expand(2, 33, 8, 64), qkv[:, :, 8:9].expand(2, 33, 2, 64), w, pos, cos, sin,
          gq[:, :, :1].expand(2, 33, 8, 64), gk[:1, :1, :1, :1].expand(2, 33, 2, 64))


@pytest.mark.parametrize("dtype", list(DT))
def test_weights_and_tables_from_anywhere(dtype):
    """Weights and tables that begin at any element of a larger tensor."""
    q, k, w, pos, cos, sin, gq, gk = data((50,), 6, 2, 64, dtype, dtype, True, 15)
    w = [torch.cat([x[:n], x])[n:] for n, x in ((1, w[0]), (3, w[1]))]
    assert w[0].is_contiguous() and w[0].data_ptr() % 4 != 0 or dtype == "float32"
    cos, sin = torch.cat([cos.view(-1)[:1], cos.view(-1)])[1:].view_as(cos), torch.cat([sin.view(-1)[:3], sin.view(-1)])[3:].view_as(sin)
    pos = torch.cat([pos[:1], pos])[1:]
    plain = htree_amd.head_norm(q, k, *w, positions=pos, cos=cos, sin=sin)
    leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
    out = htree_amd.head_norm(*leaves, positions=pos, cos=cos, sin=sin)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    same = [x.detach().clone().requires_grad_() for x in (q, k, *w)]
    want = htree_amd.head_norm(*same, positions=pos.clone(), cos=cos.clone(), sin=sin.clone())
    for x, y in zip((*out, *plain, *grads), (*want, *want, *torch.autograd.grad(want, same, (gq, gk)))):
        assert torch.equal(x, y)


def test_rows_without_a_position_are_zero():
    q, k, w, pos, cos, sin, gq, gk = data((9,), 4, 2, 64, "float32", "float32", True, 8)
    pos[::2] = torch.tensor([-1, 500, 2 ** 31 - 1, -2 ** 31, 499], dtype=torch.int32, device=DEV)
    q[0], gq[2] = float("nan"), float("inf")  # nothing of such a row counts
    leaves = [x.requires_grad_() for x in (q, k, *w)]
    out = htree_amd.head_norm(*leaves, positions=pos, cos=cos, sin=sin)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    on = torch.tensor([1, 3, 5, 7, 8], device=DEV)
    off = torch.tensor([0, 2, 4, 6], device=DEV)
    for x in (*out, *grads[:2]):
        assert bool((x[off] == 0).all())
    leaves2 = [x.detach()[on].requires_grad_() for x in (q, k)] + leaves[2:]
    out2 = htree_amd.head_norm(*leaves2, positions=pos[on].contiguous(), cos=cos, sin=sin)
    grads2 = torch.autograd.grad(out2, leaves2, (gq[on], gk[on]))
    for x, y in zip((*out, *grads[:2]), (*out2, *grads2[:2])):
        assert torch.equal(x[on], y)
    for x, y in zip(grads[2:], grads2[2:]):
        assert bool(torch.isfinite(x).all()) and float((x - y).abs().max()) < 1e-4


def test_parts_of_the_gradient():
    """Only some inputs, or only one output, take part."""
    q, k, w, pos, cos, sin, gq, gk = data((2, 50), 6, 2, 64, "bfloat16", "bfloat16", False, 9)
    full = [x.detach().clone().requires_grad_() for x in (q, k, *w)]
    want = torch.autograd.grad(htree_amd.head_norm(*full), full, (gq, gk))
    for mask in range(1, 16):
        args = [x.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, x in enumerate((q, k, *w))]
        on = [x for x in args if x.requires_grad]
        out = htree_amd.head_norm(*args)
        for x, y in zip(torch.autograd.grad(out, on, (gq, gk)), [y for i, y in enumerate(want) if mask >> i & 1]):
            assert torch.equal(x, y)
    for i, dy in ((0, gq), (1, gk)):
        got = torch.autograd.grad(htree_amd.head_norm(*full)[i], full, dy, allow_unused=True)
        assert got[1 - i] is None and got[3 - i] is None
        assert torch.equal(got[i], want[i]) and torch.equal(got[2 + i], want[2 + i])


def test_gradient_against_differences():
    """f = sum y dy along random directions: (f(x + h v) - f(x - h v)) / 2h,
    h = 2^-7, is off by h^2/6 = 1e-5 of the third derivative, about 8 for each
    of 90 heads, so 0.007 if all had one sign, and by the roundings of y, 5760
    terms of size one times 6e-8 / h: 0.04 if all had one sign."""
    q, k, w, pos, cos, sin, gq, gk = data((15,), 4, 2, 64, "float32", "float32", True, 10)
    leaves = [x.requires_grad_() for x in (q, k, *w)]

    def f(*args):
        a, b = htree_amd.head_norm(*args, positions=pos, cos=cos, sin=sin)
        return float((a.double() * gq.double()).sum() + (b.double() * gk.double()).sum())

    out = htree_amd.head_norm(*leaves, positions=pos, cos=cos, sin=sin)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    h = 2.0 ** -7
    for i in range(4):
        v = torch.randn_like(leaves[i])
        step = lambda a: [x.detach() + a * v if j == i else x.detach() for j, x in enumerate(leaves)]
        slope = (f(*step(h)) - f(*step(-h))) / (2 * h)
        want = float((grads[i].double() * v.double()).sum())
        assert abs(slope - want) < 0.05, (i, slope, want)


def test_same_every_run():
    q, k, w, pos, cos, sin, gq, gk = data((4000,), 8, 2, 128, "bfloat16", "float32", True, 11)
    leaves = [x.requires_grad_() for x in (q, k, *w)]
    runs = []
    for _ in range(3):
        out = htree_amd.head_norm(*leaves, positions=pos, cos=cos, sin=sin)
        runs.append((*out, *torch.autograd.grad(out, leaves, (gq, gk))))
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_past_32_bits():
    """More than 2^32 elements: the last rows are those of a call of their own."""
    rows, H, D = 70000, 250, 256
    q = torch.randn(1000, H, D, device=DEV).bfloat16().repeat(rows // 1000, 1, 1)
    k, w = q[:, :1].contiguous(), torch.randn(D, device=DEV)
    assert q.numel() > 2 ** 32
    q[-7:].normal_()
    pos = torch.arange(rows, device=DEV).to(torch.int32) % 500
    cos, sin = htree_amd.rope_cache(D, 500, 10000.0, DEV)
    q.requires_grad_()
    out = htree_amd.head_norm(q, k, w, w, positions=pos, cos=cos, sin=sin)[0]
    dq, = torch.autograd.grad(out, q, out.detach())
    last = q.detach()[-7:].clone().requires_grad_()
    want = htree_amd.head_norm(last, k[-7:], w, w, positions=pos[-7:].contiguous(), cos=cos, sin=sin)[0]
    assert torch.equal(out[-7:], want)
    assert torch.equal(dq[-7:], torch.autograd.grad(want, last, want.detach())[0])


def test_empty():
    z = lambda *n: torch.zeros(n, device=DEV, requires_grad=True)
    w = z(64)
    out = htree_amd.head_norm(z(0, 4, 64), z(0, 2, 64), w, w)
    assert out[0].shape == (0, 4, 64) and out[1].shape == (0, 2, 64)
    (out[0].sum() + out[1].sum()).backward()
    assert bool((w.grad == 0).all())


def test_shared_weight_and_shared_input():
    """One tensor in two places gets the sum of both gradients."""
    q, _, w, _, _, _, gq, _ = data((60,), 4, 4, 64, "float32", "float32", False, 12)
    x, s = q.clone().requires_grad_(), w[0].clone().requires_grad_()
    out = htree_amd.head_norm(x, x, s, s)
    dx, ds = torch.autograd.grad(out, (x, s), (gq, gq))
    y, y_bar, rx, rx_bar, rs, rs_bar = reference(q, s.detach(), 1e-6, None, None, gq)
    close(dx, 2 * rx, 2 * rx_bar + 2.0 ** -23 * rx.abs(), torch.float32, "x")
    close(ds, 2 * rs, 2 * rs_bar + 2.0 ** -23 * rs.abs(), torch.float32, "w")


def test_training_with_htree_forward():
    """Norms before the tree attention, which rotates by itself: its gradients
    go on through them."""
    B, T, H, Hkv, D = 1, 300, 4, 1, 64
    q, k, w, *_ = data((B, T), H, Hkv, D, "bfloat16", "float32", False, 13)
    v = torch.randn(B, T, Hkv, D, device=DEV).bfloat16()
    leaves = [x.requires_grad_() for x in (q, k, *w)]
    nq, nk = htree_amd.head_norm(*leaves)
    out = htree_amd.htree_forward_autograd(nq, nk, v, 16, 128, 16)
    dO = torch.randn_like(out)
    grads = torch.autograd.grad(out, [nq, nk] + leaves, dO)
    want = torch.autograd.grad(htree_amd.head_norm(*leaves), leaves, grads[:2])
    for x, y in zip(grads[2:], want):
        assert bool(torch.isfinite(x).all()) and torch.equal(x, y)


def test_captured():
    """Forward and backward in a graph, replayed with new inputs."""
    q, k, w, pos, cos, sin, gq, gk = data((500,), 8, 2, 128, "bfloat16", "float32", True, 14)
    leaves = [x.requires_grad_() for x in (q, k, *w)]

    def step():
        out = htree_amd.head_norm(*leaves, positions=pos, cos=cos, sin=sin)
        return (*out, *torch.autograd.grad(out, leaves, (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(4):
        with torch.no_grad():
            for x in (*leaves, gq, gk):
                x.copy_(torch.randn(x.shape, device=DEV).to(x.dtype))
            pos.copy_(torch.randint(500, (500,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, step()))


def test_refusals():
    f = lambda *n, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)
    pos = torch.zeros(3, dtype=torch.int32, device=DEV)
    ok = dict(q=f(3, 4, 64), k=f(3, 2, 64), q_weight=f(64), k_weight=f(64))
    htree_amd.head_norm(**ok)
    rope = dict(positions=pos, cos=f(9, 32), sin=f(9, 32))
    htree_amd.head_norm(**ok, **rope)
    bad = [dict(q=f(3, 4, 64, t=torch.float64)), dict(k=f(3, 2, 32)), dict(k=f(2, 2, 64)), dict(k=f(3, 2, 64, t=torch.bfloat16)),
           dict(q=f(3, 64), k=f(3, 64)), dict(q=f(3, 4, 62), k=f(3, 2, 62), q_weight=None, k_weight=None),
           dict(q=f(3, 4, 260), k=f(3, 2, 260), q_weight=None, k_weight=None), dict(q=f(3, 0, 64)), dict(k=f(3, 0, 64)),
           dict(q_weight=f(32)), dict(q_weight=f(64, t=torch.bfloat16)), dict(q_weight=f(128)[::2]), dict(k_weight=f(64).cpu()),
           dict(q=f(3, 4, 64, t=torch.bfloat16), k=f(3, 2, 64, t=torch.bfloat16), q_weight=f(64, t=torch.bfloat16)),
           dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(positions=pos), dict(cos=f(9, 32), sin=f(9, 32)),
           dict(rope, cos=f(9, 31)), dict(rope, sin=f(8, 32)), dict(rope, positions=pos.long()), dict(rope, positions=pos[:2]),
           dict(rope, cos=f(9, 32, t=torch.bfloat16)), dict(rope, cos=f(0, 32), sin=f(0, 32)), dict(q=f(3, 4, 64).cpu()),
           dict(rope, cos=f(9, 32).requires_grad_())]
    for i, kw in enumerate(bad):
        with pytest.raises(AssertionError):
            htree_amd.head_norm(**dict(ok, **kw))
            print("not refused:", i)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(f(3, 4, 64), f(3, 4, 64))
        with pytest.raises(AssertionError, match="forward-mode"):
            htree_amd.head_norm(**dict(ok, q=d))
    x = f(3, 4, 64).normal_().requires_grad_()
    g, = torch.autograd.grad(htree_amd.head_norm(**dict(ok, q=x, q_weight=f(64) + 1))[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
