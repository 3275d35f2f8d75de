"""GPU tests of the calls around the serving attention on streams other than
the default one, on which nothing waits for the host: a call on the wrong
stream, or with a workspace that another call has, finds the wrong values.

Everything the host has to send is on the GPU before; behind the products that
hold a stream up, an event that has not come yet when the calls are made shows
that they were made ahead."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 16


def hold_up(a, times):
    """Some milliseconds of work for the current stream, and the event behind it."""
    for _ in range(times):
        torch.mm(a[0], a[1], out=a[2])
    e = torch.cuda.Event()
    e.record()
    return e


def products():
    a = torch.randn(3, 8192, 8192, device=DEV)
    hold_up(a, 1)
    return a


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def verify(seed, rows, B, V, dtype, drawn, greedy=False):
    """Inputs (a dict of tensors, which may change) and the call."""
    g = gen(seed)
    soft = lambda: torch.softmax(4 * torch.randn(rows, V, generator=g, device=DEV), -1).to(dtype)
    t = dict(p=soft(), toks=torch.randint(V, (rows,), generator=g, device=DEV),
             starts=torch.arange(0, rows + 1, rows // B, device=DEV).int())
    if drawn:
        t["q"] = soft()
    if not greedy:
        t.update(u=torch.rand(rows, generator=g, device=DEV) * 1e-4, d=torch.rand(B, generator=g, device=DEV))
    return t, lambda t: list(htree_amd.verify_drafts(t["p"], t["toks"], t["starts"], t.get("u"), t.get("d"),
                                                     draft_probs=t.get("q")))


def unused(seed, B, width, pages):
    g = gen(seed)
    t = dict(table=torch.randint(pages, (B, width), generator=g, device=DEV).int(),
             lens=torch.randint(width * PAGE, (B,), generator=g, device=DEV).int(),
             held=torch.randint(pages, (99,), generator=g, device=DEV).int())
    return t, lambda t: list(htree_amd.unused_pages(t["table"], t["lens"], PAGE, pages, held=t["held"]))


def fork(seed, B, n, width):
    g = gen(seed)
    pages = B * width + n
    perm = torch.randperm(pages, generator=g, device=DEV).int()
    t = dict(table=perm[:B * width].view(B, width).clone(), free=perm[B * width:].clone(),
             lens=torch.randint(1, width * PAGE, (B,), generator=g, device=DEV).int(),
             source=torch.randint(B, (n,), generator=g, device=DEV).int())
    return t, lambda t: list(htree_amd.fork_requests(t["table"], t["lens"], t["source"], t["free"], PAGE, pages))


def caches(g, layers, pages):
    return {n: torch.randn(layers, pages, PAGE, 2, 64, generator=g, device=DEV).bfloat16() for n in "kv"}


def copy(seed, layers, n):
    g = gen(seed)
    perm = torch.randperm(2 * n, generator=g, device=DEV).int()
    t = dict(**caches(g, layers, 2 * n), frm=perm[:n].clone(), to=perm[n:].clone(),
             count=torch.randint(PAGE + 1, (n,), generator=g, device=DEV).int())

    def call(t):
        k, v = t["k"].clone(), t["v"].clone()
        htree_amd.copy_pages(k, v, t["frm"], t["to"], t["count"])
        return [k, v]
    return t, call


def keep(seed, layers, B):
    g = gen(seed)
    t = dict(**caches(g, layers, B), slots=torch.randperm(B * PAGE, generator=g, device=DEV),
             starts=torch.arange(0, B * PAGE + 1, PAGE, device=DEV).int(),
             path=(torch.rand(B, PAGE, generator=g, device=DEV).sort(1).values * PAGE).int().flatten().contiguous(),
             kept=torch.randint(PAGE + 1, (B,), generator=g, device=DEV).int())

    def call(t):
        k, v = t["k"].clone(), t["v"].clone()
        htree_amd.keep_drafts(k, v, t["slots"], t["starts"], t["path"], t["kept"])
        return [k, v]
    return t, call


def norm(seed, rows, grads):
    g = gen(seed)
    rand = lambda *n: torch.randn(*n, generator=g, device=DEV).bfloat16()
    t = dict(q=rand(rows, 16, 128), k=rand(rows, 2, 128), wq=rand(128), wk=rand(128), dq=rand(rows, 16, 128),
             dk=rand(rows, 2, 128))

    def call(t):
        x = [t[n].detach().requires_grad_(grads) for n in ("q", "k", "wq", "wk")]
        y = htree_amd.head_norm(*x)
        return [*(z.detach() for z in y), *(torch.autograd.grad(y, x, [t["dq"], t["dk"]]) if grads else ())]
    return t, call


CALLS = {
    "verify": lambda s: verify(s, 24, 4, 1001, torch.float32, False),
    "verify drawn": lambda s: verify(s, 24, 4, 1001, torch.float32, True),
    "verify, several blocks": lambda s: verify(s, 24, 4, 140001, torch.float32, True),
    "verify greedily": lambda s: verify(s, 24, 4, 140001, torch.bfloat16, False, True),
    "unused": lambda s: unused(s, 40, 300, 30000), "unused, large": lambda s: unused(s, 600, 900, 300000),
    "fork": lambda s: fork(s, 60, 300, 9), "copy": lambda s: copy(s, 3, 200), "keep": lambda s: keep(s, 3, 50),
    "norm": lambda s: norm(s, 3000, False), "norm with gradients": lambda s: norm(s, 3000, True)}


@pytest.mark.parametrize("name", list(CALLS))
def test_on_another_stream(name):
    """The call's inputs are those of another seed until a stream's long products
    are done: only behind those the right ones are there."""
    now, call = CALLS[name](1)
    later, _ = CALLS[name](2)
    call(now)
    want = call(later)
    assert any(not torch.equal(a, b) for a, b in zip(call(now), want))  # (the seeds differ)
    a, side = products(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        hold_up(a, 1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        done = hold_up(a, 6)
        for n in now:
            now[n].copy_(later[n])
        got = call(now)
        early = not done.query()
    torch.cuda.synchronize()
    assert early, "the host waited for the stream"
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("first", [0, 1])
def test_two_streams_at_once(first):
    """Calls of one kind that are ready on two streams at the same moment, in
    turn: each gives what it gives alone."""
    jobs = [{name: f(10 + i) for name, f in CALLS.items()} for i in range(2)]
    want = [{name: call(t) for name, (t, call) in j.items()} for j in jobs]
    a, gate, streams = products(), torch.cuda.Stream(), [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for name in CALLS:
        for s, j in zip(streams, jobs):  # (each stream's memory is there, and its kernels)
            with torch.cuda.stream(s):
                j[name][1](j[name][0])
        torch.cuda.synchronize()
        with torch.cuda.stream(gate):
            done = hold_up(a, 6)
        got = []
        for s in streams:
            s.wait_event(done)
        for _ in range(4):
            for i in (first, 1 - first):
                with torch.cuda.stream(streams[i]):
                    got.append((i, jobs[i][name][1](jobs[i][name][0])))
        early = not done.query()
        torch.cuda.synchronize()
        assert early, f"{name}: the host waited for a stream"
        for i, y in got:
            assert all(torch.equal(x, z) for x, z in zip(y, want[i][name])), (name, i)
