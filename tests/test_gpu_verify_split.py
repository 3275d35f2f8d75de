"""GPU tests of verify_drafts where two, three or four blocks share a request's
sums (few requests over a large vocabulary), where such a request's mass runs
out, and of drafts drawn without replacement."""
import numpy as np
import pytest
import torch

from htree_amd import _native as N
from tests.test_gpu_verify import case, check

pytestmark = pytest.mark.gpu
V = 65_600  # drawn: 131200 entries of p and q a row


@pytest.mark.parametrize("B,most,dtype,parts", [(64, 3, "bfloat16", 4), (70, 2, "bfloat16", 3), (85, 2, "float16", 3),
                                                (86, 2, "float32", 2), (100, 2, "bfloat16", 2), (128, 2, "float16", 2)])
@pytest.mark.parametrize("drawn", [False, True])
def test_blocks_that_share_a_request(B, most, dtype, parts, drawn):
    """The walk's test at each number of blocks, requests without rows among them."""
    v = V if drawn else 2 * V
    g = np.random.default_rng(B)
    new = [most, most, 0] + list(g.integers(0, most + 1, B - 3))
    n = N.ctypes.c_int64()
    N.check(N.lib().htree_verify_drafts_workspace_bytes(0, B, sum(new), v, drawn, 0, n), "")
    assert n.value == B * (24 + parts * 16 * 8)  # so many blocks' sums, of 16 waves each
    kept, _, _ = check(*case(new, v, dtype, False, drawn, B))
    assert kept.sum() > sum(x > 0 for x in new)  # drafts were accepted


@pytest.mark.parametrize("B", [3, 70, 100])
def test_mass_that_runs_out(B):
    """Targets that are wholly at their rejected drafts' tokens, or without any
    mass, or without a number; draws of any value."""
    v = 131_072
    starts = [0] + [2 * i for i in range(1, B)] + [2 * B - 2]  # the last request has no rows
    p = torch.zeros(2 * B - 2, v, dtype=torch.bfloat16)
    tokens = np.tile([0, 7], B - 1)
    p[::8, 7] = 0.5                            # rejected: nothing is left but itself
    p[2::8, 7], p[2::8, v - 1] = 0.25, 0.5      # rejected: the last one is left
    p[4::8, v // 2] = float("nan")              # no mass
    p[6::8, [3, 40_000, 100_000]] = 0.25        # not at the draft
    u = np.full(2 * B - 2, 0.75)
    wild = [0.5, np.nan, -1.0, 0.0, 1.0, np.inf, 0.99999994, 1e-40, 2.0]
    for shift in range(3):
        draws = [wild[(i + shift) % len(wild)] for i in range(B)]
        kept, _, nxt = check(p, None, tokens, starts, None, u, draws)
        assert kept.tolist() == [1] * (B - 1) + [0]
        assert nxt[0] == 7 and nxt[-1] == -1 and (B < 5 or (nxt[2] == -1 and nxt[1] == v - 1))
    q = torch.zeros_like(p)
    q[:, 7] = 1.0
    p[::8, 7], q[::8, 7] = 0.5, 2.0            # drawn: a target that its drafter's multiple covers
    check(p, q, tokens, starts, None, u, [wild[i % len(wild)] for i in range(B)])


def test_drawn_without_replacement():
    """Verified as drafts chosen in any way: the token after the first one has
    the target's probabilities (counts within 5 of their standard deviations)."""
    g = np.random.default_rng(5)
    count, v, n = 4096, 6, 4
    p0, q0 = np.array([0.4, 0.05, 0.25, 0.1, 0.15, 0.05]), np.array([0.1, 0.3, 0.05, 0.3, 0.05, 0.2])
    tokens = np.concatenate([[0, *g.choice(v, size=3, replace=False, p=q0)] for _ in range(count)])
    starts, parents = np.arange(count + 1) * n, np.tile([-1, 0, 0, 0], count)
    p = torch.as_tensor(np.tile(p0, (count * n, 1))).float()
    kept, path, nxt = check(p, None, tokens, starts, parents, g.random(count * n, dtype=np.float32),
                            g.random(count, dtype=np.float32))
    then = np.where(kept > 1, tokens[starts[:-1] + path[starts[:-1] + np.minimum(kept - 1, n - 1)]], nxt)
    counts = np.bincount(then, minlength=v)
    assert np.all(np.abs(counts - count * p0) <= 5 * np.sqrt(count * p0 * (1 - p0))), counts


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("new,v,dtype", [([6] * 9, 32000, "float32"), ([24] * 5, 7, "bfloat16"), ([2, 9, 1, 30], 8192, "float16"),
                                         ([64], 16385, "bfloat16"), ([200, 1], 50, "float16"), ([7, 8] * 3, 150001, "bfloat16")])
def test_drafts_are_accepted(new, v, dtype, tree, drawn):
    """Numbers of zero accept what has mass: every request keeps drafts, and one
    whole chain is kept."""
    p, q, tokens, starts, parents, u, d = case(new, v, dtype, tree, drawn, 1)
    kept, _, _ = check(p, q, tokens, starts, parents, u * 0, d)
    assert all(k > 1 for k, n in zip(kept, new) if n > 1)
    if not tree:
        assert kept.tolist() == new
