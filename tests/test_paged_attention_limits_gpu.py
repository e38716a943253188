"""Edges of `paged_attention` and `paged_shared_prefix_attention`: lengths past the tables, weights far below the
largest one, V scales far apart, loose caps, scales of any sign, offsets and prefixes out of range, errors of replayed
calls. Bounds as in test_paged_attention_gpu, where one term is sharper: the largest weight of a row is held as
2^7 or more in fp16, so what lies below fp16's normal range loses 2^-25 at most of it, 2^-32 relative to that weight
(INT8: weights times V's scale over a power of two that is up to twice the largest scale, so 2^-31).
"""
import math

import pytest
import torch

from test_paged_attention_gpu import H11, KV, SCALE, Pool, check, rand, reference

pytestmark = pytest.mark.gpu
INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def L():
    import llmik_cuda
    yield llmik_cuda
    llmik_cuda.check_device_errors()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- lengths past the tables

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("n", [3, 20, 70])
def test_a_length_past_its_table_is_cut_for_the_distances_too(L, kv, n):
    """A request's own length is cut to its table; the prefix's distances count the cut length."""
    g = torch.Generator().manual_seed(n)
    pool = Pool(g, kv, 2 * n + 30, 2, 16)
    pt = pool.give([300])
    said = [[40, 7, INT_MAX, 33][b % 4] for b in range(n)]
    own = [min(m, 32) for m in said]
    t = pool.give(own, width=2)
    q = rand(g, n, 8, 128)
    slopes = (2.0 ** -torch.linspace(1, 6, 8)).cuda()
    got = L.paged_shared_prefix_attention(q, pool.cache["k"], pool.cache["v"], pt, i32([300]), i32([0, n]), t, i32(said),
                                          SCALE, alibi_slopes=slopes, **pool.args())
    for b in range(n):
        rows = {x: torch.cat([pool.rows(x, pt[0], 300), pool.rows(x, t[b], own[b])], dim=1) for x in "kv"}
        m = 300 + own[b]
        seen = torch.ones(1, m, dtype=torch.bool, device="cuda")
        dist = (m - 1 - torch.arange(m, device="cuda"))[None]
        check(got[b:b + 1], *reference(q[b:b + 1], rows["k"], rows["v"], seen, dist, 0.0, slopes))


@pytest.mark.parametrize("alibi", [False, True])
def test_lengths_without_own_pages_count_nothing(L, alibi):
    g = torch.Generator().manual_seed(8)
    pool = Pool(g, "fp16", 20, 2, 16)
    pt = pool.give([200, 31])
    q = rand(g, 5, 8, 128)
    slopes = (2.0 ** -torch.linspace(1, 6, 8)).cuda() if alibi else None
    run = lambda own, lens: L.paged_shared_prefix_attention(  # noqa: E731
        q, pool.cache["k"], pool.cache["v"], pt, i32([200, 31]), i32([0, 3, 5]), own, i32(lens), SCALE, alibi_slopes=slopes)
    want = run(torch.zeros(5, 1, dtype=torch.int32, device="cuda"), [0] * 5)
    assert torch.isfinite(want).all() and want.abs().sum() > 0
    assert torch.equal(run(torch.empty(5, 0, dtype=torch.int32, device="cuda"), [7, 0, INT_MAX, -3, 1]), want)
