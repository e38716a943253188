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


# ---------------------------------------------------------------- small weights

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("nq", [1, 20, 64])
def test_many_keys_far_below_the_largest_weight(L, kv, nq):
    """One key 2^25.5 above 32767 others, which carry the whole value: they must not be lost. Sequences enough for
    every unit's keys to pass one CTA (all on the same pages)."""
    ctx, bs, seqs = 32768, 128, 300 if nq < 64 else 150
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, kv, ctx // bs, 1, bs)
    for x in "kv":
        pool.exact[x].zero_()
    if kv == "int8":
        pool.s_all["k"].fill_(0.25)
        pool.s_all["v"].fill_(2.0 ** -6)
    pool.exact["v"][:] = 1.0 if kv == "fp16" else 64
    table = [pool.free[-1 - i] for i in range(ctx // bs)]
    pool.exact["v"][table[0], :, 0] = 0
    pool.exact["k"][table[0], :, 0, 0] = 25.0 if kv == "fp16" else 100
    table = pool.give([ctx])
    q = torch.zeros(seqs * nq, 4, 128, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0                                        # 8 * 25 * SCALE = 17.68 = 25.5 ln 2
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table.expand(seqs, -1).contiguous(), i32([ctx] * seqs),
                            i32([nq * i for i in range(seqs + 1)]), SCALE, **pool.args())
    p = torch.arange(ctx - nq, ctx, device="cuda")[:, None]
    seen = torch.arange(ctx, device="cuda")[None] <= p
    ref, tol = reference(q[:nq], pool.rows("k", table[0], ctx), pool.rows("v", table[0], ctx), seen, None)
    tol = tol - ctx * 2.0 ** -25 + ctx * 2.0 ** (-32 if kv == "fp16" else -31)    # max |v| is 1
    assert (tol < 0.1 * ref).all()
    check(got.view(seqs, nq, 4, 128), ref[None], tol[None])


@pytest.mark.parametrize("nq", [1, 20, 64])
def test_a_large_v_scale_leaves_the_others_their_digits(L, nq):
    """INT8: a hardly weighted row with a scale 2^21 times the others'. Alike weights: an element is off by 2^-32
    times 127 times the power of two above the largest scale, besides the rounding of each weight."""
    ctx, bs = 300, 16
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, "int8", 40, 1, bs)
    pool.exact["k"].zero_()
    pool.s_all["k"].fill_(0.5)
    pool.exact["v"].copy_(torch.randint(60, 128, pool.exact["v"].shape, generator=g, dtype=torch.int8))
    pool.s_all["v"].fill_(2.0 ** -15.5)
    first = pool.free[-1]
    pool.exact["k"][first, :, 3, 0] = -100                 # 8 * -50 * SCALE: a weight of 2^-51
    pool.s_all["v"][first, :, 3] = 60.0
    table = pool.give([ctx])
    q = torch.zeros(nq, 4, 128, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([ctx]), i32([0, nq]), SCALE, causal=False,
                            **pool.args())
    seen = torch.ones(nq, ctx, dtype=torch.bool, device="cuda")
    v = pool.rows("v", table[0], ctx)
    ref, tol = reference(q, pool.rows("k", table[0], ctx), v, seen, None)
    tol = tol - ctx * 2.0 ** -25 * v.abs().amax() + 2.0 ** -32 * 127 * 64
    assert (tol < 0.01 * ref).all()
    check(got, ref, tol)
