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


# ---------------------------------------------------------------- loose and tight caps

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e29])
@pytest.mark.parametrize("nq", [1, 20, 64])
@pytest.mark.parametrize("far", [False, True])
def test_loose_caps_keep_the_score(L, kv, cap, nq, far):
    """Scores of single products (exact in fp32), so that a capped score is off by its own fp32 roundings: some ten of
    half a step (2^-24) and the polynomial's 2^-23.7, less than 8 * 2^-23 |score|. `far`: among them keys whose scores
    lie at twice the cap below zero, where they have no weight."""
    ctx, bs, q0 = 700, 16, 512.0
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, kv, 50, 1, bs)
    c = 8.0 + torch.randint(0, 9, pool.exact["k"].shape[:3], generator=g).float() / 2      # scores of 5.7 to 8.5
    off = (torch.rand(c.shape, generator=g) < 0.03) if far and cap < 1e20 else torch.zeros(c.shape, dtype=torch.bool)
    down = -2 * cap / (q0 * SCALE) if cap < 1e20 else 0.0
    pool.exact["k"].zero_()
    if kv == "fp16":
        pool.exact["k"][..., 0] = torch.where(off, torch.full_like(c, down), c / 64).half().cuda()
    else:
        pool.exact["k"][..., 0] = torch.where(off, torch.full_like(c, -127.0), c * 8).to(torch.int8).cuda()
        pool.s_all["k"][:] = torch.where(off, torch.full_like(c, -down / 127), torch.full_like(c, 2.0 ** -9)).half().cuda()
    table = pool.give([ctx])
    q = torch.zeros(nq, 4, 128, dtype=torch.float16, device="cuda")
    q[..., 0] = q0
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([ctx]), i32([0, nq]), SCALE, softcap=cap,
                            causal=False, **pool.args())
    k, v = pool.rows("k", table[0], ctx), pool.rows("v", table[0], ctx)
    s = q0 * k[0, :, 0] * SCALE
    s = cap * torch.tanh(s / cap)
    w = torch.exp(s - s.max())
    d = 8 * 2.0 ** -23 * s[w > 1e-9].abs().max()
    ref, A = (w @ v[0]) / w.sum(), (w @ v[0].abs()) / w.sum()
    tol = A * (H11 + 2 * torch.expm1(d)) + H11 * ref.abs() + ctx * 2.0 ** -31 * v.abs().max() + 1e-7
    check(got, ref.expand(nq, 4, 128), tol.expand(nq, 4, 128))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("cap", [1e-7, 1e-25])
@pytest.mark.parametrize("nq", [1, 20, 64])
def test_tight_caps(L, kv, cap, nq):
    """Every key weighs the same, scores of zero among them (the first sequence's)."""
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, kv, 40, 2, 16)
    table = pool.give([300, 200])
    q = rand(g, 2 * nq, 8, 128)
    q[:nq] = 0
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([300, 200]), i32([0, nq, 2 * nq]), SCALE,
                            softcap=cap, **pool.args())
    for b, m in enumerate([300, 200]):
        p = torch.arange(m - nq, m, device="cuda")[:, None]
        ref, tol = reference(q[b * nq:(b + 1) * nq], pool.rows("k", table[b], m), pool.rows("v", table[b], m),
                             torch.arange(m, device="cuda")[None] <= p, None, cap)
        check(got[b * nq:(b + 1) * nq], ref, tol)


# ---------------------------------------------------------------- scales of any sign, and none

@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("nq,ctx", [(1, 300), (3, 40), (20, 500), (64, 700), (300, 900)])
def test_scales_of_either_sign(L, nq, ctx, cap):
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, "int8", -(-ctx // 16) + 1, 2, 16)
    for x in "kv":
        s = pool.s_all[x]
        s *= torch.where(torch.rand(s.shape, generator=g) < 0.5, -1.0, 1.0).half().cuda()
        s[torch.rand(s.shape, generator=g).cuda() < 0.05] = 0.0
    table = pool.give([ctx])
    q = rand(g, nq, 8, 128)
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([ctx]), i32([0, nq]), SCALE, softcap=cap,
                            window=max(ctx // 3, 1), **pool.args())
    p = torch.arange(ctx - nq, ctx, device="cuda")[:, None]
    j = torch.arange(ctx, device="cuda")[None]
    check(got, *reference(q, pool.rows("k", table[0], ctx), pool.rows("v", table[0], ctx),
                          (j <= p) & (j > p - max(ctx // 3, 1)), None, cap))


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("nq,ctx", [(1, 300), (1, 30000), (20, 500), (64, 700), (300, 900)])
def test_a_scale_that_is_not_a_number_reaches_the_rows_that_see_it(L, side, nq, ctx, cap):
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, "int8", 2 * (-(-ctx // 64)) + 1, 2, 64)
    pool.exact["v"][pool.exact["v"] == 0] = 1
    bad, good = pool.give([ctx]), pool.give([ctx])
    pool.scale[side][bad[0, 0], 1, 5] = math.nan           # a key that every row of the first sequence sees
    q = rand(g, 2 * nq, 8, 128)
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], torch.cat([bad, good]), i32([ctx, ctx]), i32([0, nq, 2 * nq]),
                            SCALE, softcap=cap, **pool.args())
    assert torch.isnan(got[:nq, 4:]).all()
    assert torch.isfinite(got[:nq, :4]).all() and torch.isfinite(got[nq:]).all()


# ---------------------------------------------------------------- prefixes out of range

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("nq", [1, 20, 64])
def test_prefixes_below_zero_show_nothing(L, kv, nq):
    g = torch.Generator().manual_seed(nq)
    ctx = 300
    pool = Pool(g, kv, 80, 2, 16)
    table = pool.give([ctx] * 3)
    q = rand(g, 3 * nq, 8, 128)
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([ctx] * 3), i32([0, nq, 2 * nq, 3 * nq]), SCALE,
                            window=100, prefix_lens=i32([-INT_MAX - 1, -INT_MAX, -5]), **pool.args())
    p = torch.arange(ctx - nq, ctx, device="cuda")[:, None]
    j = torch.arange(ctx, device="cuda")[None]
    for b in range(3):
        check(got[b * nq:(b + 1) * nq], *reference(q[b * nq:(b + 1) * nq], pool.rows("k", table[b], ctx),
                                                   pool.rows("v", table[b], ctx), (j <= p) & (j > p - 100), None))


# ---------------------------------------------------------------- offsets out of range

def test_offsets_out_of_range_leave_other_memory_alone(L):
    """Offsets are cut to the tokens: rows of sequences that hold together are right, rows without positions zero,
    rows of no sequence and the memory around the result as they were."""
    g = torch.Generator().manual_seed(7)
    pool = Pool(g, "fp16", 40, 2, 16)
    table = pool.give([200, 150])
    q = rand(g, 20, 8, 128)
    k, v = pool.rows("k", table[0], 200), pool.rows("v", table[0], 200)
    # offsets, rows of sequence 0 (200 positions), rows of sequence 1 (none), the others untouched
    for cu, s0, s1 in (([0, 50, 20], (0, 20), (0, 0)), ([5, 3, 20], (0, 0), (3, 20)), ([-9, 10, 4000], (0, 10), (10, 20)),
                       ([0, 0, 0], (0, 0), (0, 0)), ([7, 7, 9], (0, 0), (7, 9))):
        buf = torch.full((60, 8, 128), 7.0, dtype=torch.float16, device="cuda")
        out = buf[20:40]
        L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([200, -3]), i32(cu), SCALE, out=out)
        assert (buf[:20] == 7).all() and (buf[40:] == 7).all()
        lo, hi = s0
        if hi > lo:
            p = torch.arange(200 - (hi - lo), 200, device="cuda")[:, None]
            check(out[lo:hi], *reference(q[lo:hi], k, v, torch.arange(200, device="cuda")[None] <= p, None))
        assert (out[s1[0]:s1[1]] == 0).all()
        rest = torch.ones(20, dtype=torch.bool, device="cuda")
        rest[lo:hi] = False
        rest[s1[0]:s1[1]] = False
        assert (out[rest] == 7).all()


# ---------------------------------------------------------------- results in the queries' place

@pytest.mark.parametrize("kv", KV)
def test_results_may_take_the_place_of_their_queries(L, kv):
    nq, ctx = [1, 300, 20, 2, 70], [5000, 900, 4000, 2, 100]
    g = torch.Generator().manual_seed(1)
    pool = Pool(g, kv, sum(-(-c // 32) for c in ctx) + 1, 2, 32)
    table = pool.give(ctx)
    q = rand(g, sum(nq), 8, 128)
    cu = i32([sum(nq[:i]) for i in range(len(nq) + 1)])
    call = lambda x, out: L.paged_attention(x, pool.cache["k"], pool.cache["v"], table, i32(ctx), cu, SCALE, out=out,  # noqa: E731
                                            **pool.args())
    want = call(q, None)
    place = q.clone()
    assert torch.equal(call(place, place), want)
    buf = torch.cat([q, q])
    with pytest.raises(RuntimeError, match="overlap"):
        call(buf[:len(q)], buf[1:len(q) + 1])


# ---------------------------------------------------------------- a wait that runs out

SHAPES = {"wide": ([300], [900]), "paired": ([20], [9000]), "thin": ([1, 1, 1], [300, 20000, 5]),
          "mixed": ([1, 40, 300, 2], [700, 40, 2000, 130])}
STEPS = ([("fp16", i, "mixed") for i in range(1, 8)] + [("int8", i, "mixed") for i in range(1, 9)] +
         [("fp16", 3, "thin"), ("int8", 8, "thin"), ("fp16", 5, "wide"), ("int8", 2, "paired")])


@pytest.mark.parametrize("kv,step,shape", STEPS)
def test_a_wait_that_runs_out_is_reported_and_over(L, kv, step, shape):
    """One step of every block is never seen completed: the call returns, memory around the result and later calls
    are untouched."""
    from llmik_cuda import cabi
    nq, ctx = SHAPES[shape]
    g = torch.Generator().manual_seed(step)
    pool = Pool(g, kv, sum(-(-c // 32) for c in ctx) + 1, 2, 32)
    table = pool.give(ctx)
    n = sum(nq)
    q = rand(g, n, 8, 128)
    cu = i32([sum(nq[:i]) for i in range(len(nq) + 1)])
    buf = torch.full((n + 20, 8, 128), 7.0, dtype=torch.float16, device="cuda")
    call = lambda out=None: L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32(ctx), cu, SCALE, out=out,  # noqa: E731
                                              **pool.args())
    want = call()
    L.check_device_errors()
    cabi.call("lik_selftest_attention_timeout", step)
    call(buf[10:-10])
    with pytest.raises(RuntimeError, match="wait expired"):
        L.check_device_errors()
    assert (buf[:10] == 7).all() and (buf[-10:] == 7).all()
    assert torch.equal(call(), want)
    L.check_device_errors()


@pytest.mark.parametrize("kv,step", [("fp16", 3), ("fp16", 7), ("int8", 5)])
def test_a_wait_that_runs_out_over_a_shared_prefix(L, kv, step):
    from llmik_cuda import cabi
    g = torch.Generator().manual_seed(step)
    pool = Pool(g, kv, 60, 2, 32)
    pt, own = pool.give([700]), [1, 0, 40, 3, 100]
    t = pool.give(own)
    q = rand(g, 5, 8, 128)
    call = lambda: L.paged_shared_prefix_attention(q, pool.cache["k"], pool.cache["v"], pt, i32([700]), i32([0, 5]), t,  # noqa: E731
                                                   i32(own), SCALE, **pool.args())
    want = call()
    cabi.call("lik_selftest_attention_timeout", step)
    call()
    with pytest.raises(RuntimeError, match="wait expired"):
        L.check_device_errors()
    assert torch.equal(call(), want)
    L.check_device_errors()


# ---------------------------------------------------------------- errors

def test_an_error_of_a_replay_on_a_new_stream_is_reported(L):
    """A captured call's bad page is met by a replay on a stream that no eager call used, still running at the check."""
    g = torch.Generator().manual_seed(5)
    pool = Pool(g, "fp16", 8, 1, 16)
    table = pool.give([100])
    q = rand(g, 1, 4, 128)
    ctx, cu = i32([100]), i32([0, 1])
    call = lambda: L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, ctx, cu, SCALE)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    table[0, 2] = 1 << 20
    torch.cuda.synchronize()
    L.check_device_errors()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(200_000_000)                     # about a tenth of a second of work ahead of the replay
        gr.replay()
    with pytest.raises(RuntimeError, match="out of range"):
        L.check_device_errors()
    L.check_device_errors()
    table[0, 2] = table[0, 1]
    gr.replay()
    torch.cuda.synchronize()
    L.check_device_errors()
    assert torch.isfinite(out).all() and not torch.equal(out, want)


def test_a_destroyed_stream_is_not_asked(L):
    import ctypes
    rt = ctypes.CDLL("libcudart.so.12")
    g = torch.Generator().manual_seed(6)
    pool = Pool(g, "fp16", 8, 1, 16)
    table = pool.give([100])
    q = rand(g, 1, 4, 128)
    out = torch.empty_like(q)
    call = lambda: L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([100]), i32([0, 1]), SCALE, out=out)  # noqa: E731
    call()
    want = out.clone()
    handle = ctypes.c_void_p()
    assert rt.cudaStreamCreate(ctypes.byref(handle)) == 0
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
        call()
    torch.cuda.synchronize()
    assert rt.cudaStreamDestroy(handle) == 0
    L.check_device_errors()
    assert torch.equal(out, want)
