"""Attention of several query tokens per sequence over a paged cache
(`paged_attention`) and shared-prefix decode (`paged_shared_prefix_attention`)
against a plain 64-bit implementation.

The bound of a row, with A = sum p |v| / sum p, B = the largest sum |q_i k_i|
times the softmax scale, n its keys:
  * the weights (times V's scale, in an INT8 cache) are rounded to fp16 once (half
    a step, 2^-11): 2^-11 A, and below 2^-14 by 2^-25 at most, at a largest weight of
    1 or more: n 2^-25 max|v|;
  * the result is rounded to fp16: 2^-11 |out|;
  * a score is an fp32 sum of 128 exact products in any order (128 2^-24 B),
    scaled, capped and biased by a few fp32 operations (8 2^-23 |score| and the
    2^-20 the hardware exponentials leave in tanh, times the cap): a score off
    by d moves weights and their sum by e^d - 1 each. INT8 codes are exact in the
    products, their scales one fp32 operation (among the 8).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)
H11 = 2.0 ** -11


@pytest.fixture(scope="module")
def L():
    import llmik_cuda
    yield llmik_cuda
    llmik_cuda.check_device_errors()


def rand(g, *shape, spread=1.0):
    return (torch.randn(*shape, generator=g) * spread).half().cuda()


class Pool:
    """A paged cache with scrambled pages; rows nobody owns are NaN (fp16) or have NaN scales."""

    def __init__(self, g, kv, blocks, kv_heads, bs):
        self.kv, self.bs = kv, bs
        self.free = torch.randperm(blocks, generator=g).tolist()
        shape = (blocks, kv_heads, bs, 128)
        self.cache, self.scale, self.exact = {}, {"k": None, "v": None}, {}
        for x in "kv":
            if kv == "fp16":
                self.exact[x] = rand(g, *shape)
                self.cache[x] = torch.full(shape, float("nan"), dtype=torch.float16, device="cuda")
            else:
                self.exact[x] = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).cuda()
                self.cache[x] = torch.full(shape, 99, dtype=torch.int8, device="cuda")
                self.scale[x] = torch.full(shape[:3], float("nan"), dtype=torch.float16, device="cuda")
        self.s_all = {x: ((torch.rand(shape[:3], generator=g) + 0.5) * 0.02).half().cuda() for x in "kv"}

    def give(self, lens, width=None, fill=-77):
        """Tables for sequences of these lengths; entries past a sequence's end are invalid on purpose."""
        width = max([1] + [-(-n // self.bs) for n in lens]) if width is None else width
        table = torch.full((len(lens), width), fill, dtype=torch.int32)
        for b, n in enumerate(lens):
            for i in range(-(-n // self.bs)):
                table[b, i] = p = self.free.pop()
                m = min(self.bs, n - i * self.bs)
                for x in "kv":
                    self.cache[x][p, :, :m] = self.exact[x][p, :, :m]
                    if self.scale[x] is not None:
                        self.scale[x][p, :, :m] = self.s_all[x][p, :, :m]
        return table.cuda()

    def rows(self, x, table_row, n):
        """[kv_heads, n, 128] in 64 bits."""
        idx = table_row[:-(-n // self.bs)].long()
        r = self.exact[x][idx].double()
        if self.kv != "fp16":
            r = r * self.s_all[x][idx].double()[..., None]
        return r.transpose(0, 1).reshape(r.shape[1], -1, 128)[:, :n]

    def args(self):
        return dict(k_scale=self.scale["k"], v_scale=self.scale["v"])


def reference(q, k, v, seen, dist, cap=0.0, slopes=None):
    """q [n, H, 128], k and v [Hkv, m, 128], seen [n, m], dist [n, m]: output and bound, 64 bits."""
    n, H, _ = q.shape
    G = H // k.shape[0]
    q, kk, vv = q.double().transpose(0, 1), k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = q @ kk.transpose(1, 2) * SCALE
    B = ((q.abs() @ kk.abs().transpose(1, 2)) * SCALE).masked_fill(~seen, 0).amax(-1, keepdim=True)
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * dist.double()
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True).clamp(min=1e-300)
    out, A = e @ vv / total, e @ vv.abs() / total
    near = torch.where(e > 1e-9, s.abs(), torch.zeros_like(s)).amax(-1, keepdim=True)
    # the bias and the capped score may cancel in `s`: count the bias on its own
    if slopes is not None:
        near = near + torch.where(e > 1e-9, slopes.double()[:, None, None] * dist.double(), torch.zeros_like(s)).amax(
            -1, keepdim=True)
    d = 128 * 2.0 ** -24 * B + 8 * 2.0 ** -23 * near + cap * 2.0 ** -20
    tol = A * (H11 + 2 * torch.expm1(d)) + H11 * out.abs() + kk.shape[1] * 2.0 ** -25 * vv.abs().amax() + 1e-7
    return out.transpose(0, 1), tol.transpose(0, 1)


def check(out, ref, tol):
    out = out.double()
    assert torch.isfinite(out).all()
    bad = (out - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((out - ref).abs() / tol).max().item():.2f} x bound"


def run_case(L, kv, H, Hkv, nq, ctx, bs, causal=True, cap=0.0, window=0, alibi=False, prefix=None, first=None, lead=0,
             pad=0, spread=1.0, seed=0, out=None, q_wide=0):
    g = torch.Generator().manual_seed(seed + 17 * len(nq) + sum(nq))
    pool = Pool(g, kv, sum(-(-c // bs) for c in ctx) + 2, Hkv, bs)
    table = pool.give(ctx)
    n = lead + sum(nq) + pad
    q = rand(g, n, H + q_wide, 128, spread=spread)[:, :H]
    cu = torch.tensor([lead] + [lead + sum(nq[:i + 1]) for i in range(len(nq))], dtype=torch.int32)
    slopes = (2.0 ** -torch.linspace(1, 8, H)).cuda() if alibi else None
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    fk = None
    if first is not None:
        fk = torch.zeros(n, dtype=torch.int32)
        for b, f in enumerate(first):
            fk[int(cu[b]):int(cu[b + 1])] = torch.tensor(f, dtype=torch.int32)
        fk = fk.cuda()
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32(ctx), cu.cuda(), SCALE, causal=causal,
                            softcap=cap, window=window, alibi_slopes=slopes,
                            prefix_lens=None if prefix is None else i32(prefix), first_keys=fk, out=out, **pool.args())
    for b, (m, c) in enumerate(zip(nq, ctx)):
        if m == 0:
            continue
        lo = int(cu[b])
        p = torch.arange(c - m, c, device="cuda")[:, None]
        j = torch.arange(c, device="cuda")[None]
        seen = torch.ones(m, c, dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= p
        if window:
            seen &= j > p - window
        if prefix is not None:
            seen |= j < prefix[b]
        if fk is not None:
            seen &= j >= fk[lo:lo + m, None]
        if c == 0:
            assert (got[lo:lo + m] == 0).all()
            continue
        ref, tol = reference(q[lo:lo + m], pool.rows("k", table[b], c), pool.rows("v", table[b], c), seen, (p - j).abs(),
                             cap, slopes)
        check(got[lo:lo + m], ref, tol)
        empty = ~seen.any(-1)
        assert (got[lo:lo + m][empty] == 0).all()
    return got, cu


KV = ["fp16", "int8"]


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("bs", [16, 48, 256])
def test_single_tokens_of_every_length(L, kv, bs):
    run_case(L, kv, 32, 8, [1] * 9, [1, 2, 15, 16, 17, 127, 128, 129, 1000], bs)


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("H,Hkv", [(8, 8), (4, 2), (6, 2), (5, 1), (14, 2), (16, 2), (32, 1), (33, 1), (64, 1),
                                   (65, 1), (128, 1)])
def test_head_groups(L, kv, H, Hkv):
    run_case(L, kv, H, Hkv, [1, 3, 40, 130], [200, 3, 333, 150], 16, seed=H)


@pytest.mark.parametrize("kv", KV)
def test_query_counts_around_the_tile_shapes(L, kv):
    nq = [7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129]
    run_case(L, kv, 4, 1, nq, [n + 150 for n in nq], 32)
    run_case(L, kv, 4, 1, nq, nq, 32, seed=1)


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("opts", [
    dict(window=1), dict(window=100), dict(window=128), dict(window=100000), dict(causal=False),
    dict(causal=False, window=77), dict(cap=30.0, spread=5.0), dict(cap=0.5, spread=5.0), dict(alibi=True),
    dict(alibi=True, causal=False), dict(prefix=[0, 300, 129, 5, 1]), dict(prefix=[400, 10, 900, 0, 1], window=40),
    dict(prefix=[400, 10, 900, 0, 1], window=40, cap=20.0, alibi=True, spread=3.0)])
def test_masks_and_score_changes(L, kv, opts):
    run_case(L, kv, 8, 2, [200, 1, 333, 20, 1], [200, 300, 900, 517, 1], 64, **opts)


@pytest.mark.parametrize("kv", KV)
def test_documents(L, kv):
    """Rows see their document only; a first key behind the query leaves the row empty."""
    a = [0] * 50 + [50] * 130 + [180] * 20
    b = [100] * 10 + [101] * 80 + [777] * 10
    run_case(L, kv, 8, 2, [200, 100], [200, 400], 16, first=[a, b])
    run_case(L, kv, 8, 2, [200, 100], [200, 400], 16, first=[a, b], prefix=[60, 390], window=30, seed=3)


@pytest.mark.parametrize("kv", KV)
def test_rows_that_see_nothing_and_empty_sequences(L, kv):
    """More queries than positions, no positions, no queries."""
    run_case(L, kv, 8, 2, [10, 0, 5, 300, 0, 1], [4, 50, 0, 100, 0, 0], 16)


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("nq,ctx", [(1, 300), (1, 30000), (3, 500), (20, 500), (20, 9000), (64, 700), (300, 5000)])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_a_query_that_is_not_finite_is_its_own_rows_matter(L, kv, nq, ctx, what):
    H, Hkv, bad_head = 8, 2, 5
    g = torch.Generator().manual_seed(nq + ctx)
    pool = Pool(g, kv, -(-ctx // 64) + 1, Hkv, 64)
    table = pool.give([ctx])
    q = rand(g, nq, H, 128)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    run = lambda x: L.paged_attention(x, pool.cache["k"], pool.cache["v"], table, i32([ctx]), i32([0, nq]), SCALE,  # noqa: E731
                                      **pool.args())
    dirty = q.clone()
    dirty[nq // 2, bad_head, 7] = what
    got = run(dirty)
    assert torch.isnan(got[nq // 2, bad_head]).all()
    p = torch.arange(ctx - nq, ctx, device="cuda")[:, None]
    seen = torch.arange(ctx, device="cuda")[None] <= p
    ref, tol = reference(q, pool.rows("k", table[0], ctx), pool.rows("v", table[0], ctx), seen, None)
    others = torch.ones(nq, H, dtype=torch.bool, device="cuda")
    others[nq // 2, bad_head] = False
    check(got[others], ref[others], tol[others])


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("nq", [1, 20, 64])
def test_distances_stay_exact_far_out(L, kv, nq):
    """Past 2^24 positions a position is no fp32 number; the distances that count are."""
    ctx, bs, width = (1 << 24) + 9 * 128 + 3, 128, (1 << 17) + 10
    g = torch.Generator().manual_seed(nq)
    pool = Pool(g, kv, 12, 1, bs)
    near = pool.give([10 * bs - 125])[0]                  # the last ten pages hold the last 1155 positions
    assert (ctx - 1) // bs - 9 == width - 10
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, width - 10:] = near
    m = 9 * bs + 3
    q = rand(g, nq, 2, 128)
    slopes = torch.tensor([0.5, 0.03], device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, i32([ctx]), i32([0, nq]), SCALE, window=900,
                            alibi_slopes=slopes, **pool.args())
    p = torch.arange(m - nq, m, device="cuda")[:, None]
    j = torch.arange(m, device="cuda")[None]
    ref, tol = reference(q, pool.rows("k", near, m), pool.rows("v", near, m), (j <= p) & (j > p - 900), (p - j).abs(),
                         slopes=slopes)
    check(got, ref, tol)


@pytest.mark.parametrize("kv", KV)
def test_rows_of_no_sequence(L, kv):
    got, cu = run_case(L, kv, 8, 2, [5, 70], [50, 70], 16, lead=3, pad=4)
    assert (got[:3] == 0).all() and (got[-4:] == 0).all()
    out = torch.full((3 + 75 + 4, 8, 128), 7.0, dtype=torch.float16, device="cuda")
    got, cu = run_case(L, kv, 8, 2, [5, 70], [50, 70], 16, lead=3, pad=4, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[:3] == 7).all() and (out[-4:] == 7).all()


def test_no_sequences_and_no_tokens(L):
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = torch.zeros(1, 2, 16, 128, dtype=torch.float16, device="cuda")
    q = torch.ones(3, 4, 128, dtype=torch.float16, device="cuda")
    t, c = z[:0].view(0, 1), z[:0]
    assert (L.paged_attention(q, cache, cache, t, c, z, SCALE) == 0).all()
    assert L.paged_attention(q[:0], cache, cache, t, c, z, SCALE).shape == (0, 4, 128)
    # an empty table: no positions at all
    assert (L.paged_attention(q, cache, cache, z.new_zeros(1, 0), z.new_tensor([9]), z.new_tensor([0, 3]), SCALE) == 0).all()


@pytest.mark.parametrize("kv", KV)
def test_queries_from_a_fused_projection(L, kv):
    run_case(L, kv, 8, 2, [3, 100], [40, 300], 32, q_wide=4)


@pytest.mark.parametrize("kv", KV)
def test_growing_scores_raise_the_maximum(L, kv):
    """Keys whose scores climb along the sequence: every tile rescales."""
    g = torch.Generator().manual_seed(5)
    pool = Pool(g, kv, 40, 1, 16)
    ramp = torch.arange(600, device="cuda").float()
    table_lens = [600]
    if kv == "fp16":
        pool.exact["k"].zero_()
    else:
        pool.exact["k"].zero_()
        pool.s_all["k"].fill_(1.0)
    order = pool.free[::-1]
    for i in range(38):
        m = ramp[i * 16:(i + 1) * 16]
        pool.exact["k"][order[i], :, :len(m), 0] = (m / 8).to(pool.exact["k"].dtype)
    table = pool.give(table_lens)
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    q[..., 0] = torch.tensor([1.0, 20.0, -20.0], dtype=torch.float16, device="cuda")[:, None]
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, torch.tensor([600], dtype=torch.int32, device="cuda"),
                            cu, SCALE, causal=False, **pool.args())
    seen = torch.ones(3, 600, dtype=torch.bool, device="cuda")
    ref, tol = reference(q, pool.rows("k", table[0], 600), pool.rows("v", table[0], 600), seen, seen.long())
    check(got, ref, tol)


def test_repeats_are_bit_equal_and_streams_do_not_mix(L):
    g = torch.Generator().manual_seed(2)
    pool = Pool(g, "fp16", 600, 2, 16)
    lens = [700, 30, 2000, 513]
    table = pool.give(lens)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 300, 301, 1000, 1001], dtype=torch.int32, device="cuda")
    q = rand(g, 1001, 8, 128)
    call = lambda x: L.paged_attention(x, pool.cache["k"], pool.cache["v"], table, ctx, cu, SCALE)  # noqa: E731
    want = [call(q), call(-q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(q if i == 0 else -q))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_captured_calls_replay_with_other_lengths(L):
    """Lengths, offsets and tables are read at replay; two graphs of one stream do not share state."""
    g = torch.Generator().manual_seed(3)
    pool = Pool(g, "fp16", 300, 2, 16)
    table = pool.give([1000, 1000, 1000])
    q = rand(g, 200, 8, 128)
    ctx = torch.tensor([10, 10, 10], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    call = lambda x: L.paged_attention(x, pool.cache["k"], pool.cache["v"], table, ctx, cu, SCALE)  # noqa: E731
    call(q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (q, -q):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(x))
        graphs.append(gr)
    for lens, cus in (([1000, 17, 600], [0, 100, 101, 180]), ([5, 1000, 999], [0, 5, 150, 200])):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(torch.tensor(cus, dtype=torch.int32))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], call(q)) and torch.equal(outs[1], call(-q))


def test_offsets_past_32_bits(L):
    """Pages whose bytes lie past 2^32."""
    g = torch.Generator().manual_seed(4)
    blocks, bs, hk = 70000, 32, 8                                   # 4.6 GB each
    cache = {x: torch.zeros(blocks, hk, bs, 128, dtype=torch.float16, device="cuda") for x in "kv"}
    table = torch.tensor([[69999, 3, 69000, 35000]], dtype=torch.int32, device="cuda")
    for x in "kv":
        cache[x][table[0].long()] = rand(g, 4, hk, bs, 128)
    q = rand(g, 3, 32, 128)
    ctx, cu = torch.tensor([120], dtype=torch.int32).cuda(), torch.tensor([0, 3], dtype=torch.int32).cuda()
    got = L.paged_attention(q, cache["k"], cache["v"], table, ctx, cu, SCALE)
    k, v = (cache[x][table[0].long()].double().transpose(0, 1).reshape(hk, -1, 128)[:, :120] for x in "kv")
    p, j = torch.arange(117, 120, device="cuda")[:, None], torch.arange(120, device="cuda")[None]
    check(got, *reference(q, k, v, j <= p, p - j))


@pytest.mark.parametrize("kv", KV)
def test_bad_table_entries_are_reported_and_read_as_zeros(L, kv):
    g = torch.Generator().manual_seed(6)
    pool = Pool(g, kv, 40, 2, 16)
    table = pool.give([200, 150])
    for bad in (-1, 40, 2 ** 31 - 1):
        t = table.clone()
        t[0, 5] = bad
        q = rand(g, 2, 8, 128)
        ctx = torch.tensor([200, 150], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        got = L.paged_attention(q, pool.cache["k"], pool.cache["v"], t, ctx, cu, SCALE, **pool.args())
        with pytest.raises(RuntimeError, match="out of range"):
            L.check_device_errors()
        L.check_device_errors()
        seen = torch.ones(1, 200, dtype=torch.bool, device="cuda")
        k, v = pool.rows("k", table[0], 200), pool.rows("v", table[0], 200)
        k[:, 80:96], v[:, 80:96] = 0, 0
        check(got[:1], *reference(q[:1], k, v, seen, seen.long()))
        check(got[1:], *reference(q[1:], pool.rows("k", table[1], 150), pool.rows("v", table[1], 150), seen[:, :150],
                                  seen[:, :150].long()))


def test_an_error_on_another_stream_is_reported(L):
    g = torch.Generator().manual_seed(5)
    pool = Pool(g, "fp16", 8, 1, 16)
    table = pool.give([100])
    table[0, 2] = 1 << 20
    q = rand(g, 1, 4, 128)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ctx, cu = i32([100]), i32([0, 1])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, ctx, cu, SCALE)
    with pytest.raises(RuntimeError):
        L.check_device_errors()
    L.check_device_errors()


def test_offsets_that_do_not_ascend_stay_in_bounds(L):
    """Token offsets and lengths out of range are clamped: no access outside the tensors, other rows unharmed."""
    g = torch.Generator().manual_seed(7)
    pool = Pool(g, "fp16", 40, 2, 16)
    table = pool.give([200, 150])
    q = rand(g, 20, 8, 128)
    for cu in ([0, 50, 20], [5, 3, 20], [-9, 10, 4000], [0, 0, 0]):
        L.paged_attention(q, pool.cache["k"], pool.cache["v"], table, torch.tensor([200, -3], dtype=torch.int32).cuda(),
                          torch.tensor(cu, dtype=torch.int32).cuda(), SCALE)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- shared prefixes

def shared_case(L, kv, H, Hkv, sizes, prefix, own, bs, cap=0.0, alibi=False, spread=1.0, lead=0, seed=0):
    g = torch.Generator().manual_seed(seed + sum(prefix) + sum(own))
    n = len(own)
    pool = Pool(g, kv, sum(-(-c // bs) for c in prefix + own) + 2, Hkv, bs)
    pt, t = pool.give(prefix), pool.give(own)
    q = rand(g, n, H, 128, spread=spread)
    cu = torch.tensor([lead] + [lead + sum(sizes[:i + 1]) for i in range(len(sizes))], dtype=torch.int32)
    slopes = (2.0 ** -torch.linspace(1, 8, H)).cuda() if alibi else None
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = L.paged_shared_prefix_attention(q, pool.cache["k"], pool.cache["v"], pt, i32(prefix), cu.cuda(), t, i32(own),
                                          SCALE, softcap=cap, alibi_slopes=slopes, **pool.args())
    for b in range(n):
        grp = [i for i in range(len(sizes)) if int(cu[i]) <= b < int(cu[i + 1])]
        rows = {}
        for x in "kv":
            parts = [pool.rows(x, pt[grp[0]], prefix[grp[0]])] if grp else []
            rows[x] = torch.cat(parts + [pool.rows(x, t[b], own[b])], dim=1)
        m = rows["k"].shape[1]
        if m == 0:
            assert (got[b] == 0).all()
            continue
        seen = torch.ones(1, m, dtype=torch.bool, device="cuda")
        dist = (m - 1 - torch.arange(m, device="cuda"))[None]
        check(got[b:b + 1], *reference(q[b:b + 1], rows["k"], rows["v"], seen, dist, cap, slopes))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("H,Hkv", [(8, 2), (3, 3), (16, 1), (7, 1)])
def test_shared_prefix(L, kv, H, Hkv):
    shared_case(L, kv, H, Hkv, [5], [300], [1, 0, 17, 128, 400], 16, seed=H)


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("opts", [dict(cap=20.0, spread=4.0), dict(alibi=True), dict(cap=5.0, alibi=True, spread=4.0)])
def test_shared_prefix_score_changes(L, kv, opts):
    shared_case(L, kv, 8, 2, [2, 3], [200, 77], [30, 1, 150, 0, 9], 32, **opts)


@pytest.mark.parametrize("kv", KV)
def test_shared_prefix_groups(L, kv):
    """Groups without requests or without a prefix, requests of no group, requests without any key."""
    shared_case(L, kv, 8, 2, [3, 0, 2, 2], [500, 64, 0, 130], [5, 0, 9, 0, 33, 2, 0, 4, 0], 16, lead=1)


@pytest.mark.parametrize("kv", KV)
def test_shared_prefix_many_requests(L, kv):
    """More query rows than one unit holds, and a prefix split over the whole GPU."""
    shared_case(L, kv, 16, 2, [70], [2500], [(i * 37) % 200 for i in range(70)], 64)


def test_shared_prefix_equals_attention_over_joined_tables(L):
    """A prefix of whole pages: the same keys through `paged_attention`, within both results' rounding."""
    g = torch.Generator().manual_seed(9)
    pool = Pool(g, "fp16", 200, 2, 32)
    prefix, own = 640, [10, 333, 64, 1]
    pt, t = pool.give([prefix]), pool.give(own)
    q = rand(g, 4, 8, 128)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    a = L.paged_shared_prefix_attention(q, pool.cache["k"], pool.cache["v"], pt, i32([prefix]), i32([0, 4]), t, i32(own),
                                        SCALE)
    joined = torch.cat([pt.expand(4, -1), t], dim=1).contiguous()
    b = L.paged_attention(q, pool.cache["k"], pool.cache["v"], joined, i32([prefix + n for n in own]), i32(range(5)), SCALE)
    k = pool.exact["v"].abs().max().item()
    assert ((a.float() - b.float()).abs() <= 2 * (2 * H11 * k)).all()


def test_shared_prefix_without_own_pages(L):
    """Own tables of no columns: every request has its group's prefix alone."""
    g = torch.Generator().manual_seed(8)
    pool = Pool(g, "fp16", 20, 2, 16)
    pt = pool.give([200, 31])
    q = rand(g, 5, 8, 128)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    run = lambda own, lens: L.paged_shared_prefix_attention(  # noqa: E731
        q, pool.cache["k"], pool.cache["v"], pt, i32([200, 31]), i32([0, 3, 5]), own, i32(lens), SCALE)
    none = torch.empty(5, 0, dtype=torch.int32, device="cuda")
    want = run(torch.zeros(5, 1, dtype=torch.int32, device="cuda"), [0] * 5)
    assert torch.isfinite(want).all() and want.abs().sum() > 0
    assert torch.equal(run(none, [0] * 5), want)
    assert torch.equal(run(none, [7] * 5)[:3].isfinite(), want[:3].isfinite())   # lengths are cut to the tables


# ---------------------------------------------------------------- a serving step

def test_append_prompt_and_decode_together(L):
    """Two prompts in chunks, then single tokens: rotate + append, attend, with the cache the operators filled
    themselves; against attention over separately rotated keys."""
    g = torch.Generator().manual_seed(11)
    H, Hkv, bs = 8, 2, 16
    chunks = [[40, 7], [100, 3], [1, 1], [1, 1]]
    lens = [sum(c[i] for c in chunks) for i in range(2)]
    pages = torch.randperm(40, generator=g)[:2 * 20].view(2, 20).int().cuda()
    cache = {x: torch.full((40, Hkv, bs, 128), float("nan"), dtype=torch.float16, device="cuda") for x in "kv"}
    inv = (10000.0 ** (-torch.arange(64).double() / 64)).float().cuda()
    done, keys, values = [0, 0], [[], []], [[], []]
    for c in chunks:
        n = sum(c)
        qkv = rand(g, n, H + 2 * Hkv, 128)
        pos = torch.cat([torch.arange(done[i], done[i] + c[i]) for i in range(2)]).cuda()
        seq = torch.cat([torch.full((c[i],), i) for i in range(2)]).cuda()
        slots = pages[seq, pos // bs].long() * bs + pos % bs
        q = L.paged_append_rope(qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], pos, inv, slots, cache["k"], cache["v"])
        turn = torch.polar(torch.ones(1, 64, dtype=torch.float64, device="cuda"), pos[:, None].double() * inv.double())
        x = qkv.double()
        z = torch.complex(x[..., :64], x[..., 64:]) * turn[:, None]
        rot = torch.cat([z.real, z.imag], -1).half()                    # both round the 64-bit (fp32) product
        done = [done[i] + c[i] for i in range(2)]
        cu = torch.tensor([0, c[0], n], dtype=torch.int32, device="cuda")
        ctx = torch.tensor(done, dtype=torch.int32, device="cuda")
        got = L.paged_attention(q, cache["k"], cache["v"], pages, ctx, cu, SCALE)
        # a rotated component is off by 3 fp32 roundings before its own: at most one fp16 step apart
        assert ((q.double() - rot[:, :H].double()).abs() <= 2 * H11 * rot[:, :H].double().abs() + 1e-6).all()
        for i in range(2):
            lo, hi = int(cu[i]), int(cu[i + 1])
            at = torch.arange(done[i], device="cuda")
            k = cache["k"][pages[i, at // bs].long(), :, at % bs]
            v = cache["v"][pages[i, at // bs].long(), :, at % bs]
            keys[i].append(rot[lo:hi, H:H + Hkv])
            values[i].append(qkv[lo:hi, H + Hkv:])
            want = torch.cat(keys[i])
            assert ((k.double() - want.double()).abs() <= 2 * H11 * want.double().abs() + 1e-6).all()
            assert torch.equal(v, torch.cat(values[i]))
            p, j = torch.arange(done[i] - c[i], done[i], device="cuda")[:, None], at[None]
            check(got[lo:hi], *reference(q[lo:hi], k.double().transpose(0, 1), v.double().transpose(0, 1), j <= p,
                                         p - j))
    assert done == lens
    # the decode operator that was there reads the same cache
    dec = L.paged_decode_attention(q, cache["k"], cache["v"], pages, ctx, SCALE, max(lens))
    assert ((dec.float() - got.float()).abs() <= 2e-3 + 1e-2 * got.float().abs()).all()
