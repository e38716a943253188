"""`paged_append_rope` against rotation in 64 bits and `paged_append` of the rotated rows.

A rotated component is a cos - b sin: the angle's cosine and sine are fp32
(half a step, and 2 steps for sincospif and its rounded argument: 3 * 2^-24
and pi 2^-24 relative to 1), two products and their sum round once each, so it
is within 10 * 2^-24 (|a| + |b|) before the one rounding to fp16.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    import llmik_cuda
    return llmik_cuda


def rotate64(x, pos, inv, axis, interleaved):
    """x [n, heads, 128] -> rotated in 64 bits and the bound of each component before its fp16 rounding."""
    r = inv.numel()
    angle = pos[axis].double().T * inv.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x = x.double()
    y, off = x.clone(), torch.zeros_like(x)
    i = torch.arange(r, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    off[..., ia] = off[..., ib] = 10 * 2.0 ** -24 * (a.abs() + b.abs())
    return y, off


def close(got, want, off):
    assert ((got.double() - want).abs() <= off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25).all()


CASES = [
    # tokens, heads, kv heads, frequencies, sections, interleaved, block
    (1, 32, 8, 64, None, False, 16),
    (8, 32, 8, 64, None, False, 16),
    (77, 8, 2, 64, [16, 24, 24], False, 32),
    (77, 8, 2, 64, [16, 24, 24], True, 32),
    (33, 3, 1, 32, None, False, 48),
    (33, 3, 1, 32, None, True, 48),
    (50, 5, 5, 11, [3, 8], False, 16),
    (50, 5, 5, 11, [3, 8], True, 16),
    (50, 5, 5, 1, None, False, 16),
    (29, 16, 16, 8, [2, 2, 2, 2], False, 1),
    (300, 71, 1, 48, [0, 48], False, 128),
    # enough rows for several tokens per block, the last block short or full
    (3199, 40, 8, 64, [16, 24, 24], False, 64),
    (3200, 40, 8, 24, None, False, 16),
    (3201, 40, 8, 31, None, True, 48),
    (3200, 40, 8, 31, None, False, 48),
]


@pytest.mark.parametrize("fmt", ["fp16", "int8", "v_int4", "v_int4_asym", "mixed"])
@pytest.mark.parametrize("n,H,Hkv,r,sections,interleaved,bs", CASES)
def test_rotates_and_appends(L, fmt, n, H, Hkv, r, sections, interleaved, bs):
    g = torch.Generator().manual_seed(n + r)
    qkv = torch.randn(n, H + 2 * Hkv, 128, generator=g).half().cuda()
    qkv[0, -1, 3] = 50.0
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    axes = len(sections) if sections else 1
    pos = torch.randint(-5, 200000, (axes, n), generator=g).cuda()
    axis = torch.tensor([a for a, m in enumerate(sections or [r]) for _ in range(m)]).cuda()
    inv = (10000.0 ** (-torch.arange(r).double() / r)).float().cuda()
    blocks = -(-n // bs) + 2
    slots = torch.randperm(blocks * bs, generator=g)[:n]
    slots[n // 3] = -1
    slots[n // 2] = blocks * bs if n > 2 else slots[n // 2]
    slots = slots.cuda()

    def cache(kind):
        row = 64 if "int4" in kind else 128
        c = torch.full((blocks, Hkv, bs, row), 3, dtype=torch.float16 if kind == "fp16" else torch.int8, device="cuda")
        s = None if kind == "fp16" else torch.full((blocks, Hkv, bs), 9.0, dtype=torch.float16, device="cuda")
        z = s.clone() if kind == "int4_asym" else None
        return c, s, z

    kk, vk = {"fp16": ("fp16", "fp16"), "int8": ("int8", "int8"), "v_int4": ("fp16", "int4"),
              "v_int4_asym": ("int8", "int4_asym"), "mixed": ("int8", "fp16")}[fmt]
    kc, ks, _ = cache(kk)
    vc, vs, vz = cache(vk)
    got = L.paged_append_rope(q, k, v, pos if sections else pos[0], inv, slots, kc, vc, k_scale=ks, v_scale=vs,
                              v_zero=vz, sections=sections, interleaved=interleaved)
    close(got, *rotate64(q, pos, inv, axis, interleaved))
    # the caches hold what paged_append of the rotated keys and of v leaves: the rotated keys, bit for bit,
    # are what the operator itself returns for keys passed as queries
    dummy = torch.zeros(blocks, Hkv, bs, 128, dtype=torch.float16, device="cuda")
    k_rot = L.paged_append_rope(k, k, v, pos if sections else pos[0], inv, torch.full_like(slots, -1), dummy,
                                dummy.clone(), sections=sections, interleaved=interleaved)
    assert (dummy == 0).all()
    close(k_rot, *rotate64(k, pos, inv, axis, interleaved))
    kc2, ks2, _ = cache(kk)
    vc2, vs2, vz2 = cache(vk)
    L.paged_append(k_rot, slots, kc2, ks2)
    L.paged_append(v.contiguous(), slots, vc2, vs2, vz2)
    for a, b in ((kc, kc2), (ks, ks2), (vc, vc2), (vs, vs2), (vz, vz2)):
        assert (a is None and b is None) or torch.equal(a, b)


def test_no_tokens(L):
    c = torch.zeros(2, 2, 16, 128, dtype=torch.float16, device="cuda")
    x = torch.zeros(0, 4, 128, dtype=torch.float16, device="cuda")
    i = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert L.paged_append_rope(x, x[:, :2], x[:, :2], i, torch.ones(64, device="cuda"), i, c, c.clone()).shape == (0, 4, 128)


def test_captured_append_replays_with_other_positions(L):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(4, 8, 128, generator=g).half().cuda(), torch.randn(4, 2, 128, generator=g).half().cuda()
    inv = (10000.0 ** (-torch.arange(64).double() / 64)).float().cuda()
    pos, slots = torch.arange(4).cuda(), torch.arange(4).cuda()
    cache = torch.zeros(4, 2, 16, 128, dtype=torch.float16, device="cuda")
    other = cache.clone()
    L.paged_append_rope(q, k, k, pos, inv, slots, cache, other)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = L.paged_append_rope(q, k, k, pos, inv, slots, cache, other)
    pos.copy_(torch.tensor([9, 100, 5, 77777]))
    slots.copy_(torch.tensor([63, -1, 20, 31]))
    gr.replay()
    torch.cuda.synchronize()
    c2, o2 = torch.zeros_like(cache), torch.zeros_like(other)
    want = L.paged_append_rope(q, k, k, pos, inv, slots, c2, o2)
    assert torch.equal(out, want)
    live = slots[slots >= 0]
    assert torch.equal(cache[live // 16, :, live % 16], c2[live // 16, :, live % 16])


@pytest.mark.parametrize("n,r,interleaved", [(5, 64, False), (5, 31, True), (5, 31, False), (3200, 64, False),
                                             (3200, 24, False), (3200, 31, True), (3200, 31, False)])
def test_queries_rotated_in_place(L, n, r, interleaved):
    import ctypes

    from llmik_cuda import cabi
    lib = cabi.lib()
    g = torch.Generator().manual_seed(n + r)
    q, k = torch.randn(n, 40, 128, generator=g).half().cuda(), torch.randn(n, 8, 128, generator=g).half().cuda()
    pos, slots = torch.randint(0, 100000, (n,), generator=g).cuda(), torch.arange(n).cuda()
    inv = (10000.0 ** (-torch.arange(r).double() / r)).float().cuda()
    blocks = -(-n // 16)
    caches = [torch.zeros(blocks, 8, 16, 128, dtype=torch.float16, device="cuda") for _ in range(4)]
    want = L.paged_append_rope(q, k, k, pos, inv, slots, caches[0], caches[1], interleaved=interleaved)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    torch.cuda.synchronize()
    st = lib.lik_paged_append_rope(0, 0, p(q), 40 * 128, p(k), 8 * 128, p(k), 8 * 128, p(pos), 1, None, p(inv), r,
                                   int(interleaved), p(slots), p(q), n, 40, 8, 128, p(caches[2]), None, p(caches[3]),
                                   None, None, blocks, 16, None)
    torch.cuda.synchronize()
    assert st == 0
    assert torch.equal(q, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
