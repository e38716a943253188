"""Refusals of the rotating append and of the paged attention entry points, without a GPU: the C ABI
rejects bad arguments before touching the device, the torch operators reject CPU tensors."""
import ctypes as C

import pytest

cabi = pytest.importorskip("llmik_cuda.cabi")

INVALID, UNSUPPORTED, MISALIGNED = 1, 2, 3
D = C.c_void_p(256)


def attention(**kw):
    a = dict(fmt=0, q=D, stride=32 * 128, ks=None, vs=None, tables=D, ctx=D, cu=D, out=D, n=4, seqs=2, h=32, hk=8, d=128,
             blocks=10, bs=16, width=5, scale=0.1, window=0, cap=0.0, ws=D)
    a.update(kw)
    return cabi.lib().lik_attention_paged(
        a["fmt"], a["q"], a["stride"], D, D, a["ks"], a["vs"], a["tables"], a["ctx"], a["cu"], a["out"], a["n"], a["seqs"],
        a["h"], a["hk"], a["d"], a["blocks"], a["bs"], a["width"], a["scale"], 1, a["window"], a["cap"], None, None, None, 0,
        a["ws"], 1 << 30, None)


@pytest.mark.parametrize("kw,status", [
    (dict(d=64), UNSUPPORTED), (dict(fmt=2), UNSUPPORTED), (dict(fmt=9), UNSUPPORTED), (dict(h=30), INVALID),
    (dict(h=129, hk=1), UNSUPPORTED), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(cap=-1.0), INVALID),
    (dict(cap=float("nan")), INVALID), (dict(window=-1), INVALID), (dict(bs=24), INVALID), (dict(bs=0), INVALID),
    (dict(blocks=0), INVALID), (dict(blocks=1 << 28), INVALID), (dict(width=1 << 27), INVALID), (dict(n=-1), INVALID),
    (dict(n=1 << 29), INVALID), (dict(seqs=-1), INVALID), (dict(stride=32 * 128 + 4), MISALIGNED),
    (dict(stride=31 * 128), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(tables=None), INVALID),
    (dict(ctx=None), INVALID), (dict(cu=None), INVALID), (dict(fmt=1), INVALID), (dict(fmt=1, ks=D), INVALID),
    (dict(fmt=1, ks=D, vs=C.c_void_p(264)), MISALIGNED), (dict(q=C.c_void_p(264)), MISALIGNED),
    (dict(ws=C.c_void_p(272)), MISALIGNED)])
def test_attention_refuses(kw, status):
    assert attention(**kw) == status
    assert cabi.lib().lik_last_error()


def test_attention_of_no_tokens_is_a_noop():
    assert attention(n=0, q=None, out=None, cu=None, ctx=None, tables=None, seqs=0) == 0


def shared(**kw):
    a = dict(pt=D, pl=D, cu=D, tables=D, ctx=D, n=4, groups=1, pwidth=4, width=5, scale=0.1)
    a.update(kw)
    return cabi.lib().lik_attention_shared_prefix(0, D, 4096, D, D, None, None, a["pt"], a["pl"], a["cu"], a["tables"],
                                                  a["ctx"], D, a["n"], a["groups"], 32, 8, 128, 10, 16, a["pwidth"],
                                                  a["width"], a["scale"], 0.0, None, D, 1 << 30, None)


@pytest.mark.parametrize("kw", [dict(groups=0), dict(pt=None), dict(pl=None), dict(cu=None), dict(tables=None), dict(ctx=None),
                                dict(pwidth=-1), dict(pwidth=1 << 27), dict(scale=0.0), dict(n=-2)])
def test_shared_prefix_refuses(kw):
    assert shared(**kw) == INVALID


def test_workspace_size_grows_with_the_problem_and_stays_bounded():
    f = cabi.lib().lik_attention_workspace_bytes
    assert 0 < f(1, 32, 8, 0) < f(64, 32, 8, 0) <= f(100000, 32, 8, 0) < (1 << 27)
    assert f(64, 32, 8, 1) > f(64, 32, 8, 0)


def append(sections=None, **kw):
    a = dict(kf=0, vf=0, q=D, qs=4096, ks=1024, vs=1024, axes=1, freqs=64, n=4, h=32, hk=8, d=128, kc=D, kscale=None,
             vscale=None, vzero=None, blocks=10, bs=16, out=D)
    a.update(kw)
    sec = (C.c_int64 * len(sections))(*sections) if sections else None
    return cabi.lib().lik_paged_append_rope(a["kf"], a["vf"], a["q"], a["qs"], D, a["ks"], D, a["vs"], D, a["axes"], sec, D,
                                            a["freqs"], 0, D, a["out"], a["n"], a["h"], a["hk"], a["d"], a["kc"], a["kscale"],
                                            D, a["vscale"], a["vzero"], a["blocks"], a["bs"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(d=64), UNSUPPORTED), (dict(kf=2), UNSUPPORTED), (dict(vf=4), INVALID), (dict(vf=-1), INVALID),
    (dict(h=30), INVALID), (dict(freqs=0), INVALID), (dict(freqs=65), INVALID), (dict(axes=0), INVALID),
    (dict(axes=5), INVALID), (dict(axes=2), INVALID), (dict(axes=2, sections=[32, 31]), INVALID),
    (dict(axes=2, sections=[-1, 65]), INVALID), (dict(sections=[63]), INVALID), (dict(qs=4100), MISALIGNED),
    (dict(ks=-8), MISALIGNED), (dict(n=-1), INVALID), (dict(bs=0), INVALID), (dict(blocks=-1), INVALID),
    (dict(q=None), INVALID), (dict(kc=None), INVALID), (dict(kf=1), INVALID), (dict(vf=1), INVALID),
    (dict(vf=3, vscale=D), INVALID), (dict(out=C.c_void_p(264)), MISALIGNED)])
def test_append_refuses(kw, status):
    assert append(**kw) == status
    assert cabi.lib().lik_last_error()


def test_append_of_no_tokens_is_a_noop():
    assert append(n=0, q=None, out=None, kc=None) == 0


def test_torch_operators_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    import llmik_cuda as L
    q, k = torch.zeros(2, 8, 128, dtype=torch.half), torch.zeros(2, 2, 128, dtype=torch.half)
    cache = torch.zeros(4, 2, 16, 128, dtype=torch.half)
    i64, i32 = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.paged_append_rope(q, k, k, i64, torch.ones(64), i64, cache, cache)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.paged_attention(q, cache, cache, i32[None], i32[:1], i32, 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.paged_shared_prefix_attention(q, cache, cache, i32[None], i32[:1], i32, i32[:, None], i32, 0.1)
