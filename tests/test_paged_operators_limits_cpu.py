"""Refusals of the paged operators beyond those of test_paged_operators_cpu, without a GPU."""
import ctypes as C

import pytest

cabi = pytest.importorskip("llmik_cuda.cabi")

from test_paged_operators_cpu import D, INVALID, append, attention  # noqa: E402


def at(offset):
    return C.c_void_p(D.value + offset)


@pytest.mark.parametrize("kw", [dict(scale=0.1, cap=1e-32), dict(scale=1e20, cap=1e-12)])
def test_attention_refuses_caps_that_no_score_can_be_divided_by(kw):
    assert attention(**kw) == INVALID


@pytest.mark.parametrize("step", [-1, 9, 1 << 40])
def test_the_timeout_self_test_refuses_steps_there_are_none_of(step):
    assert cabi.lib().lik_selftest_attention_timeout(step) == INVALID


# 4 tokens of 32 query and 8 KV heads: rows of 8192 and 2048 bytes
@pytest.mark.parametrize("kw", [
    dict(q=at(0), out=at(16)), dict(q=at(16), out=at(0)), dict(q=at(0), out=at(4 * 8192 - 16)),
    dict(q=at(0), stride=48 * 128, out=at(0)), dict(q=at(0), stride=48 * 128, out=at(3 * 12288 + 8192 - 16)),
    dict(q=at(4 * 8192 - 16), out=at(0)), dict(q=at(0), stride=1 << 38, out=at(1 << 40))])
def test_attention_refuses_results_over_its_queries(kw):
    assert attention(**kw) == INVALID and b"overlap" in cabi.lib().lik_last_error()


@pytest.mark.parametrize("kw", [
    dict(q=at(0), out=at(16)), dict(q=at(0), qs=48 * 128, out=at(0)), dict(q=at(0), out=at(4 * 8192 - 16)),
    dict(q=at(1 << 20), out=D), dict(q=at(1 << 20), out=at(4 * 2048 - 16)), dict(q=at(1 << 20), h=8, out=D)])
def test_append_refuses_results_over_what_it_reads(kw):
    assert append(**kw) == INVALID and b"overlap" in cabi.lib().lik_last_error()
