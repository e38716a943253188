"""Refusals of the paged operators beyond those of test_paged_operators_cpu, without a GPU."""
import pytest

cabi = pytest.importorskip("llmik_cuda.cabi")

from test_paged_operators_cpu import INVALID, attention  # noqa: E402


@pytest.mark.parametrize("kw", [dict(scale=0.1, cap=1e-32), dict(scale=1e20, cap=1e-12)])
def test_attention_refuses_caps_that_no_score_can_be_divided_by(kw):
    assert attention(**kw) == INVALID


@pytest.mark.parametrize("step", [-1, 9, 1 << 40])
def test_the_timeout_self_test_refuses_steps_there_are_none_of(step):
    assert cabi.lib().lik_selftest_attention_timeout(step) == INVALID
