"""Clipping of synced gradients and of parameter shards on two and three CPU ranks: every rank gets the
same norm."""
import pytest

from tests import _mp, clip_cases

pytest.importorskip("torch")


@pytest.mark.parametrize("ranks", [2, 3])
def test_clipping_on_ranks(ranks):
    res = _mp.run(ranks, clip_cases.run_clip, timeout=240)
    assert all(r == res[0] for r in res)


@pytest.mark.parametrize("ranks", [2, 3])
def test_replicated_parameters_count_once(ranks):
    res = _mp.run(ranks, clip_cases.run_replicated, timeout=240)
    assert all(r == res[0] for r in res)
