"""Values of the paged-cache entries' arguments that would give no result: refused
calls launch nothing, so they need no GPU."""
from __future__ import annotations

import pytest

from tests.test_paged_refusals_cpu import NH_E_ARG, _attention, _kv, _rows


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_attention_factor_is_finite(scale):
    assert _attention(_kv(), _rows(), scale=scale) == NH_E_ARG
    assert _attention(_kv(), _rows(n_rows=0), scale=scale) == NH_E_ARG


def test_attention_counts_its_blocks_before_any_launch():
    big = (1 << 31) - 1
    for n_seq in (1, 2):
        rows = _rows(n_seq=n_seq, n_rows=big, max_rows=big // 8)
        assert _attention(_kv(n_head_kv=256, head_dim=32), rows, n_head=2048) == NH_E_ARG
