"""Calls without sequences or rows (no GPU here): an empty tensor's pointer is
null, and such a call does nothing."""
import pytest

import specdec as S

L = S.lib()


@pytest.mark.parametrize("B,T", [(0, 0), (0, 5), (3, 0)])
def test_prompt(B, T):
    assert L.specdec_attention_prompt(None, 512, None, 4, 2, 64, None, 4, None, None, B, T, 8, None, 512, None, 0,
                                      None) == S.OK


def test_shared_prefix():
    assert L.specdec_attention_shared_prefix(None, None, 4, 2, 64, None, 4, None, None, None, None, 0, 0, 5, 8, None,
                                             None, 0, None) == S.OK


@pytest.mark.parametrize("B,T", [(-1, 0), (0, -1), (1025, 0), (0, (1 << 24) + 1)])
def test_sizes_are_checked_all_the_same(B, T):
    assert L.specdec_attention_prompt(None, 512, None, 4, 2, 64, None, 4, None, None, B, T, 8, None, 512, None, 0,
                                      None) == S.EINVAL
