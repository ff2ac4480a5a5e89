"""Workspace sizes of the prompt and shared-prefix attention (no GPU here): a
server asks for its largest call's and makes every smaller call with it."""
import itertools

import pytest

import specdec as S

L = S.lib()
HEADS = [(8, 2, 64), (32, 8, 128), (128, 8, 128)]


def never_less(size, ranges):
    """`size` does not fall where one of its arguments grows."""
    for args in itertools.product(*ranges):
        for i, values in enumerate(ranges):
            more = [v for v in values if v > args[i]]
            if more:
                larger = args[:i] + (more[0],) + args[i + 1:]
                assert size(*larger) >= size(*args), (args, larger)


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
def test_prompt_sizes_grow_with_the_call(Hq, Hkv, hd):
    never_less(lambda B, T, mb: L.specdec_attention_prompt_workspace_bytes(B, T, Hq, Hkv, hd, mb),
               [(1, 5, 64, 1024), (1, 2, 200, 4095, 4096, 4097, 8192, 1 << 17, 1 << 23, 1 << 24),
                (1, 16, 17, 512, 1 << 20)])


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
def test_shared_prefix_sizes_grow_with_the_call(Hq, Hkv, hd):
    size = L.specdec_attention_shared_prefix_workspace_bytes
    never_less(lambda B, R, ng, mb: size(B, R, min(ng, B), Hq, Hkv, hd, mb),
               [(1, 5, 64, 128, 1024), (1, 2, 5, 21, 64), (0, 1, 3, 64), (1, 16, 17, 512, 1 << 20)])


def test_shared_prefix_sizes_stay_near_what_the_rows_need():
    """Two results a row where there are groups; without groups and with one key
    tile or two a table, none."""
    size, row = L.specdec_attention_shared_prefix_workspace_bytes, 32 * (128 + 2) * 4
    for B, R in ((128, 64), (1024, 64), (1024, 5)):
        assert 2 * B * R * row <= size(B, R, 1, 32, 8, 128, 512) <= (2 * B * R + 8192) * row + 24 * B + 1024
        assert size(B, R, 0, 32, 8, 128, 512) <= 8192 * row + 24 * B + 1024
        assert size(B, R, 0, 32, 8, 128, 16) <= 24 * B + 1024
