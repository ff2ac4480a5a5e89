"""Few rows under tables so wide that the pages are cut into ranges, with pages
enough for a second wave of them: pieces of 1, 4, 8 and 16 rows."""
import pytest

import test_gpu_accumulate_attention as A
import test_gpu_window_attention as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,rows,tokens", [((8, 8, 64), 1, 1900), ((32, 8, 64), 1, 1900), ((64, 8, 64), 1, 11900),
                                               ((32, 8, 64), 2, 11900), ((32, 8, 64), 4, 11900)])
def test_window(cuda_device, heads, rows, tokens):
    s = W.make([(rows, tokens - 11 * i) for i in range(64)], *heads, 1 << 20, 0, seed=rows, wide=1100, gone=False)
    ws = W.call(s)
    W.verify(s)
    del ws


@pytest.mark.parametrize("heads,rows,tokens", [((32, 8, 64), 1, 1900), ((64, 8, 64), 1, 1900), ((32, 8, 64), 4, 1900)])
def test_weights(cuda_device, heads, rows, tokens):
    s = A.make([(rows, tokens - 11 * i) for i in range(64)], *heads, seed=rows, wide=1100)
    ws = A.call(s)
    A.verify(s)
    del ws
