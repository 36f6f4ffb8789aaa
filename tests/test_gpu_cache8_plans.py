"""Attention over a cache in 8 bits where its launch is shaped by what the caller
expects and the lengths turn out otherwise."""
import pytest

from cache8test import Step8
from cachetest import DTYPES
from test_gpu_cache import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("page_size,window", [(16, 0), (24, 0), (16, 1200)])
def test_shared_entries_past_the_expected_length(dev, dtype, page_size, window):
    """As captured calls whose sequences have grown: the expected length ends inside the
    shared entries, and so do some sequences; a chunk among the single tokens."""
    lens = [1620] + [1501 + 7 * i for i in range(60)] + [1100, 640, 500, 1900]
    s = Step8(dtype, [1] * 64 + [130], lens, 4, 4, 128, seed=page_size, page_size=page_size, shared=1500, window=window)
    for max_len in (600, 1499, 1):
        check_attention(s, max_len=max_len, max_new=130)
    s = Step8(dtype, [1] * 64, lens[:64], 4, 4, 128, seed=page_size + 1, page_size=page_size, shared=1500, window=window)
    for max_len in (600, 1101):
        check_attention(s, max_len=max_len, max_new=1)
