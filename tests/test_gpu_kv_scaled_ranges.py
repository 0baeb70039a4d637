"""The block-scaled FP8 cache on the GPU, at the ends of what its calls allow."""
import pytest
import torch

from test_gpu_kv_scaled import check_attention

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- weights of few rows
@pytest.mark.parametrize("d,hkv,g,lens,rows,window", [
    (128, 8, 4, [4000, 2500], [5, 2], 0),
    (64, 8, 16, [5000], [3], 0),
    (256, 4, 8, [3000, 40, 1500], [2, 3, 16], 0),
    (128, 8, 4, [2000] * 6, [4] * 6, 300),
])
def test_weights_where_one_cta_of_a_pair_has_no_rows(d, hkv, g, lens, rows, window):
    for _ in range(3):
        check_attention(d, hkv, g, lens, rows, window, True, smallest=window > 0)
