"""What a later row of a packed batch holds, finite values too, leaves the rows before it as they
were, bit for bit."""
import numpy as np
import pytest

from packed_reference import ALL, decode, encode
from test_gpu_packed_batch import packed_case, run_packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128, 96, 256, 72])
@pytest.mark.parametrize("first", [9, 75])
def test_larger_scores_of_later_rows(torch_cuda, backend, dtype, D, first):
    """K and Q of the tokens from `first` on 50 times as large: they share their 32 packed rows and
    their 64-key tile with tokens before."""
    rng = np.random.default_rng(D + first)
    H, Hkv, rows = 8, 2, [150, 21]
    qkv, tokens, width = packed_case(rng, rows, H, Hkv, D, dtype)
    clean = run_packed(torch_cuda, backend, qkv, rows, H, Hkv, D, dtype, 0)
    x = decode(qkv, dtype).reshape(tokens, width).copy()
    x[first:150, :(H + Hkv) * D] *= 50.0
    got = run_packed(torch_cuda, backend, encode(x, dtype).reshape(tokens, width), rows, H, Hkv, D, dtype, 0)
    assert np.array_equal(got[:first], clean[:first])
    assert np.array_equal(got[150:], clean[150:])
    assert np.isfinite(decode(got, dtype)).all()
