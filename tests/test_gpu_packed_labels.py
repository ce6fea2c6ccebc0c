"""A session over two views of one slot runs both."""
import numpy as np
import pytest

from hologram_amd import DTYPE_BF16, HipSession
from packed_reference import decode, encode
from test_packed_labels import COLS, ROWS, two_halves

pytestmark = pytest.mark.gpu


def test_two_views_of_one_slot(torch_cuda, backend):
    rng = np.random.default_rng(1)
    s = HipSession(backend, two_halves())
    x = encode(rng.standard_normal((2 * ROWS, COLS)), DTYPE_BF16).reshape(2 * ROWS, COLS)
    ids, values = np.array([3, 44, 499], np.int32), np.array([50.0, -1.0, 50.0], np.float32)
    want = decode(x, DTYPE_BF16).reshape(2, ROWS, COLS).copy()
    want[:, np.arange(ROWS), ids] += values
    out = s.execute([x.tobytes(), ids.tobytes(), values.tobytes()])
    for i in range(2):
        assert np.array_equal(np.frombuffer(out[i], np.int32), want[i].argmax(1))
