"""LogitsProcess (129) held element by element to the roundings of that column's own rules: a bias or
a penalty that is lost, doubled or another column's shows however long the lists are."""
import numpy as np
import pytest

from hologram_amd import DTYPE_F32
from packed_reference import ALL, HALF, decode, process_logits
from test_gpu_logits import make, run

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def roundings(x, c):
    """What the f32 operations of each column may be off by: half a step of each result."""
    off, y = np.zeros(x.shape), x.copy()
    rows, cols = x.shape
    for r in range(rows):
        if c["history"] is not None:
            n = min(int(c["spans"][r, 1]), c["history"].shape[1])
            h = c["history"][r, :n].astype(np.int64)
            here = (h >= 0) & (h < cols)
            seen = np.bincount(h[here], minlength=cols) > 0
            made = np.arange(n) >= int(c["spans"][r, 0])
            times = np.bincount(h[here & made], minlength=cols)
            rep, freq, pres = (float(v) for v in c["params"][r])
            y[r, seen] = np.where(y[r] > 0, y[r] / rep, y[r] * rep)[seen]
            off[r, seen] += U * np.abs(y[r, seen])
            g = times > 0
            pen = freq * times[g] + pres
            y[r, g] -= pen
            off[r, g] += U * (np.abs(freq * times[g]) + np.abs(pen) + np.abs(y[r, g]))
        if c["ids"] is not None:
            ids, v = c["ids"][r].astype(np.int64), c["values"][r].astype(np.float64)
            here = (ids >= 0) & (ids < cols)
            many = np.bincount(ids[here], minlength=cols)
            total = np.bincount(ids[here], weights=v[here], minlength=cols)
            size = np.bincount(ids[here], weights=np.abs(v[here]), minlength=cols)
            b = many > 0
            y[r, b] += total[b]
            off[r, b] += U * ((many[b] - 1) * size[b] + np.abs(y[r, b]))
    return off


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,cols,hist,nb,mask", [
    (2, 20000, 5, 4095, False), (9, 500, 9, 4095, True), (2, 40007, 3000, 300, True), (3, 8200, 700, 1, False),
    (4, 32000, 4096, 64, True), (3, 1000, 40, 2000, False),
])
def test_every_column_by_its_own_rules(torch_cuda, backend, rows, cols, hist, nb, mask, dtype):
    c = make(np.random.default_rng(cols + nb), rows, cols, hist, nb, mask, dtype)
    x = decode(c["x"], dtype).reshape(rows, cols)
    want = process_logits(x, c["history"], c["spans"], c["params"], c["ids"], c["values"], c["mask"])
    got = decode(run(torch_cuda, backend, c, dtype), dtype).reshape(rows, cols)
    # (the errors' own products: 1.001; f32's last operation is its last rounding)
    tol = 1.001 * roundings(x, c)
    if dtype != DTYPE_F32:
        tol = tol + HALF[dtype] * (np.abs(np.where(np.isfinite(want), want, 0)) + tol) + 2.0 ** -25
    fin = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()
    if nb > 64:
        # the bound is far below a bias where a column has one
        single = (tol > 0) & fin & (tol < 2.0 ** -7 * (1 + np.abs(np.where(fin, want, 0))))
        assert single.sum() > 0.9 * (fin & (tol > 0)).sum()
