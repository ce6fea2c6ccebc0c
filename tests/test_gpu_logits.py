"""LogitsProcess (129) on the device against 64 bits: an element that no rule names keeps its bits,
any other is within the operations' roundings."""
import numpy as np
import pytest

from conftest import from_dev, to_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, NO_BUFFER, BufferRef, DeviceWorkspace,
                          KernelCall, LogitsProcessCall)
from packed_reference import ALL, HALF, decode, encode, process_logits

pytestmark = pytest.mark.gpu


def make(rng, rows, cols, hist, nb, mask, dtype):
    c = dict(x=encode(rng.standard_normal((rows, cols)) * 4, dtype).reshape(rows, cols), history=None,
             spans=None, params=None, ids=None, values=None, mask=None)
    if hist:
        h = np.minimum(rng.integers(-1, cols + 2, (rows, hist)), rng.integers(0, cols + 2, (rows, hist)))
        h[:, ::3] = h[:, :1]
        n = rng.integers(0, hist + 1, rows)
        n[0] = hist
        c["history"] = h.astype(np.int32)
        c["spans"] = np.stack([(n * rng.random(rows)).astype(int), n], 1).astype(np.uint32)
        c["params"] = rng.uniform([1.0, -0.5, -0.5], [1.8, 1.0, 1.0], (rows, 3)).astype(np.float32)
    if nb:
        c["ids"] = rng.integers(-1, cols + 1, (rows, nb)).astype(np.int32)
        c["values"] = (rng.standard_normal((rows, nb)) * 3).astype(np.float32)
    if mask:
        c["mask"] = rng.integers(0, 2**32, (rows, -(-cols // 32)), dtype=np.uint32)
    return c


def run(torch, backend, c, dtype, offset=0):
    """offset: elements between a slot's start and the logits (and the result)."""
    rows, cols = c["x"].shape
    es = c["x"].itemsize
    ws, refs = DeviceWorkspace(), []
    shifted = np.concatenate([np.zeros(offset, c["x"].dtype), c["x"].reshape(-1)])
    for a in (shifted, c["history"], c["spans"], c["params"], c["ids"], c["values"], c["mask"]):
        if a is None:
            refs.append(NO_BUFFER)
            continue
        ws.bind(len(refs), to_dev(torch, a))
        refs.append(BufferRef(len(refs), offset * es if len(refs) == 0 else 0))
    out = torch.full((shifted.nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
    ws.bind(7, out)
    backend.dispatch(KernelCall.LogitsProcess(LogitsProcessCall(
        *refs, BufferRef(7, offset * es), rows, cols, 0 if c["history"] is None else c["history"].shape[1],
        0 if c["ids"] is None else c["ids"].shape[1], dtype)), ws)
    backend.synchronize()
    return from_dev(out, c["x"].dtype)[offset:].reshape(rows, cols)


def check(got, c, dtype):
    x = decode(c["x"], dtype).reshape(c["x"].shape)
    want = process_logits(x, c["history"], c["spans"], c["params"], c["ids"], c["values"], c["mask"])
    same = (want == x) | (np.isnan(want) & np.isnan(x))
    touched = np.zeros(x.shape, bool)
    for r in range(x.shape[0]):
        for name in ("history", "ids"):
            if c[name] is not None:
                v = c[name][r]
                v = v[:int(c["spans"][r, 1])] if name == "history" else v
                touched[r, v[(v >= 0) & (v < x.shape[1])]] = True
    allowed = np.isneginf(want) | ~touched
    assert np.array_equal(got[same & ~touched], c["x"][same & ~touched])      # bits kept
    g = decode(got, dtype).reshape(x.shape)
    assert np.array_equal(np.isneginf(g[allowed]), np.isneginf(want[allowed]))
    # f32 steps: the quotient, the penalty's two and the sum of up to n biases; magnitudes at most
    # |x| * 2 + penalty + biases. Then one rounding to the dtype.
    steps = 6 + (0 if c["ids"] is None else c["ids"].shape[1])
    mag = 2 * np.abs(x) + 1
    if c["params"] is not None:
        mag = mag + np.abs(c["params"][:, 1:2]) * c["history"].shape[1] + np.abs(c["params"][:, 2:])
    if c["values"] is not None:
        mag = mag + np.abs(c["values"]).sum(1, keepdims=True)
    fin = np.isfinite(want) & touched
    tol = (steps * 2.0 ** -24 * mag) + HALF[dtype] * np.abs(np.where(fin, want, 0)) + 2.0 ** -25
    assert (np.abs(g[fin] - want[fin]) <= tol[fin]).all()


CASES = [  # rows, cols, history, biases, mask
    (1, 1, 1, 1, True), (3, 33, 10, 3, True), (2, 1000, 0, 0, True), (2, 1000, 0, 5, False),
    (4, 5001, 700, 0, False), (5, 8191, 64, 40, True), (2, 40007, 3000, 300, True),
    (70, 4097, 33, 2, False), (1, 32000, 1024, 8, False), (2, 20000, 5, 4095, False), (3, 777, 0, 0, False),
    (260, 130, 20, 4, True), (130, 16400, 50, 3, True), (260, 500, 9, 4095, False),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,cols,hist,nb,mask", CASES)
def test_logits_parity(torch_cuda, backend, rows, cols, hist, nb, mask, dtype):
    rng = np.random.default_rng(rows * cols + hist)
    c = make(rng, rows, cols, hist, nb, mask, dtype)
    for offset in (0, 1, 5):
        check(run(torch_cuda, backend, c, dtype, offset), c, dtype)


@pytest.mark.parametrize("dtype", ALL)
def test_rules_on_odd_values(torch_cuda, backend, dtype):
    """NaN and infinities in the logits, a mask that leaves a row empty, a row without history, one
    token said every time, the same bias id many times, a NaN bias, parameters of 0 and infinity."""
    rng = np.random.default_rng(8)
    c = make(rng, 6, 500, 64, 9, True, dtype)
    x = decode(c["x"], dtype).reshape(6, 500).copy()
    x[:, 0], x[:, 1], x[:, 2], x[:, 3], x[:, 4] = np.nan, np.inf, -np.inf, 0.0, -0.0
    c["x"] = encode(x, dtype).reshape(6, 500)
    c["mask"][:, 0] |= 0x1F
    c["mask"][1] = 0
    c["mask"][2] = 0xFFFFFFFF
    c["history"][0, :8] = [0, 1, 2, 3, 4, 0, 1, 2]
    c["spans"][1] = [5, 0]
    c["spans"][2] = [100, 2**32 - 1]          # all of it a prompt
    c["history"][3] = 17
    c["spans"][3] = [1, 64]
    c["ids"][:] = rng.permutation(400)[:9] + 20
    c["ids"][4] = 77
    c["values"][5, 0] = np.nan
    c["params"][5] = [2.0, 0.0, 0.0]
    got = decode(run(torch_cuda, backend, c, dtype), dtype).reshape(6, 500)
    want = process_logits(x, c["history"], c["spans"], c["params"], c["ids"], c["values"], c["mask"])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isneginf(got[1]).all() and np.array_equal(np.isinf(got), np.isinf(want))
    fin = np.isfinite(want)
    # |x| <= 16, penalties <= 65, nine biases of |3 * 4|: at most 190; 15 steps in f32
    assert (np.abs(got[fin] - want[fin]) <= 15 * 190 * 2.0 ** -24 + HALF[dtype] * np.abs(want[fin])).all()
    # a division by zero and an infinite penalty are the formula's
    c["params"][0] = [0.0, np.inf, 1.0]
    got = decode(run(torch_cuda, backend, c, dtype), dtype).reshape(6, 500)
    want = process_logits(x, c["history"], c["spans"], c["params"], c["ids"], c["values"], c["mask"])
    assert np.array_equal(np.isnan(got[0]), np.isnan(want[0]))
    assert np.array_equal(np.isposinf(got[0]), np.isposinf(want[0]))


def test_biases_of_one_token_add_in_the_lists_order(torch_cuda, backend):
    """1e8 - 1e8 + 1 in list order is 1 in f32; another order gives 0."""
    c = dict(x=np.zeros((1, 10), np.float32), history=None, spans=None, params=None, mask=None,
             ids=np.array([[3, 5, 3, 3, 5]], np.int32),
             values=np.array([[1e8, 2.0, -1e8, 1.0, 3.0]], np.float32))
    got = run(torch_cuda, backend, c, DTYPE_F32)
    assert got[0, 3] == 1.0 and got[0, 5] == 5.0 and np.count_nonzero(got) == 2


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("offset", [0, 3])
def test_more_columns_with_a_rule_than_are_listed(torch_cuda, backend, dtype, offset):
    """Histories that name most of a workgroup's 8192 columns, beside ones that name few."""
    rng = np.random.default_rng(offset)
    c = make(rng, 4, 17000, 9001, 30, True, dtype)
    c["history"][1] = rng.integers(8000, 8400, 9001)      # one workgroup's end and the next one's start
    c["history"][2] = rng.integers(0, 2100, 9001)
    c["spans"][:, 1] = [9001, 9000, 9001, 8192]
    check(run(torch_cuda, backend, c, dtype, offset), c, dtype)
