"""KvBlockAppend (127) on the device: bytes and scales equal to the 64-bit restatement (powers of
two leave nothing to round but the values themselves), rows it does not write untouched."""
import numpy as np
import pytest

from conftest import from_dev, to_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F32, BufferRef, DeviceWorkspace, KernelCall,
                          KvBlockAppendCall, SlotOutOfRange, UnsupportedOp)
from packed_reference import ALL, block_append, decode, encode

pytestmark = pytest.mark.gpu


def make(rng, rows, kv, D, bucket, block, dtype, pad=0, spread=3.0):
    B, nb, tokens = len(rows), -(-bucket // block), sum(rows)
    x = rng.standard_normal((tokens, pad + kv * D)) * np.exp2(rng.uniform(-spread, spread, (tokens, 1)))
    return dict(new=encode(x, dtype).reshape(tokens, pad + kv * D),
                cache=rng.integers(-127, 128, (B, kv, bucket, D), dtype=np.int8),
                scales=(2.0 ** rng.integers(-9, -4, (B, kv, nb))).astype(np.float32), pad=pad)


def run(torch, backend, c, rows, pos, block, dtype, in_place=True, starts=None):
    B, kv, bucket, D = c["cache"].shape
    tokens, es = c["new"].shape[0], c["new"].itemsize
    if starts is None:
        starts = np.concatenate([[0], np.cumsum(rows)])
    ws, ts = DeviceWorkspace(), []
    for a in (c["new"], np.asarray(starts, np.uint32), np.asarray(pos, np.uint32), c["cache"], c["scales"]):
        ts.append(to_dev(torch, a) if a.nbytes else torch.zeros(16, dtype=torch.uint8, device="cuda"))
    if not in_place:
        ts += [torch.full_like(ts[3], 0x55), torch.full_like(ts[4], 0x55)]
    for s, t in enumerate(ts):
        ws.bind(s, t)
    o = 3 if in_place else 5
    backend.dispatch(KernelCall.KvBlockAppend(KvBlockAppendCall(
        BufferRef(0, c["pad"] * es), BufferRef(1), BufferRef(2), BufferRef(3), BufferRef(4), BufferRef(o),
        BufferRef(o + 1), tokens, B, kv, bucket, block, D, c["pad"] + kv * D, dtype)), ws)
    backend.synchronize()
    return (from_dev(ts[o], np.int8).reshape(c["cache"].shape),
            from_dev(ts[o + 1], np.float32).reshape(c["scales"].shape))


def want_of(c, rows, pos, block, dtype):
    B, kv, bucket, D = c["cache"].shape
    new = decode(c["new"], dtype).reshape(c["new"].shape)[:, c["pad"]:].reshape(-1, kv, D)
    return block_append(c["cache"], c["scales"], new, rows, pos, block)


SHAPES = [  # rows, pos, kv, D, bucket, block, pad
    ([1, 1, 1, 1], [0, 31, 32, 63], 2, 128, 64, 32, 0),       # decode: block ends and starts
    ([1] * 40, list(range(40)), 8, 64, 48, 16, 0),
    ([100, 0, 37], [5, 9, 0], 2, 128, 128, 32, 0),            # a prompt over a held prefix, an empty one
    ([64, 65], [0, 63], 1, 96, 128, 64, 8),
    ([33, 2], [10, 90], 3, 80, 100, 16, 0),                   # a bucket that ends inside a block
    ([20, 5], [3, 0], 2, 33, 30, 7, 1),                       # nothing aligned
    ([9], [2], 1, 1, 16, 1, 0),                               # a scale a row
    ([10], [0], 1, 5, 20, 64, 0),                             # one block, longer than the bucket
    ([300], [1], 1, 1024, 301, 128, 0),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,pos,kv,D,bucket,block,pad", SHAPES)
def test_append_is_exact(torch_cuda, backend, rows, pos, kv, D, bucket, block, pad, dtype):
    rng = np.random.default_rng(D + bucket)
    c = make(rng, rows, kv, D, bucket, block, dtype, pad)
    want = want_of(c, rows, pos, block, dtype)
    for in_place in (True, False):
        got = run(torch_cuda, backend, c, rows, pos, block, dtype, in_place)
        for g, w in zip(got, want):
            assert np.array_equal(g, w)


@pytest.mark.parametrize("dtype", ALL)
def test_row_by_row_equals_the_restatement(torch_cuda, backend, dtype):
    """Forty decode steps, the rows' magnitudes growing: scales double, held rows are rounded again."""
    rng = np.random.default_rng(1)
    c = make(rng, [1, 1], 2, 64, 64, 32, dtype)
    grew = 0
    for step in range(40):
        c["new"] = encode(rng.standard_normal((2, 128)) * (1.0 + step % 32), dtype).reshape(2, 128)
        want = want_of(c, [1, 1], [step, step + 3], 32, dtype)
        got = run(torch_cuda, backend, c, [1, 1], [step, step + 3], 32, dtype)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        grew += int((got[1] > c["scales"]).sum())
        c["cache"], c["scales"] = got
    assert grew > 8


@pytest.mark.parametrize("dtype", ALL)
def test_odd_values(torch_cuda, backend, dtype):
    """Zeros, subnormal and largest values, the border 127 * 2^e, NaN and infinity; blocks held over a
    zero, a NaN and another NaN scale."""
    rng = np.random.default_rng(5)
    D, block = 32, 16
    x = np.zeros((9 * 16, D))
    big = {7: 3.3e38, 6: 65504.0, 8: 3.4e38}[dtype]
    tiny = {7: 1e-40, 6: 6e-8, 8: 1e-45}[dtype]
    x[16:32, 3] = big
    x[32:48] = tiny
    x[48, 0], x[49, 1] = 127.0, -127.0
    x[64, 0] = 127.5 if dtype != 7 else 128.0
    x[80:96] = rng.standard_normal((16, D))
    x[85, 7] = np.nan
    x[100, 2] = -np.inf
    x[112:] = np.rint(rng.standard_normal((32, D)) * 60) / 2      # ties
    c = dict(new=encode(x, dtype).reshape(-1, D), pad=0,
             cache=rng.integers(-127, 128, (1, 1, 160, D), dtype=np.int8),
             scales=np.ones((1, 1, 10), np.float32))
    want = want_of(c, [144], [0], block, dtype)
    got = run(torch_cuda, backend, c, [144], [0], block, dtype)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1], equal_nan=True)
    for s, n in ((0.0, 3), (np.nan, 3), (2.0 ** -20, 3), (2.0 ** 40, 3), (0.37, 3), (-0.25, 3)):
        c["scales"][:] = s
        c["new"] = encode(rng.standard_normal((n, D)), dtype).reshape(n, D)
        want = want_of(c, [n], [18], block, dtype)
        got = run(torch_cuda, backend, c, [n], [18], block, dtype)
        if s != 0.37:          # (its quotients round in f32: a value may sit on either side of a half)
            assert np.array_equal(got[0], want[0])
        else:
            assert np.abs(got[0].astype(int) - want[0]).max() <= 1
        assert np.array_equal(got[1], want[1], equal_nan=True)


def test_rows_past_the_bucket_are_dropped_and_reported(torch_cuda, backend):
    rng = np.random.default_rng(6)
    c = make(rng, [4, 5, 1], 2, 64, 40, 16, DTYPE_F32)
    pos = [37, 1, 2**32 - 1]
    with pytest.raises(UnsupportedOp, match="bucket_rows"):
        run(torch_cuda, backend, c, [4, 5, 1], pos, 16, DTYPE_F32)
    backend.synchronize()
    with pytest.raises(SlotOutOfRange, match="starts"):
        run(torch_cuda, backend, c, [4, 5, 1], [0, 0, 0], 16, DTYPE_F32, starts=[0, 4, 2, 10])
    backend.synchronize()


def test_dropped_rows_leave_the_rest_exact(torch_cuda, backend):
    rng = np.random.default_rng(7)
    c = make(rng, [4, 5], 2, 64, 40, 16, DTYPE_BF16)
    want = want_of(c, [4, 5], [37, 1], 16, DTYPE_BF16)
    ws, ts = DeviceWorkspace(), []
    for a in (c["new"], np.array([0, 4, 9], np.uint32), np.array([37, 1], np.uint32), c["cache"], c["scales"]):
        ts.append(to_dev(torch_cuda, a))
    for s, t in enumerate(ts):
        ws.bind(s, t)
    backend.dispatch(KernelCall.KvBlockAppend(KvBlockAppendCall(
        BufferRef(0), BufferRef(1), BufferRef(2), BufferRef(3), BufferRef(4), BufferRef(3), BufferRef(4),
        9, 2, 2, 40, 16, 64, 0, DTYPE_BF16)), ws)
    with pytest.raises(UnsupportedOp):
        backend.synchronize()
    assert np.array_equal(from_dev(ts[3], np.int8).reshape(want[0].shape), want[0])
    assert np.array_equal(from_dev(ts[4], np.float32).reshape(want[1].shape), want[1])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("off", [0, 16, 5])
@pytest.mark.parametrize("channels,inner", [(6, 4096), (7, 16), (1, 48), (3, 24)])
def test_a_cache_reads_back_through_dequantize(torch_cuda, backend, dtype, off, channels, inner):
    """Runs of whole 16-byte chunks and others, aligned and not, with more runs than channels:
    (q - zero point) * scale, narrowed as the reference narrows, bit for bit."""
    import oracle
    from hologram_amd import DTYPE_I8, DequantizeCall
    rng = np.random.default_rng(channels)
    n = 2 * channels * inner
    q = rng.integers(0, 256, n + off, dtype=np.uint8)
    scales = (2.0 ** rng.integers(-9, 3, channels)).astype(np.float32)
    zps = rng.integers(-300, 300, channels).astype(np.int32)
    out = torch_cuda.zeros(n * (4 if dtype == DTYPE_F32 else 2) + off * 4, dtype=torch_cuda.uint8, device="cuda")
    ws = DeviceWorkspace()
    for s, t in enumerate((to_dev(torch_cuda, q), to_dev(torch_cuda, scales), to_dev(torch_cuda, zps), out)):
        ws.bind(s, t)
    backend.dispatch(KernelCall.Dequantize(DequantizeCall(
        BufferRef(0, off), BufferRef(1), BufferRef(2), BufferRef(3, off * 4), n, channels, inner, DTYPE_I8, dtype)), ws)
    backend.synchronize()
    want = oracle.dequantize(q[off:], n, DTYPE_I8, dtype, scales=scales, zps=zps, channels=channels, inner=inner)
    assert np.array_equal(out.cpu().numpy()[off * 4:], np.ascontiguousarray(want).view(np.uint8).reshape(-1))
