"""AttentionPacked (126) and AttentionI8Blocks (128) on the device against 64 bits, row by row
within the bound that packed_reference derives; the rows, lengths and masks where they could go
wrong; and what the device reports."""
import numpy as np
import pytest

from conftest import from_dev, to_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, AttentionI8BlocksCall,
                          AttentionPackedCall, BufferRef, DeviceWorkspace, KernelCall,
                          SlotOutOfRange)
from packed_reference import ALL, attend, bound, decode, encode

pytestmark = pytest.mark.gpu


def starts_of(rows, before=0):
    return (np.concatenate([[0], np.cumsum(rows)]) + before).astype(np.uint32)


def dispatch(torch, backend, call, arrays, sync=True):
    ws = DeviceWorkspace()
    ts = [a if isinstance(a, torch.Tensor) else to_dev(torch, a) for a in arrays]
    for s, t in enumerate(ts):
        ws.bind(s, t)
    backend.dispatch(call, ws)
    if sync:
        backend.synchronize()
    return ws, ts


def packed_case(rng, rows, H, Hkv, D, dtype, pad=0, gap=0, tail=0):
    """q, k, v as views of one buffer [tokens, pad + row], `gap` rows before the first sequence
    and `tail` behind the last."""
    tokens, width = gap + sum(rows) + tail, (H + 2 * Hkv) * D + pad
    qkv = rng.standard_normal((tokens, width)) * 1.5
    return encode(qkv, dtype).reshape(tokens, width), tokens, width


def run_packed(torch, backend, qkv, rows, H, Hkv, D, dtype, pad, gap=0, starts=None):
    tokens, width = qkv.shape
    es = qkv.itemsize
    fill = np.full(tokens * H * D, 7, encode(np.zeros(1), dtype).dtype)
    call = KernelCall.AttentionPacked(AttentionPackedCall(
        BufferRef(0, pad * es), BufferRef(0, (pad + H * D) * es), BufferRef(0, (pad + (H + Hkv) * D) * es),
        BufferRef(1), BufferRef(2), tokens, len(rows), H, Hkv, D, width, width, width, 0, dtype))
    _, ts = dispatch(torch, backend, call, [qkv, starts_of(rows, gap) if starts is None else starts, fill])
    return from_dev(ts[2], fill.dtype).reshape(tokens, H, D)


def check_packed(got, qkv, rows, H, Hkv, D, dtype, pad, gap=0):
    x = decode(qkv, dtype).reshape(qkv.shape)
    at = gap
    for n in rows:
        r = x[at:at + n, pad:]
        q, k, v = np.split(r, [H * D, (H + Hkv) * D], axis=1)
        want, slack, top = attend(q.reshape(n, H, D), k.reshape(n, Hkv, D), v.reshape(n, Hkv, D),
                                  np.arange(1, n + 1), H, Hkv, np.sqrt(D))
        err = np.abs(decode(got[at:at + n], dtype).reshape(n, H, D) - want)
        assert (err <= bound(slack, top, dtype)).all(), (n, float((err / bound(slack, top, dtype)).max()))
        at += n
    sentinel = np.full(1, 7, got.dtype)[0]
    assert (got[:gap] == sentinel).all() and (got[at:] == sentinel).all()


SHAPES = [  # rows, H, Hkv, D, pad (elements before each token's q)
    ([1], 1, 1, 64, 0),
    ([1, 0, 5, 64, 65, 2], 8, 2, 64, 0),       # an empty sequence, tiles' ends
    ([130, 33, 0], 4, 1, 128, 8),              # past one tile, an empty last sequence
    ([31, 97], 6, 2, 128, 0),                  # three heads a kv head straddle the tiles
    ([40, 1, 200], 2, 2, 96, 0),
    ([77], 3, 3, 80, 16),
    ([50, 13], 2, 1, 256, 0),
    ([20, 3], 16, 1, 64, 0),
    ([9, 30], 2, 1, 72, 3),                    # nothing 16-byte aligned
    ([7], 2, 1, 5, 1),
    ([6, 2], 2, 2, 320, 0),                    # past the tiles' head sizes
    ([3], 1, 1, 1024, 0),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,H,Hkv,D,pad", SHAPES)
def test_packed_parity(torch_cuda, backend, rows, H, Hkv, D, pad, dtype):
    rng = np.random.default_rng(sum(rows) + D)
    qkv, _, _ = packed_case(rng, rows, H, Hkv, D, dtype, pad, gap=2, tail=3)
    got = run_packed(torch_cuda, backend, qkv, rows, H, Hkv, D, dtype, pad, gap=2)
    check_packed(got, qkv, rows, H, Hkv, D, dtype, pad, gap=2)


@pytest.mark.parametrize("dtype", ALL)
def test_packed_many_sequences(torch_cuda, backend, dtype):
    """More sequences than one probe of the search holds, most of them a row or none."""
    rng = np.random.default_rng(4)
    rows = list(rng.integers(0, 4, 300))
    rows[150] = 70
    qkv, _, _ = packed_case(rng, rows, 4, 2, 64, dtype)
    got = run_packed(torch_cuda, backend, qkv, rows, 4, 2, 64, dtype, 0)
    check_packed(got, qkv, rows, 4, 2, 64, dtype, 0)


@pytest.mark.parametrize("dtype", ALL)
def test_packed_longest_first(torch_cuda, backend, dtype):
    """More workgroups than the GPU holds at once: the tiles that see most keys go first."""
    rng = np.random.default_rng(5)
    rows = [129, 1, 0, 90, 200, 128]
    qkv, _, _ = packed_case(rng, rows, 64, 64, 32, dtype, gap=1, tail=1)
    got = run_packed(torch_cuda, backend, qkv, rows, 64, 64, 32, dtype, 0, gap=1)
    check_packed(got, qkv, rows, 64, 64, 32, dtype, 0, gap=1)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128, 96])
def test_what_a_row_does_not_see_stays_out(torch_cuda, backend, dtype, D):
    """NaN and infinities in later rows of the sequence (K, V and Q) and all over its neighbours:
    the rows before are what they are without them; the rows that see them are not finite."""
    rng = np.random.default_rng(D)
    H, Hkv, rows, bad = 8, 2, [40, 150, 40], 40 + 100
    qkv, tokens, width = packed_case(rng, rows, H, Hkv, D, dtype)
    clean = run_packed(torch_cuda, backend, qkv, rows, H, Hkv, D, dtype, 0)
    x = decode(qkv, dtype).reshape(tokens, width).copy()
    x[bad, H * D:(H + Hkv) * D:3] = np.nan          # K of one row
    x[bad + 1, (H + Hkv) * D:] = np.inf             # V of the next
    x[bad + 7, (H + Hkv) * D::5] = -np.inf
    x[bad + 9, :H * D] = np.nan                     # Q of a row: its own result only
    x[:40, :], x[190:, ::2] = np.nan, np.inf
    got = run_packed(torch_cuda, backend, encode(x, dtype).reshape(tokens, width), rows, H, Hkv, D, dtype, 0)
    assert np.array_equal(got[40:bad], clean[40:bad])
    assert not np.isfinite(decode(got[bad:190], dtype)).any()


@pytest.mark.parametrize("dtype", ALL)
def test_infinite_v_reaches_the_rows_that_see_it(torch_cuda, backend, dtype):
    """One V element infinite: exactly its dim of the rows from there on is infinite."""
    rng = np.random.default_rng(2)
    n, bad, H, Hkv, D = 90, 33, 4, 2, 64
    qkv, _, width = packed_case(rng, [n], H, Hkv, D, dtype)
    x = decode(qkv, dtype).reshape(n, width).copy()
    x[bad, (H + Hkv) * D + 5] = np.inf              # kv head 0, dim 5: heads 0 and 1
    got = decode(run_packed(torch_cuda, backend, encode(x, dtype).reshape(n, width), [n], H, Hkv, D, dtype, 0), dtype)
    want = np.zeros((n, H, D), bool)
    want[bad:, :2, 5] = True
    assert np.array_equal(np.isposinf(got.reshape(n, H, D)), want)
    assert np.isfinite(got.reshape(n, H, D)[~want]).all()


@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [0, 5, 9, 21], [2**32 - 1, 0, 3, 20], [20, 0, 20, 0]])
def test_bad_offsets_are_reported(torch_cuda, backend, starts):
    rng = np.random.default_rng(0)
    qkv, _, _ = packed_case(rng, [20], 4, 2, 64, DTYPE_BF16)
    with pytest.raises(SlotOutOfRange):
        run_packed(torch_cuda, backend, qkv, [1, 1, 1], 4, 2, 64, DTYPE_BF16, 0, starts=np.array(starts, np.uint32))
    backend.synchronize()
    c = blocks_case(rng, [9, 5, 6], [30, 20, 10], 4, 2, 64, 64, 16, DTYPE_BF16)
    c["starts"] = np.array(starts, np.uint32)
    with pytest.raises(SlotOutOfRange):
        run_blocks(torch_cuda, backend, c)
    backend.synchronize()


# ------------------------------------------------------------------- cache ----
def blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, dtype, scales="powers", pad=0):
    B, nb = len(rows), -(-bucket // block)
    c = dict(rows=rows, lens=np.array(lens, np.uint32), H=H, Hkv=Hkv, D=D, bucket=bucket, block=block,
             dtype=dtype, pad=pad, starts=starts_of(rows))
    tokens = sum(rows)
    c["q"] = encode(rng.standard_normal((tokens, pad + H * D)) * 1.5, dtype).reshape(tokens, pad + H * D)
    for n in "kv":
        c[n] = rng.integers(-127, 128, (B, Hkv, bucket, D), dtype=np.int8)
        s = rng.uniform(0.2, 1.0, (B, Hkv, nb)) / 127 if scales == "any" else \
            2.0 ** rng.integers(-9, -5, (B, Hkv, nb))
        c[n + "s"] = s.astype(np.float32)
    return c


def run_blocks(torch, backend, c, stream=None):
    tokens, es = c["q"].shape[0], c["q"].itemsize
    fill = np.full((tokens, c["H"], c["D"]), 7, c["q"].dtype)
    call = KernelCall.AttentionI8Blocks(AttentionI8BlocksCall(
        BufferRef(0, c["pad"] * es), *[BufferRef(s) for s in range(1, 8)], tokens, len(c["rows"]),
        c["H"], c["Hkv"], c["bucket"], c["block"], c["D"], c["pad"] + c["H"] * c["D"], 0, c["dtype"]))
    _, ts = dispatch(torch, backend, call, [c["q"], c["k"], c["v"], c["ks"], c["vs"], c["starts"],
                                            c["lens"], fill])
    return from_dev(ts[7], fill.dtype).reshape(fill.shape)


def check_blocks(got, c, sequences=None):
    dtype, H, Hkv, D = c["dtype"], c["H"], c["Hkv"], c["D"]
    q = decode(c["q"], dtype).reshape(c["q"].shape)[:, c["pad"]:].reshape(-1, H, D)
    at = 0
    for b, n in enumerate(c["rows"]):
        if sequences is None or b in sequences:
            keys = np.clip(int(c["lens"][b]) - (n - 1 - np.arange(n)), 0, c["bucket"])
            m = int(keys.max()) if n else 0
            of = np.arange(m) // c["block"]
            k, v = (c[x][b, :, :m].astype(np.float64) * c[x + "s"][b][:, of, None].astype(np.float64)
                    for x in "kv")
            want, slack, top = attend(q[at:at + n], k.transpose(1, 0, 2), v.transpose(1, 0, 2), keys, H,
                                      Hkv, np.sqrt(D))
            err = np.abs(decode(got[at:at + n], dtype).reshape(want.shape) - want)
            tol = bound(slack, top, dtype)
            assert (err <= tol).all(), (b, n, float(np.nanmax(err / np.maximum(tol, 1e-30))))
        at += n


BLOCK_SHAPES = [  # rows, lens, H, Hkv, D, bucket, block, pad
    ([1, 1, 1, 1, 1], [1, 0, 33, 500, 257], 8, 2, 128, 512, 32, 0),     # decode; a row with no key
    ([1] * 9, list(range(120, 129)), 4, 4, 64, 130, 16, 0),             # one head a kv head, a short last block
    ([1, 0, 1], [700, 3, 64], 32, 2, 64, 701, 64, 8),                   # 16 heads a kv head, an empty sequence
    ([1, 1], [90, 2000], 24, 1, 128, 2048, 128, 0),                     # more heads than 16 columns hold
    ([2, 4, 1], [2, 300, 17], 4, 2, 96, 320, 32, 0),                    # a few rows: drafts
    ([3, 5], [1, 4], 2, 1, 64, 64, 16, 0),                              # rows before the first key
    ([70, 33], [70, 400], 8, 2, 128, 512, 64, 0),                       # a chunk
    ([129, 1, 200], [500, 80, 150], 4, 2, 64, 512, 16, 0),              # rows that see nothing, a decode row among chunks
    ([40], [250], 6, 2, 256, 256, 32, 0),
    ([150], [150], 3, 1, 128, 150, 32, 8),                              # a bucket that ends inside a block
    ([1, 1], [50, 20], 2, 1, 48, 64, 16, 0),
    ([20, 1], [90, 60], 2, 1, 72, 100, 10, 3),                          # neither blocks nor heads of the tiles
    ([5], [9], 1, 1, 320, 16, 7, 0),
    ([1, 4], [40, 50], 2, 1, 64, 50, 100, 0),                           # one block, longer than the bucket
    ([1], [4000000000], 2, 1, 64, 96, 32, 0),                           # a length past the bucket
    ([1, 1, 4, 0, 1], [2500, 0, 2100, 9, 17], 4, 2, 128, 2500, 32, 0),  # shares that end inside a sequence
    ([1, 2], [2500, 1], 34, 2, 256, 2560, 128, 0),                      # two units a row
    ([1, 9], [5000, 4001], 3, 3, 96, 5000, 16, 0),                      # few: shares of two quads
    ([300], [4000], 2, 1, 64, 4096, 64, 0),                             # a chunk whose keys are split
    ([40, 1], [4000, 3000], 6, 2, 256, 4096, 32, 0),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block,pad", BLOCK_SHAPES)
def test_blocks_parity(torch_cuda, backend, rows, lens, H, Hkv, D, bucket, block, pad, dtype):
    rng = np.random.default_rng(sum(rows) + D + bucket)
    for scales in ("powers", "any"):
        c = blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, dtype, scales, pad)
        check_blocks(run_blocks(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,bucket", [(1, 1500), (1, 2500), (3, 2500), (60, 1500), (60, 2500)])
def test_blocks_many_ragged_sequences(torch_cuda, backend, rows, bucket, dtype):
    """Keys split among workgroups wherever a share ends, lengths from 0 to the bucket."""
    rng = np.random.default_rng(rows)
    B = 70
    lens = np.concatenate([[0, 1, 127, 128, 129, bucket], rng.integers(0, bucket + 1, B - 6)])
    c = blocks_case(rng, [rows] * B, lens, 8, 2, 64, bucket, 32, dtype)
    check_blocks(run_blocks(torch_cuda, backend, c), c, sequences=(0, 1, 2, 3, 4, 5, 20, 69))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [1, 4, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_unseen_rows_and_blocks_stay_out(torch_cuda, backend, dtype, n, D):
    """The block scales past a sequence's length, and a later block that only its last rows see,
    are NaN and infinite; other sequences' are too: the rest is what it is without them."""
    rng = np.random.default_rng(n + D)
    c = blocks_case(rng, [n, n], [200, 300], 4, 2, D, 320, 16, dtype)
    clean = run_blocks(torch_cuda, backend, c)
    for s in ("ks", "vs"):
        c[s] = c[s].copy()
        c[s][1, :, 19:] = np.nan          # rows 304 on: past every row's length
        c[s][0, :, 13:] = np.inf          # rows 208 on
    assert np.array_equal(run_blocks(torch_cuda, backend, c), clean)
    c["vs"][1, 0, 18] = np.nan            # rows 288-303 of kv head 0: the last 12 rows' keys
    got = run_blocks(torch_cuda, backend, c)
    sees = np.arange(2 * n) - n >= n - 12
    sees[:n] = False
    assert np.array_equal(got[~sees], clean[~sees])
    assert np.array_equal(got[:, 2:], clean[:, 2:])                # kv head 1
    assert np.isnan(decode(got[sees][:, :2], dtype)).all()


def test_large_and_small_block_scales(torch_cuda, backend):
    """Block scales from 2^-30 to 2^30 in one cache: weights and sums keep their precision, as the
    bound's largest |v| that the row sees allows; a zero scale reads as zeros."""
    rng = np.random.default_rng(9)
    for n in (1, 80):
        c = blocks_case(rng, [n, n], [400, 90], 4, 2, 64, 400, 16, DTYPE_F32)
        c["vs"] = (2.0 ** rng.integers(-30, 31, c["vs"].shape)).astype(np.float32)
        c["vs"][:, :, 3] = 0.0
        c["vs"][:, :, ::5] *= -1.0
        check_blocks(run_blocks(torch_cuda, backend, c), c)


def test_another_stream_and_replays(torch_cuda):
    """Captured on a stream of its own and replayed over changing inputs, with eager calls between:
    every replay is the eager result."""
    torch = torch_cuda
    from hologram_amd import HipBackend
    rng = np.random.default_rng(3)
    cases = [blocks_case(rng, [2, 40], [700, 333], 8, 2, 64, 704, 32, DTYPE_BF16) for _ in range(3)]
    stream = torch.cuda.Stream()
    be, eager = HipBackend(0, stream.cuda_stream), HipBackend(0, torch.cuda.current_stream().cuda_stream)
    want = [run_blocks(torch, eager, c) for c in cases]
    ws, ts = DeviceWorkspace(), []
    c = cases[0]
    for name in ("q", "k", "v", "ks", "vs", "starts", "lens"):
        ts.append(to_dev(torch, c[name]))
    ts.append(torch.zeros(c["q"].nbytes, dtype=torch.uint8, device="cuda"))
    for s, t in enumerate(ts):
        ws.bind(s, t)
    call = KernelCall.AttentionI8Blocks(AttentionI8BlocksCall(
        *[BufferRef(s) for s in range(8)], 42, 2, 8, 2, 704, 32, 64, 0, 0, DTYPE_BF16))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        be.dispatch(call, ws)              # sizes the scratch
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        be.dispatch(call, ws)
    for turn in (1, 2, 0, 2):
        for name, t in zip(("q", "k", "v", "ks", "vs", "starts", "lens"), ts):
            t.copy_(to_dev(torch, cases[turn][name]))
        ts[7].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(ts[7], np.uint16).reshape(want[turn].shape), want[turn])
        assert np.array_equal(run_blocks(torch, eager, cases[turn]), want[turn])
    be.close()
    eager.close()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block", [
    ([1, 3], [300, 40], 8, 2, 128, 512, 32),          # a unit a workgroup
    ([1, 3], [1500, 40], 8, 2, 128, 1536, 32),        # shares of units
    ([70, 33], [70, 400], 8, 2, 64, 512, 64),         # row tiles
    ([150, 33], [4000, 400], 4, 2, 64, 4096, 64),     # cut row tiles
    ([3, 20], [30, 90], 2, 1, 72, 100, 10),           # a row a wavefront
])
def test_rows_outside_the_sequences_stay_as_they_were(torch_cuda, backend, rows, lens, H, Hkv, D, bucket,
                                                      block, dtype):
    rng = np.random.default_rng(bucket)
    c = blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, dtype)
    width, n = c["q"].shape[1], sum(rows)
    c["q"] = np.concatenate([encode(np.full((2, width), np.nan), dtype).reshape(2, width), c["q"],
                             encode(np.full((3, width), np.nan), dtype).reshape(3, width)])
    c["starts"] = starts_of(rows, 2)
    got = run_blocks(torch_cuda, backend, c)
    assert (got[:2] == 7).all() and (got[2 + n:] == 7).all()
    check_blocks(got[2:2 + n], {**c, "q": c["q"][2:2 + n]})


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [4, 70])
def test_unseen_rows_and_blocks_stay_out_of_split_keys(torch_cuda, backend, dtype, n):
    """As above where a row's keys are several workgroups'."""
    rng = np.random.default_rng(n)
    c = blocks_case(rng, [n, n], [2500, 2990], 4, 2, 64, 3008, 16, dtype)
    clean = run_blocks(torch_cuda, backend, c)
    for s in ("ks", "vs"):
        c[s] = c[s].copy()
        c[s][1, :, 187:] = np.nan         # rows 2992 on
        c[s][0, :, 157:] = np.inf         # rows 2512 on
    assert np.array_equal(run_blocks(torch_cuda, backend, c), clean)
    c["vs"][1, 0, 186] = np.nan           # rows 2976-2991 of kv head 0: the last 14 rows' keys
    got = run_blocks(torch_cuda, backend, c)
    sees = np.arange(2 * n) - n >= n - 14
    sees[:n] = False
    assert np.array_equal(got[~sees], clean[~sees])
    assert np.array_equal(got[:, 2:], clean[:, 2:])
    assert np.isnan(decode(got[sees][:, :2], dtype)).all()


def test_a_graph_of_two_calls_over_changing_lengths(torch_cuda):
    """A chunk and a decode step over one cache in one graph, both in the backend's scratch:
    replayed with lengths that a workgroup takes whole, that several split, and none at all, each
    replay is the eager result, and within the bound."""
    torch = torch_cuda
    from hologram_amd import HipBackend
    rng = np.random.default_rng(5)
    rows, H, Hkv, D, bucket, block = [70, 33], 8, 2, 64, 4096, 32
    chunks = [blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, DTYPE_F16)
              for lens in ([70, 120], [4000, 3000], [0, 33], [2100, 33])]
    steps = [blocks_case(rng, [1, 1], c["lens"] + 1, H, Hkv, D, bucket, block, DTYPE_F16) for c in chunks]
    for c, s in zip(chunks, steps):
        for name in ("k", "v", "ks", "vs"):
            s[name] = c[name]
    stream = torch.cuda.Stream()
    be, eager = HipBackend(0, stream.cuda_stream), HipBackend(0, torch.cuda.current_stream().cuda_stream)
    want = [(run_blocks(torch, eager, c), run_blocks(torch, eager, s)) for c, s in zip(chunks, steps)]
    for (a, b), c, s in zip(want, chunks, steps):
        check_blocks(a, c)
        check_blocks(b, s)
    ws, ts, calls = DeviceWorkspace(), {}, []
    for tag, c in (("chunk", chunks[0]), ("step", steps[0])):
        names = ["q", "k", "v", "ks", "vs", "starts", "lens"]
        at = []
        for name in names:
            key = name if name in ("k", "v", "ks", "vs") else tag + name
            if key not in ts:
                ts[key] = (len(ts), to_dev(torch, c[name]))
            at.append(BufferRef(ts[key][0]))
        ts[tag + "out"] = (len(ts), torch.zeros(c["q"].nbytes, dtype=torch.uint8, device="cuda"))
        calls.append(KernelCall.AttentionI8Blocks(AttentionI8BlocksCall(
            *at, BufferRef(ts[tag + "out"][0]), sum(c["rows"]), 2, H, Hkv, bucket, block, D, 0, 0, DTYPE_F16)))
    for slot, t in ts.values():
        ws.bind(slot, t)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for call in calls:
            be.dispatch(call, ws)          # sizes the scratch
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in calls:
            be.dispatch(call, ws)
    for turn in (0, 1, 2, 3, 1, 0):
        for tag, c in (("chunk", chunks[turn]), ("step", steps[turn])):
            for name in ("q", "k", "v", "ks", "vs", "starts", "lens"):
                key = name if name in ("k", "v", "ks", "vs") else tag + name
                ts[key][1].copy_(to_dev(torch, c[name]))
            ts[tag + "out"][1].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for tag, w in zip(("chunk", "step"), want[turn]):
            assert np.array_equal(from_dev(ts[tag + "out"][1], w.dtype).reshape(w.shape), w), (turn, tag)
        assert np.array_equal(run_blocks(torch, eager, chunks[turn]), want[turn][0])
    be.close()
    eager.close()


@pytest.mark.parametrize("n", [1, 40])
def test_blocks_more_sequences_than_a_workgroup_has_threads(torch_cuda, backend, n):
    """Shares cut on a line of 300 sequences, several a thread, some of them empty."""
    rng = np.random.default_rng(n)
    B, bucket = 300, 2600
    rows = [0 if b % 7 == 3 else n for b in range(B)]
    lens = rng.integers(0, bucket + 1, B)
    lens[[0, 255, 256, 299]] = [bucket, 1, 2599, 1300]
    c = blocks_case(rng, rows, lens, 4, 1, 64, bucket, 32, DTYPE_BF16)
    check_blocks(run_blocks(torch_cuda, backend, c), c, sequences=(0, 1, 2, 150, 254, 255, 256, 257, 298, 299))
