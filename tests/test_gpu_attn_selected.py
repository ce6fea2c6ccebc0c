"""AttentionI8Selected (133) on the device against 64 bits, row by row within the bound that
packed_reference derives, and the run of a long-context step's calls (130-133 and 127): by
themselves, as a session's walk, captured and replayed."""
import numpy as np
import pytest

from conftest import from_dev, to_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, AttentionI8SelectedCall, BufferRef,
                          DeviceWorkspace, HipBackend, HipSession, KernelCall, SlotOutOfRange)
from long_context_reference import attend_listed, block_bounds, rotary, select_blocks
from packed_reference import ALL, block_append, bound, decode, encode
from test_gpu_packed_batch import blocks_case, dispatch, run_blocks, starts_of
from test_long_context import long_step_graph

pytestmark = pytest.mark.gpu


def selected_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, scales="powers", pad=0, kind="choice"):
    c = blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, dtype, scales, pad)
    c["top"], nb = top, -(-bucket // block)
    tokens = sum(rows)
    if kind == "choice":                     # distinct blocks of the plane, in any order, -1 among them
        lists = np.stack([rng.permutation(max(nb, top))[:top] for _ in range(tokens * Hkv)])
        lists[lists >= nb] = -1
    else:                                    # any entry at all, the same ones again, none in range
        lists = rng.integers(-3, nb + 3, (tokens * Hkv, top))
        lists[::3] = lists[::3, :1]
        lists[1::5] = -1
        lists[2::7] = np.resize([nb, -2**31, 2**31 - 1, -1], top)
    c["lists"] = lists.reshape(tokens, Hkv, top).astype(np.int32)
    return c


def run_selected(torch, backend, c):
    tokens, es = c["q"].shape[0], c["q"].itemsize
    fill = np.full((tokens, c["H"], c["D"]), 7, c["q"].dtype)
    call = KernelCall.AttentionI8Selected(AttentionI8SelectedCall(
        BufferRef(0, c["pad"] * es), *[BufferRef(s) for s in range(1, 9)], tokens, len(c["rows"]), c["H"], c["Hkv"],
        c["bucket"], c["block"], c["D"], c["pad"] + c["H"] * c["D"], c["top"], 0, c["dtype"]))
    _, ts = dispatch(torch, backend, call, [c["q"], c["k"], c["v"], c["ks"], c["vs"], c["lists"], c["starts"],
                                            c["lens"], fill])
    return from_dev(ts[8], fill.dtype).reshape(fill.shape)


def check_selected(got, c, gap=0):
    dtype, n = c["dtype"], sum(c["rows"])
    q = decode(c["q"], dtype).reshape(c["q"].shape)[gap:gap + n, c["pad"]:].reshape(n, c["H"], c["D"])
    want, slack, top = attend_listed(q, c["k"], c["v"], c["ks"], c["vs"], c["lists"][gap:gap + n], c["lens"], c["rows"],
                                     c["Hkv"], c["block"], np.sqrt(c["D"]))
    err = np.abs(decode(got[gap:gap + n], dtype).reshape(want.shape) - want)
    tol = bound(slack, top, dtype)
    assert (err <= tol).all(), float(np.nanmax(err / np.maximum(tol, 1e-30)))
    assert (got[:gap] == 7).all() and (got[gap + n:] == 7).all()


SHAPES = [  # rows, lens, H, Hkv, D, bucket, block, top, pad
    ([1, 1, 1, 1, 1], [1, 0, 33, 500, 257], 8, 2, 128, 512, 32, 5, 0),    # decode; a row with no key
    ([1] * 9, list(range(120, 129)), 4, 4, 64, 130, 16, 7, 0),            # one head a kv head, a short last block
    ([1, 0, 1], [700, 3, 64], 32, 2, 64, 701, 64, 3, 8),                  # 16 heads a kv head, an empty sequence
    ([1, 1], [90, 2000], 24, 1, 128, 2048, 128, 16, 0),                   # more heads than 16
    ([2, 4, 1], [2, 300, 17], 4, 2, 96, 320, 32, 10, 0),                  # drafts
    ([3, 5], [1, 4], 2, 1, 64, 64, 16, 4, 0),                             # rows before the first key
    ([70, 33], [70, 400], 8, 2, 128, 512, 64, 6, 0),                      # a chunk
    ([5, 1], [250, 249], 6, 2, 256, 256, 32, 8, 0),
    ([9], [150], 3, 1, 128, 150, 32, 5, 8),                               # a bucket that ends inside a block
    ([1, 1], [50, 20], 2, 1, 48, 64, 16, 4, 0),
    ([20, 1], [90, 60], 2, 1, 72, 100, 10, 4, 3),                         # nothing of the tiles' sizes
    ([5], [9], 1, 1, 320, 16, 7, 3, 0),
    ([1, 4], [40, 50], 2, 1, 64, 50, 100, 1, 0),                          # one block, longer than the bucket
    ([1], [4000000000], 2, 1, 64, 96, 32, 3, 0),                          # a length past the bucket
    ([1], [6000], 4, 1, 128, 6016, 16, 300, 0),                           # one row, a long list
    ([1, 2], [9000, 8000], 34, 2, 64, 9024, 64, 130, 0),                  # three times 16 heads' tiles
    ([1], [64], 1, 1, 1024, 64, 16, 4, 0),
    ([2], [5000], 2, 1, 16, 5000, 256, 20, 0),
    ([1, 2], [60, 33], 4, 2, 64, 70, 1 << 31, 40, 0),                     # one block, longer than any cache
    ([3], [900], 2, 1, 128, 1000, 1 << 16, 3, 0),
    ([2, 1], [5, 4100], 2, 1, 64, 12288, 4096, 3, 0),                     # a block of which few rows are seen
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block,top,pad", SHAPES)
def test_selected_parity(torch_cuda, backend, rows, lens, H, Hkv, D, bucket, block, top, pad, dtype):
    rng = np.random.default_rng(sum(rows) + D + bucket)
    for scales, kind in (("powers", "choice"), ("any", "anything")):
        c = selected_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, scales, pad, kind)
        check_selected(run_selected(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128, 72])
def test_every_block_is_all_of_the_cache(torch_cuda, backend, D, dtype):
    """With a list of every block the rows are those of AttentionI8Blocks, each within the bound of
    the same exact result."""
    rng = np.random.default_rng(D)
    c = selected_case(rng, [1, 6], [300, 512], 4, 2, D, 512, 32, 16, dtype)
    c["lists"] = np.broadcast_to(np.arange(16, dtype=np.int32), c["lists"].shape).copy()
    check_selected(run_selected(torch_cuda, backend, c), c)
    check_selected(run_blocks(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,top", [(1, 6), (1, 200), (30, 6)])
@pytest.mark.parametrize("D", [64, 128, 72])
def test_what_a_row_does_not_see_stays_out(torch_cuda, backend, dtype, n, top, D):
    """Scales of blocks that no list names or that lie past a row's keys are NaN and infinite: every
    bit is what it is without them. One that a row does see reaches its heads alone."""
    rng = np.random.default_rng(n + D)
    bucket, block = 16 * (2 * top + 8), 16
    nb = bucket // block
    c = selected_case(rng, [n, n], [bucket - 8, bucket - 40], 4, 2, D, bucket, block, top, dtype)
    odd = 2 * rng.permutation(nb // 2 - 4)[:top] + 1                   # odd blocks, not the last ones
    c["lists"][:] = odd[None, None, :]
    c["lists"][:, :, 0] = nb - 1                                       # part of it seen by some rows, by some none
    clean = run_selected(torch_cuda, backend, c)
    check_selected(clean, c)
    for s in ("ks", "vs"):
        c[s] = c[s].copy()
        c[s][:, :, 0:nb - 1:2] = np.nan if s == "ks" else np.inf
        c[s][1, :, nb - 1] = np.nan                                    # sequence 1 ends before it
    assert np.array_equal(run_selected(torch_cuda, backend, c), clean)
    c["vs"][0, 1, odd[1]] = np.nan
    got = run_selected(torch_cuda, backend, c)
    assert np.array_equal(got[:, :2], clean[:, :2]) and np.array_equal(got[n:], clean[n:])
    assert np.isnan(decode(got[:n, 2:], dtype)).all()


def test_large_and_small_block_scales(torch_cuda, backend):
    rng = np.random.default_rng(9)
    for n, top in ((1, 25), (3, 200), (80, 25)):
        c = selected_case(rng, [n, n], [4000, 90], 4, 2, 64, 4000, 16, top, DTYPE_F32)
        c["vs"] = (2.0 ** rng.integers(-30, 31, c["vs"].shape)).astype(np.float32)
        c["vs"][:, :, 3] = 0.0
        c["vs"][:, :, ::5] *= -1.0
        check_selected(run_selected(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 72])
def test_rows_outside_the_sequences_stay_as_they_were(torch_cuda, backend, D, dtype):
    rng = np.random.default_rng(D)
    for rows, top in (([1, 3], 150), ([20, 33], 5)):
        c = selected_case(rng, rows, [2600, 400], 8, 2, D, 2608, 16, top, dtype)
        width, n = c["q"].shape[1], sum(rows)
        c["q"] = np.concatenate([encode(np.full((2, width), np.nan), dtype).reshape(2, width), c["q"],
                                 encode(np.full((3, width), np.nan), dtype).reshape(3, width)])
        c["lists"] = np.concatenate([c["lists"][:2], c["lists"], c["lists"][:3]])[:n + 5]
        c["lists"] = np.resize(c["lists"], (n + 5, 2, top)).astype(np.int32)
        c["starts"] = starts_of(rows, 2)
        check_selected(run_selected(torch_cuda, backend, c), c, gap=2)


def test_selected_many_sequences(torch_cuda, backend):
    rng = np.random.default_rng(3)
    rows = list(rng.integers(0, 4, 300))
    c = selected_case(rng, rows, rng.integers(0, 400, 300), 4, 1, 64, 384, 32, 6, DTYPE_BF16)
    check_selected(run_selected(torch_cuda, backend, c), c)


@pytest.mark.parametrize("D", [64, 72])
@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [0, 5, 9, 21], [2**32 - 1, 0, 3, 20], [20, 0, 20, 0]])
def test_bad_offsets_are_reported(torch_cuda, backend, starts, D):
    c = selected_case(np.random.default_rng(0), [9, 5, 6], [30, 20, 10], 4, 2, D, 64, 16, 3, DTYPE_BF16)
    c["starts"] = np.array(starts, np.uint32)
    with pytest.raises(SlotOutOfRange):
        run_selected(torch_cuda, backend, c)
    backend.synchronize()


# -------------------------------------------------------------------- a step ----
class Step:
    """A server's cache and the session that takes one packed step over it."""
    def __init__(self, rng, backend, batch, tokens, heads, kv, d, bucket, block, top, dtype, interleaved):
        self.shape = (heads, kv, d, bucket, block, top, dtype, interleaved)
        self.gamma = encode(1 + 0.3 * rng.standard_normal(d), dtype)
        self.freqs = (10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
        nb = -(-bucket // block)
        self.k, self.v = (np.zeros((batch, kv, bucket, d), np.int8) for _ in "kv")
        self.ks, self.vs = (np.zeros((batch, kv, nb), np.float32) for _ in "kv")
        self.bounds = np.zeros((batch, kv, nb, 2, d), np.int8)
        self.tokens, self.batch = tokens, batch
        self.session = HipSession(backend, long_step_graph(tokens, batch, heads, kv, d, bucket, block, top, dtype,
                                                           self.gamma, self.freqs, d, interleaved))
        for i, x in ((4, self.k), (5, self.v), (6, self.ks), (7, self.vs), (8, self.bounds)):
            self.session.write_input(i, x.tobytes())

    def write(self, qkv, rows, pos):
        self.session.write_input(0, qkv.tobytes())
        self.session.write_input(1, starts_of(rows).tobytes())
        self.session.write_input(2, np.array(pos, np.uint32).tobytes())
        self.session.write_input(3, (np.array(pos) + rows).astype(np.uint32).tobytes())

    def check(self, qkv, rows, pos):
        """The session's outputs against the restatement: its rotated rows and its result within their
        bounds, and what follows from the rows as the device rounded them, caches, scales, bounds and
        lists, equal."""
        heads, kv, d, bucket, block, top, dtype, interleaved = self.shape
        n, lens = sum(rows), np.array(pos) + rows
        x = decode(qkv, dtype).reshape(qkv.shape)[:n].reshape(n, heads + 2 * kv, d)
        at = np.concatenate([p + np.arange(r) for r, p in zip(rows, pos)])
        raw = lambda i, t, s: np.frombuffer(self.session.read_output(i), t).reshape(s)  # noqa: E731
        q, k = (decode(raw(i, qkv.dtype, (self.tokens, h, d))[:n], dtype).reshape(n, h, d) for i, h in ((7, heads), (8, kv)))
        for got, rows_in in ((q, x[:, :heads]), (k, x[:, heads:heads + kv])):
            want, tol = rotary(rows_in, decode(self.gamma, dtype), 1e-6, at, self.freqs, d, interleaved, 1.0, dtype)
            assert (np.abs(got - want) <= tol).all()
        self.k, self.ks = block_append(self.k, self.ks, k, rows, pos, block)
        self.v, self.vs = block_append(self.v, self.vs, x[:, heads + kv:], rows, pos, block)
        self.bounds = block_bounds(self.k, self.bounds, rows, pos, block)
        for i, w in enumerate((self.k, self.v, self.ks, self.vs, self.bounds)):
            assert np.array_equal(raw(i, w.dtype, w.shape), w), i
        lists = raw(5, np.int32, (self.tokens, kv, top))[:n]
        assert np.array_equal(lists, select_blocks(q, self.bounds, self.ks, lens, rows, kv, bucket, block, top, 1, 2))
        out = raw(6, qkv.dtype, (self.tokens, heads, d))[:n]
        want, slack, most = attend_listed(q, self.k, self.v, self.ks, self.vs, lists, lens, rows, kv, block, np.sqrt(d))
        assert (np.abs(decode(out, dtype).reshape(want.shape) - want) <= bound(slack, most, dtype)).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("interleaved", [0, 1])
def test_steps_of_a_long_context(torch_cuda, backend, dtype, interleaved):
    """Prompts, then chunks and single tokens behind them, over one cache: eager, then captured and
    replayed with other rows, lengths and positions."""
    rng = np.random.default_rng(5 + interleaved)
    s = Step(rng, backend, 3, 40, 4, 2, 64, 256, 16, 5, dtype, interleaved)
    turns = [[20, 0, 20], [20, 19, 1], [1, 1, 1], [0, 30, 1], [1, 1, 1], [16, 1, 23], [1, 1, 1]]
    pos = np.zeros(3, np.int64)
    for turn, rows in enumerate(turns):
        qkv = encode(rng.standard_normal((40, 8 * 64)), dtype).reshape(40, 8 * 64)
        s.write(qkv, rows, pos)
        if turn < 2:
            s.session.run()
        elif turn == 2:
            s.session.capture()
        else:
            s.session.replay()
        s.session.synchronize()
        s.check(qkv, rows, pos)
        pos = pos + rows
    s.session.close()


@pytest.mark.parametrize("bucket,top", [(2048, 40), (20480, 100)])
def test_captured_on_a_stream_of_its_own(torch_cuda, bucket, top):
    """The four calls in one graph on another stream than torch's: every replay, over other inputs and
    lengths, is the eager result, bit for bit; with lists and attention of one launch each, and of
    two that share the backend's scratch."""
    torch = torch_cuda
    from hologram_amd import (KvBlockBoundsCall, KvBlockSelectCall, QkNormRotaryCall)
    rng = np.random.default_rng(11)
    H, Hkv, D, block, tokens, dtype = 8, 2, 64, 16, 12, DTYPE_BF16
    far = bucket - 2048
    nb = bucket // block
    cases = []
    for rows, lens in (([1, 1, 1], [far + 2000, 40, 900]), ([4, 4, 4], [2000, bucket, 5]), ([12, 0, 0], [far + 1500, 0, 0]),
                       ([0, 1, 11], [0, 1, far + 2000])):
        c = blocks_case(rng, rows, lens, H, Hkv, D, bucket, block, dtype)
        c["x"] = encode(rng.standard_normal((tokens, (H + Hkv) * D)), dtype).reshape(tokens, -1)
        c["pos"] = np.maximum(np.array(lens, np.int64) - rows, 0).astype(np.uint32)
        cases.append(c)
    freqs = (10000.0 ** (-np.arange(32) / 32)).astype(np.float32)
    names = ["x", "starts", "pos", "lens", "k", "v", "ks", "vs"]
    outs = [((tokens, H, D), np.uint16), ((tokens, Hkv, D), np.uint16), ((3, Hkv, nb, 2, D), np.int8),
            ((tokens, Hkv, top), np.int32), ((tokens, H, D), np.uint16)]

    def calls():
        R, w = BufferRef, (H + Hkv) * D
        return [KernelCall.QkNormRotary(QkNormRotaryCall(R(0), R(0, 2 * H * D), BufferRef(0xFFFFFFFF), BufferRef(0xFFFFFFFF),
                                                         R(1), R(2), R(8), R(9), R(10), tokens, 3, H, Hkv, D, D, w, w)),
                KernelCall.KvBlockBounds(KvBlockBoundsCall(R(4), R(1), R(2), R(11), R(11), tokens, 3, Hkv, bucket, block, D)),
                KernelCall.KvBlockSelect(KvBlockSelectCall(R(9), R(11), R(6), R(1), R(3), R(12), tokens, 3, H, Hkv, bucket,
                                                           block, D, 0, top, 1, 2)),
                KernelCall.AttentionI8Selected(AttentionI8SelectedCall(R(9), R(4), R(5), R(6), R(7), R(12), R(1), R(3), R(13),
                                                                       tokens, 3, H, Hkv, bucket, block, D, 0, top))]

    def bind(c):
        ts = [to_dev(torch, c[n]) for n in names] + [to_dev(torch, freqs)]
        ts += [to_dev(torch, np.zeros(s, t)) for s, t in outs]
        ws = DeviceWorkspace()
        for s, t in enumerate(ts):
            ws.bind(s, t)
        return ws, ts

    def read(ts):
        return [from_dev(t, d).reshape(s) for t, (s, d) in zip(ts[9:], outs)]
    stream = torch.cuda.Stream()
    be, eager = HipBackend(0, stream.cuda_stream), HipBackend(0, torch.cuda.current_stream().cuda_stream)
    want = []
    for c in cases:
        ws, ts = bind(c)
        for call in calls():
            eager.dispatch(call, ws)
        eager.synchronize()
        want.append(read(ts))
    ws, ts = bind(cases[0])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for call in calls():
            be.dispatch(call, ws)              # sizes the scratch
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in calls():
            be.dispatch(call, ws)
    for turn in (1, 2, 0, 3, 1, 0):
        for name, t in zip(names, ts):
            t.copy_(to_dev(torch, cases[turn][name]))
        for t in ts[9:]:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(read(ts), want[turn]):
            assert np.array_equal(got, w), turn
        ws2, ts2 = bind(cases[turn])           # eager work between the replays
        for call in calls():
            eager.dispatch(call, ws2)
        eager.synchronize()
        for got, w in zip(read(ts2), want[turn]):
            assert np.array_equal(got, w)
    be.close()
    eager.close()


# ------------------------------------------------- many rows of few heads ----
MANY = [  # sequences' rows, lens, H, Hkv, D, bucket, block, top
    ([130, 1, 0, 60], [700, 33, 9, 60], 16, 4, 64, 704, 16, 7),      # steps that end inside a turn
    ([180], [900], 3, 3, 128, 1000, 32, 9),                          # one head a kv head, a bucket off the blocks
    ([70, 70, 70], [300, 3, 800], 12, 4, 96, 800, 64, 5),            # three heads a kv head, rows that see nothing
    ([1] * 300, [700 - 2 * i for i in range(300)], 4, 2, 128, 704, 128, 3),   # one token each
    ([90, 50], [500, 520], 16, 4, 80, 520, 16, 1),                   # one step a row
    ([300], [640], 10, 2, 64, 640, 16, 21),                          # five heads: not of them
    ([130, 20], [900, 640], 8, 4, 256, 900, 16, 5),                  # nor 256 dims
    ([200], [120], 8, 4, 64, 128, 1 << 20, 4),                       # one block, listed several times
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block,top", MANY)
def test_many_rows_of_few_heads(torch_cuda, backend, rows, lens, H, Hkv, D, bucket, block, top, dtype):
    rng = np.random.default_rng(sum(rows) + D)
    for scales, kind in (("powers", "choice"), ("any", "anything")):
        c = selected_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, scales, 0, kind)
        check_selected(run_selected(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D,block", [(64, 16), (128, 32)])
def test_many_rows_what_a_row_does_not_see_stays_out(torch_cuda, backend, dtype, D, block):
    """As above for many rows of few heads: the steps of one turn lie in different columns, and a
    scale that is NaN or infinite reaches none but the rows that see its block."""
    rng = np.random.default_rng(D)
    n, nb, top = 150, 24, 7
    c = selected_case(rng, [n, n], [nb * block - 3, nb * block - 2 * block], 8, 2, D, nb * block, block, top, dtype)
    odd = 2 * rng.permutation(nb // 2 - 2)[:top] + 1
    c["lists"][:] = odd[None, None, :]
    c["lists"][:, :, 3] = nb - 1
    clean = run_selected(torch_cuda, backend, c)
    check_selected(clean, c)
    for s in ("ks", "vs"):
        c[s] = c[s].copy()
        c[s][:, :, 0:nb - 1:2] = np.nan if s == "ks" else np.inf
        c[s][1, :, nb - 1] = np.nan
    assert np.array_equal(run_selected(torch_cuda, backend, c), clean)
    for s in ("ks", "vs"):
        old = c[s][0, 1, odd[1]]
        c[s][0, 1, odd[1]] = np.nan
        got = run_selected(torch_cuda, backend, c)
        c[s][0, 1, odd[1]] = old
        sees = np.array([int(c["lens"][0]) - (n - 1 - t) > odd[1] * block for t in range(n)])
        assert np.array_equal(got[:, :4], clean[:, :4]) and np.array_equal(got[n:], clean[n:])
        assert np.isnan(decode(got[:n][sees][:, 4:], dtype)).all()
        assert np.array_equal(got[:n][~sees], clean[:n][~sees])


def test_many_rows_large_and_small_block_scales(torch_cuda, backend):
    rng = np.random.default_rng(9)
    c = selected_case(rng, [150, 150], [4000, 390], 8, 2, 64, 4000, 16, 25, DTYPE_F32)
    c["vs"] = (2.0 ** rng.integers(-30, 31, c["vs"].shape)).astype(np.float32)
    c["vs"][:, :, 3] = 0.0
    c["vs"][:, :, ::5] *= -1.0
    check_selected(run_selected(torch_cuda, backend, c), c)


@pytest.mark.parametrize("n", [3, 300])
def test_a_row_of_scores_that_are_infinite(torch_cuda, backend, n):
    """K scales of -infinity give scores of either infinity, which make the row NaN as the formula
    does; a query that is not finite makes its own head's row NaN and no other."""
    rng = np.random.default_rng(n)
    c = selected_case(rng, [n], [600], 8, 2, 64, 640, 16, 5, DTYPE_BF16)
    c["lists"][:] = np.array([3, 9, 20, 21, 36])
    clean = run_selected(torch_cuda, backend, c)
    q = decode(c["q"], DTYPE_BF16).reshape(n, -1).copy()
    q[1, 64 + 5], q[2, 5 * 64] = np.nan, np.inf                # head 1 of row 1, head 5 of row 2
    c["q"] = encode(q, DTYPE_BF16).reshape(n, -1)
    got = run_selected(torch_cuda, backend, c)
    keep = np.ones((n, 8), bool)
    keep[1, 1] = keep[2, 5] = False
    assert np.array_equal(got[keep], clean[keep]) and np.isnan(decode(got[~keep], DTYPE_BF16)).all()
    c["ks"][0, 1, 20] = -np.inf
    got = run_selected(torch_cuda, backend, c)
    assert np.array_equal(got[:, :4][keep[:, :4]], clean[:, :4][keep[:, :4]])
    # a score of +infinity, or 0 times infinity, among those that the row sees: weights that are NaN
    q = decode(c["q"], DTYPE_BF16).reshape(n, 8, 64)
    with np.errstate(invalid="ignore"):
        dots = q[:, 4:] @ c["k"][0, 1, 320:336].astype(np.float64).T              # [n, 4, 16]
    sees = (320 + np.arange(16) < 600 - (n - 1 - np.arange(n))[:, None])[:, None]   # [n, 1, 16]
    nan = (sees & ~(dots > 0)).any(axis=2) | ~keep[:, 4:]
    assert np.array_equal(np.isnan(decode(got[:, 4:], DTYPE_BF16)).reshape(n, 4, 64).all(axis=2), nan)
    assert np.array_equal(np.isnan(decode(got[:, 4:], DTYPE_BF16)).reshape(n, 4, 64).any(axis=2), nan)


# ------------------------------------------------- lists past one workgroup's ----
def long_lists(rng, tokens, kv, top, nb, filled):
    """Lists of `top` entries of which `filled` name blocks, among them the places about each 512th;
    the others are out of range."""
    lists = rng.choice([-1, nb, nb + 5, -2**31, 2**31 - 1], (tokens, kv, top)).astype(np.int64)
    edges = [i for c in range(0, top + 1, 512) for i in (c - 1, c, c + 1) if 0 <= i < top]
    for _ in range(filled):
        at = rng.integers(0, top, (tokens, kv))
        at = np.where(rng.random((tokens, kv)) < 0.6, rng.choice(edges, (tokens, kv)), at)
        np.put_along_axis(lists, at[..., None], rng.integers(0, nb, (tokens, kv, 1)), axis=2)
    lists[::5] = -1                          # rows whose list names nothing
    lists[1::5, :, :min(top, 512)] = -1      # and whose first 512 do not
    return lists.astype(np.int32)


@pytest.mark.parametrize("dtype", [DTYPE_BF16, DTYPE_F32])
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block,top", [
    ([4100, 0, 60], [4000, 3, 700], 8, 2, 64, 4096, 16, 513),        # one share: two rounds of a list
    ([2100], [2200], 16, 4, 128, 2208, 32, 1300),                    # three rounds
    ([8200], [9000], 17, 1, 64, 9008, 16, 600),                      # more heads than 16
    ([3000], [3000], 1, 1, 128, 3008, 16, 1600),                     # two shares of two rounds each
    ([700], [700], 4, 1, 256, 704, 16, 1100),                        # a share a round
    ([2], [700], 4, 2, 64, 704, 16, 30000),                          # few rows, more shares than rounds
])
def test_lists_of_several_rounds(torch_cuda, backend, rows, lens, H, Hkv, D, bucket, block, top, dtype):
    rng = np.random.default_rng(top)
    c = selected_case(rng, rows, lens, H, Hkv, D, bucket, block, 1, dtype)
    c["top"], nb = top, -(-bucket // block)
    c["lists"] = long_lists(rng, sum(rows), Hkv, top, nb - 2, 5)
    c["ks"], c["vs"] = c["ks"].copy(), c["vs"].copy()
    c["ks"][:, :, nb - 2:], c["vs"][:, :, nb - 2:] = np.nan, np.inf          # blocks that nothing names
    c["lists"][c["lists"] == nb - 2] = -1
    check_selected(run_selected(torch_cuda, backend, c), c)


def test_long_lists_of_many_rows_take_little_scratch(torch_cuda):
    """16384 rows with lists of 513 entries: what the backend allocates stays below the 136 MB that
    the header states, and the result is the formula's."""
    torch = torch_cuda
    rng = np.random.default_rng(1)
    c = selected_case(rng, [16384], [16400], 1, 1, 256, 16400, 16, 1, DTYPE_BF16)
    c["top"], c["lists"] = 513, long_lists(rng, 16384, 1, 513, 1025, 3)
    be = HipBackend(0, torch.cuda.current_stream().cuda_stream)
    before = []

    class Watched:
        def dispatch(self, call, ws):
            torch.cuda.synchronize()
            before.append(torch.cuda.mem_get_info()[0])
            be.dispatch(call, ws)

        def synchronize(self):
            be.synchronize()
            before.append(torch.cuda.mem_get_info()[0])
    got = run_selected(torch, Watched(), c)
    assert before[0] - before[1] < 140 << 20, (before[0] - before[1]) >> 20
    check_selected(got, c)
    be.close()
