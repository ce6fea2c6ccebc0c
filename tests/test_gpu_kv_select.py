"""KvBlockBounds (131) and KvBlockSelect (132) on the device: both are whole numbers, so they equal
the 64-bit restatement."""
import math

import numpy as np
import pytest

from conftest import from_dev, to_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, DTYPE_I8, BufferRef, DequantizeCall,
                          DeviceWorkspace, HipBackend, KernelCall, KvBlockBoundsCall, KvBlockSelectCall, SlotOutOfRange)
from long_context_reference import block_bounds, eight_bits, select_blocks
from packed_reference import ALL, decode, encode
from test_gpu_packed_batch import dispatch, starts_of

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ bounds ----
def run_bounds(torch, backend, cache, bounds, rows, pos, block, gap=0, tail=0, in_place=True, starts=None):
    B, kv, bucket, D = cache.shape
    call = KernelCall.KvBlockBounds(KvBlockBoundsCall(
        BufferRef(0), BufferRef(1), BufferRef(2), BufferRef(3), BufferRef(3 if in_place else 4),
        gap + sum(rows) + tail, B, kv, bucket, block, D))
    arrays = [cache, starts_of(rows, gap) if starts is None else starts, np.array(pos, np.uint32), bounds,
              np.full_like(bounds, 55)]
    _, ts = dispatch(torch, backend, call, arrays)
    if not in_place:
        assert np.array_equal(from_dev(ts[3], np.int8).reshape(bounds.shape), bounds)
    return from_dev(ts[3 if in_place else 4], np.int8).reshape(bounds.shape)


BOUND_SHAPES = [  # rows, pos, kv, D, bucket, block
    ([1], [0], 1, 64, 64, 16),
    ([1, 1, 1, 1], [0, 15, 16, 63], 8, 128, 64, 16),
    ([5, 0, 40, 17], [3, 9, 20, 0], 2, 128, 96, 32),          # an empty sequence, several blocks
    ([100, 200], [0, 56], 2, 96, 256, 64),
    ([70], [11], 1, 256, 130, 32),                            # a bucket that ends inside a block
    ([30, 3], [90, 98], 2, 64, 100, 16),                      # rows past the bucket
    ([1, 2], [100, 4000000000], 2, 64, 100, 16),              # nothing of them in it
    ([9, 20], [5, 1], 3, 37, 50, 7),                          # nothing of the wide form's sizes
    ([4], [0], 1, 1024, 16, 4),
    ([6, 6], [2, 3], 1, 1, 20, 5),
    ([20], [3], 2, 80, 40, 1000),                             # a block longer than the bucket
    ([300], [40], 1, 16, 400, 1),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("rows,pos,kv,D,bucket,block", BOUND_SHAPES)
def test_bounds_equal(torch_cuda, backend, rows, pos, kv, D, bucket, block, in_place):
    rng = np.random.default_rng(sum(rows) + D)
    cache = rng.integers(-128, 128, (len(rows), kv, bucket, D), dtype=np.int8)
    bounds = rng.integers(-128, 128, (len(rows), kv, -(-bucket // block), 2, D), dtype=np.int8)
    want = block_bounds(cache, bounds, rows, pos, block)
    for gap, tail in ((0, 0), (2, 3)):
        got = run_bounds(torch_cuda, backend, cache, bounds, rows, pos, block, gap, tail, in_place)
        assert np.array_equal(got, want)


def test_bounds_many_sequences(torch_cuda, backend):
    rng = np.random.default_rng(1)
    rows = list(rng.integers(0, 30, 300))
    pos = rng.integers(0, 120, 300)
    cache = rng.integers(-100, 100, (300, 2, 128, 64), dtype=np.int8)
    bounds = np.zeros((300, 2, 8, 2, 64), np.int8)
    assert np.array_equal(run_bounds(torch_cuda, backend, cache, bounds, rows, pos, 16),
                          block_bounds(cache, bounds, rows, pos, 16))


def test_bounds_are_what_dequantize_reads(torch_cuda, backend):
    """With one channel a block and the cache's scales they become the values they stand for."""
    rng = np.random.default_rng(2)
    bounds = rng.integers(-127, 128, (2, 3, 5, 2, 64), dtype=np.int8)
    scales = 2.0 ** rng.integers(-8, 0, (2, 3, 5)).astype(np.float32)
    call = KernelCall.Dequantize(DequantizeCall(BufferRef(0), BufferRef(1), BufferRef(2), BufferRef(3), bounds.size,
                                                scales.size, 128, DTYPE_I8, DTYPE_F32))
    _, ts = dispatch(torch_cuda, backend, call, [bounds, scales, np.zeros(scales.size, np.int32),
                                                 np.zeros(bounds.size, np.float32)])
    assert np.array_equal(from_dev(ts[3], np.float32).reshape(bounds.shape), bounds * scales[..., None, None])


# ------------------------------------------------------------------ select ----
def select_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, first=1, last=1, pad=0, gap=0, tail=0):
    B, nb, tokens = len(rows), -(-bucket // block), gap + sum(rows) + tail
    c = dict(rows=rows, lens=np.array(lens, np.uint32), H=H, Hkv=Hkv, D=D, bucket=bucket, block=block, top=top,
             first=first, last=last, dtype=dtype, pad=pad, gap=gap, starts=starts_of(rows, gap))
    c["q"] = encode(rng.standard_normal((tokens, pad + H * D)) * 1.5, dtype).reshape(tokens, pad + H * D)
    x = np.sort(rng.integers(-128, 128, (B, Hkv, nb, 2, D), dtype=np.int8), axis=3)
    c["bounds"], c["ks"] = x, (rng.uniform(0.2, 1.0, (B, Hkv, nb)) / 127).astype(np.float32)
    return c


def run_select(torch, backend, c):
    tokens, es = c["q"].shape[0], c["q"].itemsize
    fill = np.full((tokens, c["Hkv"], c["top"]), -7, np.int32)
    call = KernelCall.KvBlockSelect(KvBlockSelectCall(
        BufferRef(0, c["pad"] * es), *[BufferRef(s) for s in range(1, 6)], tokens, len(c["rows"]), c["H"], c["Hkv"],
        c["bucket"], c["block"], c["D"], c["pad"] + c["H"] * c["D"], c["top"], c["first"], c["last"], c["dtype"]))
    _, ts = dispatch(torch, backend, call, [c["q"], c["bounds"], c["ks"], c["starts"], c["lens"], fill])
    return from_dev(ts[5], np.int32).reshape(fill.shape)


def check_select(got, c):
    gap, n = c["gap"], sum(c["rows"])
    q = decode(c["q"], c["dtype"]).reshape(c["q"].shape)[gap:gap + n, c["pad"]:].reshape(n, c["H"], c["D"])
    want = select_blocks(q, c["bounds"], c["ks"], c["lens"], c["rows"], c["Hkv"], c["bucket"], c["block"], c["top"],
                         c["first"], c["last"])
    assert np.array_equal(got[gap:gap + n], want)
    assert (got[:gap] == -7).all() and (got[gap + n:] == -7).all()


SELECT_SHAPES = [  # rows, lens, H, Hkv, D, bucket, block, top, first, last, pad
    ([1, 1, 1, 1, 1], [1, 0, 200, 500, 512], 8, 2, 128, 512, 16, 6, 1, 2, 0),  # decode; rows with no key, with few
    ([1], [5000], 4, 4, 64, 5000, 16, 10, 0, 1, 0),                            # one head a kv head, 313 blocks
    ([1, 0, 1], [9000, 3, 4000], 32, 2, 64, 9000, 16, 40, 2, 3, 8),            # 16 heads, 563 blocks
    ([1, 1], [4500, 9000], 24, 1, 128, 9000, 4, 64, 1, 1, 0),                  # 2250 blocks, 24 heads
    ([2, 4, 1], [300, 1000, 17], 4, 2, 96, 1024, 32, 5, 1, 2, 0),              # drafts
    ([70, 33], [70, 1400], 8, 2, 128, 1500, 64, 4, 1, 1, 0),                   # a chunk across block ends
    ([129, 1, 40], [500, 480, 150], 4, 2, 64, 512, 16, 8, 1, 2, 0),
    ([40], [1250], 6, 2, 256, 1256, 32, 7, 3, 4, 0),                           # nothing left to choose
    ([5], [90], 2, 1, 48, 100, 8, 3, 1, 1, 0),
    ([20, 1], [90, 60], 2, 1, 72, 100, 5, 3, 1, 1, 3),                         # nothing aligned
    ([5], [900], 1, 1, 320, 1000, 7, 9, 0, 9, 0),
    ([3], [64], 2, 1, 1024, 64, 4, 6, 1, 1, 0),
    ([2], [700], 3, 1, 5, 700, 3, 50, 2, 2, 1),
    ([1], [4000000000], 2, 1, 64, 960, 32, 4, 1, 1, 0),                        # a length past the bucket
    ([1, 2], [600, 640], 4, 2, 64, 640, 64, 10, 1, 1, 0),                      # every block fits the list
    ([1, 1], [600, 640], 4, 2, 64, 640, 64, 12, 1, 1, 0),                      # the list is longer
    ([17, 16], [333, 3000], 12, 4, 128, 3001, 16, 16, 1, 1, 0),
    ([9, 1], [700, 650], 4, 2, 64, 704, 16, 6, 1, 1, 1),                       # the tiles' sizes, rows off 16 bytes
    ([3], [900], 256, 1, 64, 900, 16, 9, 1, 1, 0),                             # more heads than two int8 parts hold
    ([2, 1], [2500, 2000], 16, 1, 128, 2500, 4, 20, 1, 1, 0),                  # sums past 2^24
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,lens,H,Hkv,D,bucket,block,top,first,last,pad", SELECT_SHAPES)
def test_select_equal(torch_cuda, backend, rows, lens, H, Hkv, D, bucket, block, top, first, last, pad, dtype):
    rng = np.random.default_rng(sum(rows) + D + bucket)
    c = select_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, first, last, pad)
    check_select(run_select(torch_cuda, backend, c), c)
    c = select_case(rng, rows, lens, H, Hkv, D, bucket, block, top, dtype, first, last, pad, gap=2, tail=3)
    c["ks"][:, :, ::3] *= -1.0               # negative scales: the bounds change sides
    check_select(run_select(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 72])
@pytest.mark.parametrize("rows,bucket", [([1, 1], 1000), ([20, 33], 1000), ([1, 1], 12000)])
def test_select_equal_scores_go_by_their_order(torch_cuda, backend, rows, bucket, D, dtype):
    """Whole runs of equal scores, among them zeros of both signs; NaN and infinite scales, whose
    scores rank first, or last where they are negative infinity; a border inside such a run."""
    rng = np.random.default_rng(bucket + D)
    c = select_case(rng, rows, [bucket - 5, bucket], 4, 2, D, bucket, 4, 37, dtype)
    for kind in range(5):
        if kind == 0:
            c["bounds"][:] = c["bounds"][:, :, :1]
            c["ks"][:] = 0.25
        elif kind == 1:                      # three kinds of blocks in turn
            c["bounds"][:, :, 1::3] = c["bounds"][:, :, :1] // 2
            c["ks"][:, :, 2::3] = -0.125
        elif kind == 2:
            c["ks"][:] = 0.0
            c["ks"][:, :, ::2] = -0.0
        elif kind == 3:
            c["bounds"][:] = 0
            c["ks"][:] = 1.0
            c["ks"][:, :, 5::7] = -1.0
            c["ks"][:, :, 50::9] = np.inf    # zero times infinity: NaN, first
        else:
            c = select_case(rng, rows, [bucket - 5, bucket], 4, 2, D, bucket, 4, 37, dtype)
            c["ks"][:, :, ::11], c["ks"][:, :, 1::13] = np.nan, np.inf
            c["ks"][:, :, 2::17] = -np.inf
        check_select(run_select(torch_cuda, backend, c), c)


@pytest.mark.parametrize("H", [2, 64])
@pytest.mark.parametrize("D", [64, 72])
@pytest.mark.parametrize("rows,bucket", [([1, 1], 1200), ([20, 33], 1200), ([1, 1], 8000), ([1, 1], 20000)])
def test_select_scores_next_to_one_another(torch_cuda, backend, rows, bucket, D, H):
    """Scales from the least subnormal to the largest number, scores that differ in their last bit
    or past f32's: the exact order decides, not a rounded one's."""
    rng = np.random.default_rng(bucket + D + H)
    c = select_case(rng, rows, [bucket - 5, bucket], H, 2, D, bucket, 4, 37, DTYPE_BF16)
    c["ks"] = np.ldexp(rng.uniform(0.5, 1.0, c["ks"].shape), rng.integers(-148, 129, c["ks"].shape)).astype(np.float32)
    c["ks"][:, :, ::4] *= -1.0
    check_select(run_select(torch_cuda, backend, c), c)
    c["bounds"][:] = c["bounds"][:, :, :1]          # one block's bounds under scales a step apart
    c["ks"] = (1.0 + rng.integers(0, 40, c["ks"].shape) * 2.0 ** -23).astype(np.float32)
    check_select(run_select(torch_cuda, backend, c), c)
    c["ks"][:] = np.float32(3.3e38)                 # all past f32's largest
    c["bounds"] = select_case(rng, rows, [0, 0], H, 2, D, bucket, 4, 37, DTYPE_BF16)["bounds"]
    check_select(run_select(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 72])
def test_select_rows_that_are_not_finite(torch_cuda, backend, D, dtype):
    """Elements that are not finite count as 0, rows of zeros and of the smallest numbers score
    what they score, and the largest do not overflow."""
    rng = np.random.default_rng(D)
    c = select_case(rng, [9], [800], 4, 2, D, 800, 8, 12, dtype)
    q = decode(c["q"], dtype).reshape(9, -1).copy()
    q[1, ::5], q[2, 3], q[3, 1::2], q[4] = np.nan, np.inf, -np.inf, 0.0
    q[5, :2 * D] = np.nan
    q[6] *= 2.0 ** -24 if dtype == DTYPE_F16 else 2.0 ** -133
    q[7] *= 2.0 ** 13 if dtype == DTYPE_F16 else 2.0 ** 125
    c["q"] = encode(np.clip(q, -3e38, 3e38) if dtype != DTYPE_F16 else q, dtype).reshape(9, -1)
    q = decode(c["q"], dtype).reshape(9, -1)
    q[2, 3] = np.inf
    q[3, 1::2] = -np.inf
    c["q"] = encode(q, dtype).reshape(9, -1)
    check_select(run_select(torch_cuda, backend, c), c)


@pytest.mark.parametrize("D", [64, 72])
def test_what_a_row_does_not_see_stays_out_of_its_list(torch_cuda, backend, D):
    """The bounds and scales of the block that holds a row's last key, and of every later one, do
    not count: the lists are the same whatever they hold."""
    rng = np.random.default_rng(D)
    c = select_case(rng, [40], [1000], 4, 2, D, 1040, 16, 9, DTYPE_BF16)
    clean = run_select(torch_cuda, backend, c)
    check_select(clean, c)
    c["ks"][0, :, 60:] = np.inf              # rows 960 on: the last row's block 62, the first's 60
    c["bounds"][0, :, 60:] = 127
    got = run_select(torch_cuda, backend, c)
    assert np.array_equal(got[:16], clean[:16])      # (they see up to 976 keys: 61 blocks, the last kept)
    check_select(got, c)


def test_select_many_sequences_and_rows(torch_cuda, backend):
    rng = np.random.default_rng(7)
    rows = list(rng.integers(0, 4, 300))
    c = select_case(rng, rows, rng.integers(0, 700, 300), 4, 2, 64, 640, 16, 8, DTYPE_BF16)
    check_select(run_select(torch_cuda, backend, c), c)
    c = select_case(rng, [700, 3, 300], [900, 1000, 1000], 4, 1, 64, 1000, 16, 8, DTYPE_F16, gap=1, tail=1)
    check_select(run_select(torch_cuda, backend, c), c)


def test_select_many_blocks(torch_cuda, backend):
    """More blocks a plane than a workgroup holds keys of."""
    rng = np.random.default_rng(8)
    c = select_case(rng, [1, 2], [70000, 69000], 2, 1, 16, 70000, 2, 300, DTYPE_BF16)
    check_select(run_select(torch_cuda, backend, c), c)


@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [0, 5, 9, 21], [2**32 - 1, 0, 3, 20], [20, 0, 20, 0]])
def test_bad_offsets_are_reported(torch_cuda, backend, starts):
    rng = np.random.default_rng(0)
    cache = rng.integers(-100, 100, (3, 2, 64, 64), dtype=np.int8)
    with pytest.raises(SlotOutOfRange):
        run_bounds(torch_cuda, backend, cache, np.zeros((3, 2, 4, 2, 64), np.int8), [9, 5, 6], [0, 1, 2], 16,
                   starts=np.array(starts, np.uint32))
    backend.synchronize()
    for D in (64, 72):
        c = select_case(rng, [9, 5, 6], [300, 200, 100], 4, 2, D, 320, 16, 4, DTYPE_BF16)
        c["starts"] = np.array(starts, np.uint32)
        with pytest.raises(SlotOutOfRange):
            run_select(torch_cuda, backend, c)
        backend.synchronize()


def nearly_equal_pair(rng, sums, scale_sign):
    """Blocks a < b and mantissas (24 bits) whose products with their sums differ, b's score the larger,
    by less than f64 tells apart; whole numbers throughout."""
    while True:
        a, b = sorted(rng.choice(np.arange(1, len(sums) - 1), 2, replace=False).tolist())
        sa, sb = int(sums[a]), int(sums[b])
        if math.gcd(sa, sb) != 1:
            continue
        for d in (1, 2, 3):
            d *= -scale_sign                 # sa ma - sb mb = d
            ma = d * pow(sa, -1, sb) % sb
            mb = (sa * ma - d) // sb
            if all(1 << 23 <= m < 1 << 24 for m in (ma, mb)) and float(sa * ma) == float(sb * mb):
                return a, b, ma, mb


@pytest.mark.parametrize("nb", [90, 4200])
@pytest.mark.parametrize("H,D", [(2048, 64), (1820, 72)])
def test_select_scores_past_53_bits(torch_cuda, backend, H, D, nb):
    """Groups of 2^17 elements, whose sums have 31 bits and whose scores 55: two of them that f64
    would round to the same number are not equal, and the later block, whose score is the larger,
    is the one. (Scores of either sign; all others far below.)"""
    rng = np.random.default_rng(H + nb)
    B, block = 12, 4
    q = rng.integers(100, 128, (H, D))
    q[0, 0] = 127
    lo = rng.integers(100, 128, (nb, D))
    sums = lo @ q.sum(axis=0)
    assert sums.min() > 1 << 30 and sums.max() < 1 << 31
    ks, want = np.zeros((B, 1, nb), np.float32), np.zeros((B, 1, 3), np.int32)
    for s in range(B):
        sign = 1 if s % 2 else -1
        ks[s] = sign * 2.0 ** (-60 if sign > 0 else 60)
        a, b, ma, mb = nearly_equal_pair(rng, sums, sign)
        ks[s, 0, a], ks[s, 0, b] = (sign * m * 2.0 ** -30 for m in (ma, mb))
        want[s, 0] = 0, b, nb - 1
    c = dict(rows=[1] * B, lens=np.full(B, nb * block, np.uint32), H=H, Hkv=1, D=D, bucket=nb * block, block=block,
             top=3, first=1, last=1, dtype=DTYPE_BF16, pad=0, gap=0, starts=starts_of([1] * B), ks=ks)
    c["q"] = encode(np.broadcast_to(q.reshape(-1), (B, H * D)).astype(np.float64), DTYPE_BF16).reshape(B, -1)
    c["bounds"] = np.broadcast_to(lo[None, None, :, None], (B, 1, nb, 2, D)).astype(np.int8)
    assert np.array_equal(run_select(torch_cuda, backend, c), want)


@pytest.mark.parametrize("D,bucket,block,top", [
    (72, 320, 16, 20),                       # the general form, as many entries as blocks
    (72, 320, 16, 33),
    (64, 1300, 2, 650),                      # two launches
    (64, 9000, 2, 4600),                     # and more blocks than a workgroup holds
])
@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [0, 5, 9, 21], [2**32 - 1, 0, 3, 20], [20, 0, 20, 0]])
def test_bad_offsets_are_reported_where_every_block_fits_the_list(torch_cuda, backend, starts, D, bucket, block, top):
    rng = np.random.default_rng(0)
    c = select_case(rng, [9, 5, 6], [300, 200, 100], 4, 2, D, bucket, block, top, DTYPE_BF16)
    check_select(run_select(torch_cuda, backend, c), c)
    c["starts"] = np.array(starts, np.uint32)
    with pytest.raises(SlotOutOfRange):
        run_select(torch_cuda, backend, c)
    backend.synchronize()


@pytest.mark.parametrize("D,top", [(64, 700), (72, 640)])
def test_a_list_of_every_block_is_captured_without_an_eager_run(torch_cuda, D, top):
    """It takes no scratch: nothing has to be dispatched before the capture. Each replay over other
    lengths is the restatement's."""
    torch = torch_cuda
    rng = np.random.default_rng(D)
    cases = [select_case(rng, [5, 0, 15], lens, 4, 2, D, 1280, 2, top, DTYPE_BF16)
             for lens in ([1280, 7, 15], [6, 0, 1279], [1, 1, 900])]
    stream = torch.cuda.Stream()
    be = HipBackend(0, stream.cuda_stream)
    ts = [to_dev(torch, cases[0][n]) for n in ("q", "bounds", "ks", "starts", "lens")]
    out = torch.empty((20, 2, top), dtype=torch.int32, device="cuda")
    ws = DeviceWorkspace()
    for s, t in enumerate([*ts, out]):
        ws.bind(s, t)
    call = KernelCall.KvBlockSelect(KvBlockSelectCall(*[BufferRef(s) for s in range(6)], 20, 3, 4, 2, 1280, 2, D, 0,
                                                      top, 1, 1, DTYPE_BF16))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        be.dispatch(call, ws)
    for turn in (1, 2, 0, 2):
        for n, t in zip(("q", "bounds", "ks", "starts", "lens"), ts):
            t.copy_(to_dev(torch, cases[turn][n]))
        out.fill_(-7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_select(out.cpu().numpy(), cases[turn])
    be.close()


@pytest.mark.parametrize("D", [64, 72])
def test_select_bounds_that_are_not_in_order(torch_cuda, backend, D):
    """Where lo is above hi, a block that nothing has bounded yet, hi still goes with the positive
    elements of Q and lo with the negative ones, the other way round under a negative scale."""
    rng = np.random.default_rng(D)
    c = select_case(rng, [30], [1000], 4, 2, D, 1000, 8, 9, DTYPE_F32)
    c["bounds"] = rng.integers(-128, 128, c["bounds"].shape, dtype=np.int8)
    c["ks"][:, :, ::3] *= -1.0
    got = run_select(torch_cuda, backend, c)
    q = decode(c["q"], DTYPE_F32).reshape(30, 2, 2, D)
    lo, hi = c["bounds"][0].astype(np.int64).transpose(2, 0, 1, 3)               # [kv, nb, D]
    for t in range(30):
        seen = -(-(1000 - 29 + t) // 8)
        j = np.arange(1, seen - 1)
        for h in range(2):
            x = eight_bits(q[t, h]).astype(np.int64)
            up, down = np.maximum(x, 0).sum(axis=0), np.minimum(x, 0).sum(axis=0)
            s = c["ks"][0, h, j].astype(np.float64)
            score = s * np.where(s < 0, lo[h, j] @ up + hi[h, j] @ down, hi[h, j] @ up + lo[h, j] @ down)
            best = j[np.argsort(-score, kind="stable")[:7]]
            assert got[t, h].tolist() == sorted([0, *best.tolist(), seen - 1])
