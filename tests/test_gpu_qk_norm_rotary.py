"""QkNormRotary (130) on the device against 64 bits, within the bound that long_context_reference
derives."""
import struct

import numpy as np
import pytest

from conftest import from_dev
from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, NO_BUFFER, BufferRef, KernelCall,
                          QkNormRotaryCall, SlotOutOfRange)
from long_context_reference import rotary
from packed_reference import ALL, decode, encode
from test_gpu_packed_batch import dispatch, starts_of

pytestmark = pytest.mark.gpu
EPS = 1e-6


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


def rotary_case(rng, rows, pos, H, Hkv, D, rot, dtype, norms=3, interleaved=0, pad=0, gap=0, tail=0, magnitude=0.0,
                gammas=(True, True)):
    tokens, width = gap + sum(rows) + tail, pad + (H + 2 * Hkv) * D
    c = dict(rows=rows, pos=np.array(pos, np.uint32), H=H, Hkv=Hkv, D=D, rot=rot, dtype=dtype, norms=norms,
             interleaved=interleaved, pad=pad, gap=gap, magnitude=magnitude, starts=starts_of(rows, gap))
    c["qkv"] = encode(rng.standard_normal((tokens, width)) * 2.0, dtype).reshape(tokens, width)
    c["freqs"] = (10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1))).astype(np.float32)
    c["gammas"] = [encode(1 + 0.3 * rng.standard_normal(D), dtype) if g else None for g in gammas]
    return c


def run_rotary(torch, backend, c):
    tokens, width = c["qkv"].shape
    es, H, Hkv, D, pad = c["qkv"].itemsize, c["H"], c["Hkv"], c["D"], c["pad"]
    kv = max(Hkv, 1)
    fills = [np.full((tokens, n, D), 7, c["qkv"].dtype) for n in (H, kv)]
    arrays = [c["qkv"], c["starts"], c["pos"], c["freqs"] if c["rot"] else np.zeros(1, np.float32), *fills]
    gammas = []
    for g in c["gammas"]:
        gammas.append(NO_BUFFER if g is None else BufferRef(len(arrays)))
        if g is not None:
            arrays.append(g)
    call = KernelCall.QkNormRotary(QkNormRotaryCall(
        BufferRef(0, pad * es), BufferRef(0, (pad + H * D) * es) if Hkv else NO_BUFFER, *gammas, BufferRef(1),
        BufferRef(2), BufferRef(3) if c["rot"] else NO_BUFFER, BufferRef(4), BufferRef(5) if Hkv else NO_BUFFER,
        tokens, len(c["rows"]), H, Hkv, D, c["rot"], width, width, bits(EPS),
        bits(c["magnitude"]) if c["magnitude"] else 0, c["norms"], c["interleaved"], c["dtype"]))
    _, ts = dispatch(torch, backend, call, arrays)
    return [from_dev(ts[4 + i], f.dtype).reshape(f.shape) for i, f in enumerate(fills)]


def check_rotary(got, c):
    dtype, H, Hkv, D, pad, gap = (c[x] for x in ("dtype", "H", "Hkv", "D", "pad", "gap"))
    x = decode(c["qkv"], dtype).reshape(c["qkv"].shape)
    n = sum(c["rows"])
    at = np.concatenate([int(p) + np.arange(r) for p, r in zip(c["pos"], c["rows"])]).astype(np.int64)
    for i, (h, off) in enumerate(((H, pad), (Hkv, pad + H * D))):
        if h == 0:
            assert (got[i] == 7).all()
            continue
        rows = x[gap:gap + n, off:off + h * D].reshape(n, h, D)
        gamma = c["gammas"][i]
        want, tol = rotary(rows, None if gamma is None else decode(gamma, dtype),
                           EPS if c["norms"] >> i & 1 else None, at, c["freqs"], c["rot"], c["interleaved"],
                           c["magnitude"] or 1.0, dtype)
        err = np.abs(decode(got[i][gap:gap + n], dtype).reshape(want.shape) - want)
        assert (err <= tol).all(), (i, float((err / tol).max()))
        assert (got[i][:gap] == 7).all() and (got[i][gap + n:] == 7).all()


SHAPES = [  # rows, pos, H, Hkv, D, rot, pad
    ([1], [0], 1, 1, 64, 64, 0),
    ([1] * 5, [0, 9, 1000, 131071, 77], 32, 8, 128, 128, 0),
    ([3, 0, 17, 1], [5, 0, 0, 40], 8, 2, 128, 64, 8),       # part of the head, an empty sequence
    ([70, 33], [0, 2000], 6, 2, 96, 96, 0),
    ([9], [3], 5, 5, 80, 32, 16),
    ([20, 2], [100, 7], 2, 1, 256, 256, 0),
    ([5, 6], [1, 2], 3, 1, 64, 6, 0),                       # pairs that are no whole 16 bytes
    ([5, 6], [1, 2], 3, 1, 64, 64, 1),                      # the wide form's sizes, rows off 16 bytes
    ([2], [1], 100, 4, 128, 128, 0),                        # several passes a token
    ([2], [1], 33000, 33000, 16, 16, 0),                    # more passes than workgroups share
    ([4, 4], [8, 9], 2, 2, 37, 20, 1),                      # nothing aligned, an odd head
    ([6], [50], 2, 1, 1024, 1024, 0),
    ([6], [50], 1, 1, 1000, 500, 0),
    ([2], [1], 2, 1, 16, 16, 0),
    ([2], [1], 2, 1, 2, 2, 0),
    ([3], [1], 2, 1, 1, 0, 0),                              # no rotation
    ([40], [9], 4, 2, 128, 0, 0),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("rows,pos,H,Hkv,D,rot,pad", SHAPES)
def test_rotary_parity(torch_cuda, backend, rows, pos, H, Hkv, D, rot, pad, interleaved, dtype):
    rng = np.random.default_rng(D + rot + sum(rows))
    c = rotary_case(rng, rows, pos, H, Hkv, D, rot, dtype, 3, interleaved, pad, gap=2, tail=3)
    check_rotary(run_rotary(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (72, 10)])
@pytest.mark.parametrize("norms,gammas", [(0, (True, True)), (1, (False, True)), (2, (True, False)), (3, (False, False))])
def test_norms_and_gammas(torch_cuda, backend, norms, gammas, D, rot, dtype):
    rng = np.random.default_rng(norms)
    c = rotary_case(rng, [5, 2], [3, 60], 6, 2, D, rot, dtype, norms, 0, magnitude=1.25, gammas=gammas)
    if norms == 0:
        c["gammas"] = [None, None]
    check_rotary(run_rotary(torch_cuda, backend, c), c)


def test_a_gamma_whose_norm_is_off_is_not_read(torch_cuda, backend):
    rng = np.random.default_rng(1)
    c = rotary_case(rng, [5], [3], 4, 2, 64, 64, DTYPE_F32, 0)
    c["gammas"] = [encode(np.full(64, np.nan), DTYPE_F32)] * 2
    got = run_rotary(torch_cuda, backend, c)
    c["gammas"] = [None, None]
    for a, b in zip(got, run_rotary(torch_cuda, backend, c)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [128, 72])
def test_queries_alone(torch_cuda, backend, D, dtype):
    rng = np.random.default_rng(2)
    c = rotary_case(rng, [7, 1], [3, 60], 6, 0, D, D // 2, dtype)
    check_rotary(run_rotary(torch_cuda, backend, c), c)


@pytest.mark.parametrize("D", [128, 36])
def test_far_positions_keep_their_angles(torch_cuda, backend, D):
    """Positions up to the last of 32 bits, frequencies from a radian a position down: f32's
    precision throughout (an angle taken in f32 would be off by radians)."""
    rng = np.random.default_rng(3)
    pos = [0, 4095, 1 << 20, (1 << 24) + 1, 0x7FFFFFFF, 0xFFFFFFF0]
    c = rotary_case(rng, [3] * 6, pos, 2, 1, D, D, DTYPE_F32, 0)
    check_rotary(run_rotary(torch_cuda, backend, c), c)
    c["freqs"] = (c["freqs"] * 1000.0).astype(np.float32)      # many turns a position
    check_rotary(run_rotary(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [128, 36])
def test_a_row_that_is_not_finite_stays_alone(torch_cuda, backend, D, dtype):
    """A NaN or infinity reaches its own head's row and no other; so do zero rows (their norm is
    the epsilon's)."""
    rng = np.random.default_rng(4)
    c = rotary_case(rng, [9], [3], 4, 2, D, D, dtype)
    x = decode(c["qkv"], dtype).reshape(c["qkv"].shape).copy()
    x[7, :D] = 0.0
    c["qkv"] = encode(x, dtype).reshape(x.shape)
    clean = run_rotary(torch_cuda, backend, c)
    check_rotary(clean, c)
    assert (clean[0][7, 0] == 0).all() or (decode(clean[0][7, 0], dtype) == 0).all()
    x[2, D + 3], x[5, 4 * D + 1] = np.nan, np.inf              # head 1 of row 2, k head 0 of row 5
    c["qkv"] = encode(x, dtype).reshape(x.shape)
    got = run_rotary(torch_cuda, backend, c)
    for i, (row, head) in enumerate(((2, 1), (5, 0))):
        other = np.ones(got[i].shape[:2], bool)
        other[row, head] = False
        assert np.array_equal(got[i][other], clean[i][other])
        assert np.isnan(decode(got[i][row, head], dtype)).any()


def test_many_sequences(torch_cuda, backend):
    rng = np.random.default_rng(5)
    rows = list(rng.integers(0, 4, 300))
    c = rotary_case(rng, rows, rng.integers(0, 100000, 300), 4, 2, 64, 64, DTYPE_BF16, gap=1, tail=2)
    check_rotary(run_rotary(torch_cuda, backend, c), c)


def test_many_rows(torch_cuda, backend):
    """More tokens than a workgroup takes, by far, and not a multiple of what one does."""
    rng = np.random.default_rng(6)
    for dtype, D in ((DTYPE_BF16, 128), (DTYPE_F32, 80), (DTYPE_F16, 64)):
        c = rotary_case(rng, [2001, 1, 1500], [7, 0, 100], 5, 1, D, D, dtype, gap=3, tail=2)
        check_rotary(run_rotary(torch_cuda, backend, c), c)


@pytest.mark.parametrize("D", [64, 36])
@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [0, 5, 9, 21], [2**32 - 1, 0, 3, 20], [20, 0, 20, 0]])
def test_bad_offsets_are_reported(torch_cuda, backend, starts, D):
    c = rotary_case(np.random.default_rng(0), [9, 5, 6], [1, 2, 3], 4, 2, D, D, DTYPE_BF16)
    c["starts"] = np.array(starts, np.uint32)
    with pytest.raises(SlotOutOfRange):
        run_rotary(torch_cuda, backend, c)
    backend.synchronize()


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("D", [128, 36])
def test_positions_past_32_bits(torch_cuda, backend, D, interleaved):
    """A position is pos[b] + t, also where the sum passes 32 bits."""
    rng = np.random.default_rng(D)
    c = rotary_case(rng, [5, 40, 3], [0xFFFFFFFE, 0xFFFFFFFF, 0xFFFFFFF0], 2, 1, D, D, DTYPE_F32, 0, interleaved)
    check_rotary(run_rotary(torch_cuda, backend, c), c)
