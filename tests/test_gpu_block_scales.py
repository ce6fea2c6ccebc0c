"""AttentionI8Blocks (128) over caches whose V scales are zero, far apart, tiny or not finite, in
each of its forms, against 64 bits."""
import numpy as np
import pytest

from hologram_amd import DTYPE_BF16, DTYPE_F16, DTYPE_F32
from packed_reference import ALL, attend, bound, decode
from test_gpu_packed_batch import blocks_case, run_blocks

pytestmark = pytest.mark.gpu

# half the least step of the result's type
FLOOR = {DTYPE_BF16: 2.0 ** -134, DTYPE_F16: 2.0 ** -25, DTYPE_F32: 2.0 ** -150}
# rows of each of two sequences, their lengths, the bucket: a unit a workgroup, shares of units, row
# tiles whole, row tiles cut
FORMS = [(1, [400, 90], 400), (1, [2500, 90], 2512), (80, [400, 90], 400), (80, [4000, 300], 4000)]


def make(rng, n, lens, bucket, dtype, D=64):
    return blocks_case(rng, [n, n], lens, 4, 2, D, bucket, 16, dtype)


def check(got, c):
    """Within packed_reference's bound and half a least step of the type."""
    dtype, H, Hkv, D = c["dtype"], c["H"], c["Hkv"], c["D"]
    q = decode(c["q"], dtype).reshape(c["q"].shape)[:, c["pad"]:].reshape(-1, H, D)
    at = 0
    for b, n in enumerate(c["rows"]):
        keys = np.clip(int(c["lens"][b]) - (n - 1 - np.arange(n)), 0, c["bucket"])
        of = np.arange(int(keys.max())) // c["block"]
        k, v = ((c[x][b, :, :len(of)].astype(np.float64) * c[x + "s"][b][:, of, None].astype(np.float64))
                .transpose(1, 0, 2) for x in "kv")
        want, slack, top = attend(q[at:at + n], k, v, keys, H, Hkv, np.sqrt(D))
        err = np.abs(decode(got[at:at + n], dtype).reshape(want.shape) - want)
        tol = bound(slack, top, dtype) + FLOOR[dtype]
        assert (err <= tol).all(), (b, float(np.nanmax(err / tol)))
        at += n


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("exponent", [-13, -20, -24, -34, -40])
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_a_zero_v_scale_costs_the_other_blocks_nothing(torch_cuda, backend, n, lens, bucket, exponent, dtype):
    """A block of zeros, as KvBlockAppend writes it (scale 0), among blocks of one small scale."""
    c = make(np.random.default_rng(-exponent), n, lens, bucket, dtype)
    c["vs"][:] = 2.0 ** exponent
    c["vs"][:, :, 3] = 0.0
    c["vs"][1, 0, 0] = -0.0
    check(run_blocks(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("few", [[-149, -126, -6, 8], [-149], [-126], [-60, 8]])
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_far_apart_v_scales(torch_cuda, backend, n, lens, bucket, few, dtype):
    """Scales whose ratio passes what f32 holds: the keys of the small ones weigh in the softmax like
    any other. (The first block's is ordinary, so every row that sees a key sees a value to measure
    by.)"""
    rng = np.random.default_rng(sum(few) + 1000)
    c = make(rng, n, lens, bucket, dtype)
    c["vs"] = np.ldexp(1.0, rng.choice(few, c["vs"].shape)).astype(np.float32)
    c["vs"][:, :, 0] = 2.0 ** 8 if max(few) == 8 else 2.0 ** -6
    check(run_blocks(torch_cuda, backend, c), c)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_a_zero_v_scale_is_a_block_of_zeros(torch_cuda, backend, n, lens, bucket, dtype):
    """The same bits whichever of the two says so."""
    c = make(np.random.default_rng(n), n, lens, bucket, dtype)
    c["vs"][:] = 2.0 ** -9
    by_scale = {**c, "vs": c["vs"].copy()}
    by_scale["vs"][:, :, 3] = 0.0
    by_bytes = {**c, "v": c["v"].copy()}
    by_bytes["v"][:, :, 48:64] = 0
    assert np.array_equal(run_blocks(torch_cuda, backend, by_scale), run_blocks(torch_cuda, backend, by_bytes))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_an_infinite_v_scale(torch_cuda, backend, n, lens, bucket, dtype):
    """Infinity times the bytes: infinite of their sign in a dim where all are of one, NaN where some
    are zero, for the rows that see a key of the block; the rest as it was. (Q is small, so that no
    weight is 0.)"""
    c = make(np.random.default_rng(n), n, lens, bucket, dtype)
    c["q"] = np.zeros_like(c["q"])
    block = (lens[0] - 1 - n // 2) // 16        # half of the first sequence's rows see some of it
    clean = decode(run_blocks(torch_cuda, backend, c), dtype).reshape(2 * n, 4, 64)
    c["v"][0, 0, 16 * block:16 * block + 16] = np.array([3, -5, 0, 1], np.int8)[np.arange(64) % 4]
    plain = decode(run_blocks(torch_cuda, backend, c), dtype).reshape(2 * n, 4, 64)
    c["vs"][0, 0, block] = np.inf
    got = decode(run_blocks(torch_cuda, backend, c), dtype).reshape(2 * n, 4, 64)
    keys = np.concatenate([lens[0] - (n - 1 - np.arange(n)), np.zeros(n, int)])
    sees = keys > 16 * block
    assert sees.any()
    assert np.array_equal(got[~sees], plain[~sees]) and np.array_equal(got[:, 2:], clean[:, 2:])
    want = np.array([np.inf, -np.inf, np.nan, np.inf])[np.arange(64) % 4]
    assert np.array_equal(got[sees][:, :2], np.broadcast_to(want, (sees.sum(), 2, 64)), equal_nan=True)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_a_nan_v_scale(torch_cuda, backend, n, lens, bucket, dtype):
    """Every dim of the rows that see a key of the block is NaN, whatever its bytes."""
    c = make(np.random.default_rng(n), n, lens, bucket, dtype)
    block = (lens[0] - 1 - n // 2) // 16
    clean = run_blocks(torch_cuda, backend, c)
    c["v"][0, 0, 16 * block:16 * block + 16] = 0
    plain = run_blocks(torch_cuda, backend, c)
    c["vs"][0, 0, block] = np.nan
    got = run_blocks(torch_cuda, backend, c)
    sees = np.concatenate([lens[0] - (n - 1 - np.arange(n)), np.zeros(n, int)]) > 16 * block
    assert np.array_equal(got[~sees], plain[~sees]) and np.array_equal(got[:, 2:], clean[:, 2:])
    assert np.isnan(decode(got[sees][:, :2], dtype)).all()


@pytest.mark.parametrize("dtype", [DTYPE_BF16, DTYPE_F32])
@pytest.mark.parametrize("exponent", [-140, -126, -110, 100])
@pytest.mark.parametrize("n,lens,bucket", FORMS)
def test_v_scales_at_the_ends_of_f32(torch_cuda, backend, n, lens, bucket, exponent, dtype):
    """2^-126 is the least scale that KvBlockAppend writes; 2^-140 a subnormal."""
    c = make(np.random.default_rng(200 + exponent), n, lens, bucket, dtype)
    c["vs"][:] = 2.0 ** exponent
    check(run_blocks(torch_cuda, backend, c), c)


@pytest.mark.parametrize("B,n,H,Hkv,bucket", [
    (20, 4, 64, 8, 128),          # a unit a workgroup
    (100, 2, 64, 8, 1040),        # shares of units
    (16, 128, 16, 2, 128),        # row tiles whole
    (2, 200, 16, 2, 4000),        # row tiles cut
])
def test_f32_weights_keep_both_their_parts(torch_cuda, backend, B, n, H, Hkv, bucket):
    """f32 rows against a bound without the scores' sums: q has one element, so a score is a product.
    The 16-bit halves of a weight make it up to 2^-22 of itself, in every one of many rows whose few
    largest weights are most of their sum."""
    rng = np.random.default_rng(B + n)
    D, dtype = 64, DTYPE_F32
    c = blocks_case(rng, [n] * B, [min(bucket, 128 + 7 * b) for b in range(B)] if bucket != 4000 else [4000, 900],
                    H, Hkv, D, bucket, 16, dtype, "any")
    c["q"][:] = 0.0
    c["q"][:, ::D] = rng.standard_normal((n * B, H)) * 30
    got = run_blocks(torch_cuda, backend, c)
    q = c["q"].astype(np.float64).reshape(B, n, Hkv, H // Hkv, D)[..., 0]
    got = got.astype(np.float64).reshape(B, n, Hkv, H // Hkv, D)
    of = np.arange(bucket) // 16
    for b in range(B):
        keys = int(c["lens"][b]) - (n - 1 - np.arange(n))
        k, v = (c[x][b].astype(np.float64) * c[x + "s"][b][:, of, None].astype(np.float64) for x in "kv")
        for kh in range(Hkv):
            s = q[b, :, kh, :, None] * k[kh, :, 0] / np.sqrt(D)
            s = np.where(np.arange(bucket) < keys[:, None, None], s, -np.inf)
            p = np.exp(s - s.max(2, keepdims=True))
            want = p @ v[kh] / p.sum(2, keepdims=True)
            # the score's five roundings; exp2's argument and result, a weight's product and second
            # part; the sums of keys that are not negligible, in f32, each by each
            size = np.abs(np.where(np.isfinite(s), s, 0)).max(2, keepdims=True)
            many = (p > 2.0 ** -24).sum(2, keepdims=True)
            tol = (2 * 5 * 2.0 ** -24 * size + 2.0 ** -21 + 2 * (many + 8) * 2.0 ** -24) * np.abs(v[kh]).max()
            err = np.abs(got[b, :, kh] - want)
            assert (err <= tol).all(), (b, kh, float((err / tol).max()))
