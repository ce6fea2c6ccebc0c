"""The long-context calls where offsets pass 32 bits, and lists of more rows than one pass of the
scratch takes: the same bits as the same rows in small operands."""
import numpy as np
import pytest

from hologram_amd import (DTYPE_BF16, NO_BUFFER, AttentionI8SelectedCall, BufferRef, DeviceWorkspace,
                          KernelCall, KvBlockBoundsCall, KvBlockSelectCall, QkNormRotaryCall)
from long_context_reference import select_blocks
from packed_reference import decode

pytestmark = pytest.mark.gpu
R = BufferRef


def dispatch(backend, call, tensors):
    ws = DeviceWorkspace()
    for s, t in enumerate(tensors):
        ws.bind(s, t)
    backend.dispatch(call, ws)
    backend.synchronize()


def u32(torch, values):
    return torch.tensor(values, dtype=torch.int64, device="cuda").to(torch.int32)


@pytest.mark.parametrize("D,tokens", [(256, 140_003), (320, 110_001)])
def test_rotary_rows_past_four_gigabytes(torch_cuda, backend, D, tokens):
    torch = torch_cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(D)
    H = 64
    x = torch.zeros((tokens, H * D), dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn((3, H * D), generator=g, device="cuda").to(torch.bfloat16)
    out, small = torch.zeros_like(x), torch.zeros((3, H * D), dtype=torch.bfloat16, device="cuda")
    assert (x.numel() - 3 * H * D) * 2 > 1 << 32
    freqs = torch.rand(D // 2, generator=g, device="cuda")

    def call(n):
        return KernelCall.QkNormRotary(QkNormRotaryCall(R(0), NO_BUFFER, NO_BUFFER, NO_BUFFER, R(1), R(2), R(3),
                                                        R(4), NO_BUFFER, n, 1, H, 0, D, D, norms=1))
    dispatch(backend, call(tokens), [x, u32(torch, [0, tokens]), u32(torch, [7]), freqs, out])
    dispatch(backend, call(3), [x[-3:].contiguous(), u32(torch, [0, 3]), u32(torch, [tokens + 4]), freqs, small])
    assert torch.equal(out[-3:], small) and small.abs().sum() > 0


@pytest.mark.parametrize("D", [256, 320])
def test_bounds_and_attention_past_four_gigabytes(torch_cuda, backend, D):
    """The last of five planes of a gigabyte: rows at its end appended, and a list over all of it."""
    torch = torch_cuda
    rng = np.random.default_rng(D)
    block, B = 4096, 5
    bucket = (1 << 30) // D // block * block
    nb = bucket // block
    k, v = (torch.zeros((B, bucket, D), dtype=torch.int8, device="cuda") for _ in "kv")
    assert (B - 1) * bucket * D >= 1 << 31 and k.numel() > 1 << 32
    ids = [1, 77, nb - 2, nb - 1]
    sk, sv = (torch.from_numpy(rng.integers(-127, 128, (len(ids) * block, D), dtype=np.int8)).cuda() for _ in "kv")
    for big, little in ((k, sk), (v, sv)):
        for i, j in enumerate(ids):
            big[B - 1, j * block:(j + 1) * block] = little[i * block:(i + 1) * block]
    bounds = torch.zeros((B, nb, 2, D), dtype=torch.int8, device="cuda")
    n, rows = 5000, [0, 0, 0, 0, 5000]
    starts = u32(torch, np.concatenate([[0], np.cumsum(rows)]).tolist())
    dispatch(backend, KernelCall.KvBlockBounds(KvBlockBoundsCall(R(0), R(1), R(2), R(3), R(3), n, B, 1, bucket, block, D)),
             [k, starts, u32(torch, [0, 0, 0, 0, bucket - n]), bounds])
    at = (bucket - n) // block
    assert at == nb - 2
    for j, i in ((nb - 2, 2), (nb - 1, 3)):
        x = sk[i * block:(i + 1) * block]
        assert torch.equal(bounds[B - 1, j, 0], x.amin(0)) and torch.equal(bounds[B - 1, j, 1], x.amax(0))
    assert not bounds[:B - 1].any() and not bounds[B - 1, :nb - 2].any()
    H = 4
    q = torch.randn((1, H * D), device="cuda").to(torch.bfloat16)
    scales = torch.full((B, nb), 2.0 ** -8, device="cuda")
    out, small = torch.zeros_like(q), torch.zeros_like(q)

    def call(batch, bucket):
        return KernelCall.AttentionI8Selected(AttentionI8SelectedCall(*[R(s) for s in range(9)], 1, batch, H, 1, bucket,
                                                                      block, D, 0, len(ids)))
    listed = torch.tensor(ids, dtype=torch.int32, device="cuda")
    dispatch(backend, call(B, bucket), [q, k, v, scales, scales, listed, u32(torch, [0, 0, 0, 0, 0, 1]),
                                        u32(torch, [0, 0, 0, 0, bucket]), out])
    dispatch(backend, call(1, len(ids) * block), [q, sk, sv, scales[0, :len(ids)].contiguous(),
                                                  scales[0, :len(ids)].contiguous(), torch.arange(4, dtype=torch.int32, device="cuda"),
                                                  u32(torch, [0, 1]), u32(torch, [len(ids) * block]), small])
    assert torch.equal(out, small) and small.abs().sum() > 0


@pytest.mark.parametrize("D", [256, 320])
def test_lists_past_four_gigabytes_of_bounds(torch_cuda, backend, D):
    torch = torch_cuda
    rng = np.random.default_rng(D)
    B, nb, block, H, top = 10, 1 << 20, 4, 4, 50
    bounds = torch.zeros((B, nb, 2, D), dtype=torch.int8, device="cuda")
    assert (B - 1) * nb * 2 * D > 1 << 32
    some = 3000
    x = np.sort(rng.integers(-128, 128, (some, 2, D), dtype=np.int8), axis=1)
    bounds[B - 1, :some] = torch.from_numpy(x).cuda()
    ks = torch.zeros((B, nb), device="cuda")
    s = rng.uniform(0.5, 1.0, some).astype(np.float32)
    ks[B - 1, :some] = torch.from_numpy(s).cuda()
    q = torch.randn((1, H * D), device="cuda").to(torch.bfloat16)
    out = torch.zeros((1, 1, top), dtype=torch.int32, device="cuda")
    dispatch(backend, KernelCall.KvBlockSelect(KvBlockSelectCall(
        *[R(s) for s in range(6)], 1, B, H, 1, nb * block, block, D, 0, top, 1, 1)),
        [q, bounds, ks, u32(torch, [0] * B + [1]), u32(torch, [0] * (B - 1) + [some * block]), out])
    qn = decode(q.view(torch.int16).cpu().numpy(), DTYPE_BF16).reshape(1, H, D)
    want = select_blocks(qn, x[None, None], s[None, None], [some * block], [1], 1, some * block, block, top, 1, 1)
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("D", [16, 20])
def test_lists_of_more_rows_than_a_pass(torch_cuda, backend, D):
    """35000 blocks a row: the sums of 1917 rows fill the scratch, the rest is another pass; the rows
    about the border are checked."""
    torch = torch_cuda
    rng = np.random.default_rng(D)
    n, nb, block, top = 2100, 35_000, 2, 300
    x = np.sort(rng.integers(-128, 128, (nb, 2, D), dtype=np.int8), axis=1)
    s = rng.uniform(0.5, 1.0, nb).astype(np.float32)
    q = torch.randn((n, D), device="cuda").to(torch.bfloat16)
    out = torch.zeros((n, 1, top), dtype=torch.int32, device="cuda")
    dispatch(backend, KernelCall.KvBlockSelect(KvBlockSelectCall(
        *[R(s) for s in range(6)], n, 1, 1, 1, nb * block, block, D, 0, top, 2, 3)),
        [q, torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), u32(torch, [0, n]), u32(torch, [nb * block]), out])
    qn = decode(q.view(torch.int16).cpu().numpy(), DTYPE_BF16).reshape(n, 1, D)
    got = out.cpu().numpy()
    for t in (0, 1, 15, 16, 1900, 1915, 1916, 1917, 1918, 1935, n - 2, n - 1):
        want = select_blocks(qn[t:t + 1], x[None, None], s[None, None], [nb * block - (n - 1 - t)], [1], 1, nb * block,
                             block, top, 2, 3)
        assert np.array_equal(got[t:t + 1], want), t
