"""The largest launches of 126, 127 and 129, of the smallest rows."""
import pytest

from hologram_amd import DeviceWorkspace, KernelCall
from test_packed_largest import APPEND, LOGITS, ROWS

pytestmark = pytest.mark.gpu


def run(backend, call, tensors):
    ws = DeviceWorkspace()
    for slot, t in enumerate(tensors):
        ws.bind(slot, t)
    backend.dispatch(call, ws)
    backend.synchronize()


def test_attention_of_as_many_rows_as_a_launch_holds(torch_cuda, backend):
    """One row a sequence: the result is its V."""
    torch, n = torch_cuda, ROWS.tokens
    q, k, v = (torch.randn(n * 64, device="cuda").to(torch.bfloat16) for _ in range(3))
    starts = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    run(backend, KernelCall.AttentionPacked(ROWS), [q, k, v, starts, out])
    assert torch.equal(out, v)


def test_append_of_as_many_blocks_as_a_launch_holds(torch_cuda, backend):
    """One element a block: it is 64 to 127 of its own power of two."""
    torch, n = torch_cuda, APPEND.tokens
    new = torch.randn(n * 4, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    cache = torch.full((4 << 22,), 5, dtype=torch.int8, device="cuda")
    scales = torch.full((4 << 22,), 2.0, device="cuda")
    run(backend, KernelCall.KvBlockAppend(APPEND), [new, starts, pos, cache, scales])
    q, s = cache.view(4, 1 << 22), scales.view(4, 1 << 22)
    got = (q.float() * s)[:, 3:]
    want = new.float().view(n, 4).T
    # a bf16 of 8 bits in a step of 2^-6 to 2^-7 of itself: half a step at most
    assert ((got - want).abs() <= want.abs() * 2.0 ** -7).all()
    assert (q[:, :3] == 5).all() and (s[:, :3] == 2.0).all()


def test_rules_on_as_many_rows_as_a_launch_holds(torch_cuda, backend):
    torch, n = torch_cuda, LOGITS.rows
    x = torch.randn(n, 4, device="cuda")
    ids = torch.arange(n, dtype=torch.int32, device="cuda") % 5        # (4: no column)
    values = torch.randn(n, device="cuda")
    out = torch.zeros_like(x)
    run(backend, KernelCall.LogitsProcess(LOGITS), [x, ids, values, out])
    want = x.clone()
    rows = torch.arange(n, device="cuda")[ids < 4]
    at = ids[ids < 4].long()
    want[rows, at] = x[rows, at] + values[rows]
    assert torch.equal(out, want)
