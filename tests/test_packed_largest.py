"""The packed-batch calls (126-129) whose launch would hold 2^32 threads or more are refused, and the
ones just below are taken."""
from dataclasses import replace

import pytest

from hologram_amd import (DTYPE_BF16, DTYPE_F32, NO_BUFFER, AttentionI8BlocksCall, AttentionPackedCall,
                          BufferRef, KernelCall, KvBlockAppendCall, LogitsProcessCall, UnsupportedOp,
                          validate)

R = [BufferRef(i) for i in range(8)]
ROWS = AttentionPackedCall(*R[:5], (1 << 20) - 1, (1 << 20) - 1, 64, 64, 1, 0, 0, 0, 0, DTYPE_BF16)
APPEND = KvBlockAppendCall(*R[:5], R[3], R[4], (1 << 22) - 3, 1, 4, 1 << 22, 1, 1, 0, DTYPE_BF16)
LOGITS = LogitsProcessCall(R[0], NO_BUFFER, NO_BUFFER, NO_BUFFER, R[1], R[2], NO_BUFFER, R[3],
                           (1 << 23) - 1, 4, 0, 1, DTYPE_F32)
TILES = AttentionPackedCall(*R[:5], 8, (1 << 21) - 1, 8, 8, 8, 0, 0, 0, 0, DTYPE_BF16)
CACHE_ROWS = AttentionI8BlocksCall(*R, (1 << 20) - 1, 1, 64, 64, 64, 10, 5, 0, 0, DTYPE_BF16)
CACHE_TILES = AttentionI8BlocksCall(*R, 8, (1 << 21) - 1, 8, 8, 16, 16, 16, 0, 0, DTYPE_BF16)


@pytest.mark.parametrize("make,c,past", [
    (KernelCall.AttentionPacked, ROWS, dict(tokens=1 << 20)),
    (KernelCall.AttentionPacked, TILES, dict(batch=1 << 21)),
    (KernelCall.AttentionPacked, replace(TILES, dtype=DTYPE_F32), dict(batch=1 << 21)),
    (KernelCall.AttentionPacked, replace(TILES, dtype=DTYPE_F32, head_dim=132, batch=(1 << 22) - 1),
     dict(batch=1 << 22)),
    (KernelCall.KvBlockAppend, APPEND, dict(tokens=(1 << 22) - 2)),
    (KernelCall.AttentionI8Blocks, CACHE_ROWS, dict(tokens=1 << 20)),
    (KernelCall.AttentionI8Blocks, CACHE_TILES, dict(batch=1 << 21)),
    (KernelCall.LogitsProcess, LOGITS, dict(rows=1 << 23)),
    (KernelCall.LogitsProcess, replace(LOGITS, rows=(1 << 22) - 1, cols=8190), dict(rows=1 << 22)),
])
def test_the_largest_launches(make, c, past):
    sizes = [1 << 40] * 8
    validate(make(c), sizes)
    with pytest.raises(UnsupportedOp, match="one launch"):
        validate(make(replace(c, **past)), sizes)
