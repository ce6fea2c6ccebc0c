"""The labels of the packed-batch calls (126-129): calls that read or write other parts of the same
slots, or leave other operands out, are other values."""
from dataclasses import fields, replace

import pytest

from hologram_amd import (DTYPE_BF16, DTYPE_F32, DTYPE_I32, NO_BUFFER, ArgMaxCall, BufferRef,
                          HipSession, HoloWriter, KernelCall, LogitsProcessCall, PortDescriptor)
from hologram_amd.kappa import address_bytes, op_signature
from test_packed_batch import CALLS

ROWS, COLS = 3, 500


@pytest.mark.parametrize("make,c,sizes", CALLS)
def test_where_each_operand_starts_is_part_of_the_signature(make, c, sizes):
    seen = {op_signature(make(c))}
    refs = [f.name for f in fields(c) if isinstance(getattr(c, f.name), BufferRef)]
    assert len(refs) >= 5
    for name in refs:
        for offset in (64, 128, 1 << 40):
            seen.add(op_signature(make(replace(c, **{name: BufferRef(getattr(c, name).slot, offset)}))))
    assert len(seen) == 1 + 3 * len(refs)


def test_which_operands_the_logits_rules_use_is_part_of_the_signature():
    c = CALLS[3][1]
    none = dict(history=NO_BUFFER, spans=NO_BUFFER, params=NO_BUFFER, history_len=0, bias_ids=NO_BUFFER,
                bias_values=NO_BUFFER, biases=0, mask=NO_BUFFER)
    # one other label in the call's list of them: a mask, or a history of length 0
    a = op_signature(KernelCall.LogitsProcess(replace(c, **{**none, "mask": BufferRef(6)})))
    b = op_signature(KernelCall.LogitsProcess(replace(c, **{**none, "history": BufferRef(6)})))
    assert a != b


def two_halves():
    """Rules on the first and on the second half of one slot of logits, picked apart."""
    w = HoloWriter()
    half = ROWS * COLS * 2
    w.inputs = [PortDescriptor("logits", 0, 2 * ROWS * COLS, DTYPE_BF16, [2 * ROWS, COLS]),
                PortDescriptor("ids", 1, ROWS, DTYPE_I32, [ROWS]),
                PortDescriptor("values", 2, ROWS, DTYPE_F32, [ROWS])]
    w.outputs = [PortDescriptor(f"picks{i}", 5 + i, ROWS, DTYPE_I32, [ROWS]) for i in range(2)]
    for i in range(2):
        w.kernel_calls.append(KernelCall.LogitsProcess(LogitsProcessCall(
            BufferRef(0, i * half, half), NO_BUFFER, NO_BUFFER, NO_BUFFER, BufferRef(1, 0, ROWS * 4),
            BufferRef(2, 0, ROWS * 4), NO_BUFFER, BufferRef(3 + i, 0, half), ROWS, COLS, 0, 1, DTYPE_BF16)))
        w.kernel_calls.append(KernelCall.ArgMax(ArgMaxCall(
            BufferRef(3 + i, 0, half), BufferRef(5 + i, 0, ROWS * 4), ROWS, COLS, DTYPE_BF16)))
    w.exec_plan = [[0, 2], [1, 3]]
    return w.finish()


def test_a_session_takes_two_views_for_two_values():
    s = HipSession(None, two_halves())
    assert s.n_nodes == 4              # neither half's rules stand in for the other's
    labels = s.output_labels([address_bytes(bytes([i])) for i in range(3)])
    assert labels[0] != labels[1]
