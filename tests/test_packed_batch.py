"""The packed-batch calls (126-129) on the host: the codec, the C layouts' packed form, the op
signatures, the refusals, and a dry load of a graph that holds them."""
import struct
from dataclasses import replace

import numpy as np
import pytest

from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, DTYPE_I32, NO_BUFFER, ArgMaxCall,
                          AttentionI8BlocksCall, AttentionPackedCall, BufferRef, HipSession,
                          HoloWriter, KernelCall, KvBlockAppendCall, LogitsProcessCall,
                          PortDescriptor, ShapeMismatch, SlotOutOfRange, UnsupportedOp, decode_call,
                          validate)
from hologram_amd import kernel_call as kc
from hologram_amd.kappa import op_signature
from packed_reference import block_append, encode

R = BufferRef
PACKED = AttentionPackedCall(R(0), R(1), R(2), R(3), R(4), 10, 3, 8, 2, 64, 0, 0, 0, 0, DTYPE_BF16)
PACKED_SIZES = [10 * 8 * 64 * 2, 10 * 2 * 64 * 2, 10 * 2 * 64 * 2, 16, 10 * 8 * 64 * 2]
APPEND = KvBlockAppendCall(R(0), R(1), R(2), R(3), R(4), R(3), R(4), 10, 3, 2, 100, 32, 64, 0,
                           DTYPE_F32)
APPEND_SIZES = [10 * 2 * 64 * 4, 16, 12, 6 * 100 * 64, 6 * 4 * 4]
BLOCKS = AttentionI8BlocksCall(R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), 10, 3, 8, 2, 100,
                               32, 64, 0, 0, DTYPE_F16)
BLOCKS_SIZES = [10 * 8 * 64 * 2, 6 * 100 * 64, 6 * 100 * 64, 6 * 4 * 4, 6 * 4 * 4, 16, 12,
                10 * 8 * 64 * 2]
LOGITS = LogitsProcessCall(R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), 4, 1000, 50, 7,
                           DTYPE_BF16)
LOGITS_SIZES = [8000, 4 * 50 * 4, 32, 48, 4 * 7 * 4, 4 * 7 * 4, 4 * 32 * 4, 8000]
CALLS = [(KernelCall.AttentionPacked, PACKED, PACKED_SIZES),
         (KernelCall.KvBlockAppend, APPEND, APPEND_SIZES),
         (KernelCall.AttentionI8Blocks, BLOCKS, BLOCKS_SIZES),
         (KernelCall.LogitsProcess, LOGITS, LOGITS_SIZES)]


@pytest.mark.parametrize("make,c,sizes", CALLS)
def test_codec_and_validation(make, c, sizes):
    call = make(c)
    wire = call.encode()
    got, used = decode_call(wire + b"\xff")
    assert used == len(wire) and bytes(got) == bytes(call.to_c()) == kc.dispatch_form(call)
    assert struct.unpack_from("<H", wire)[0] == call.tag and call.name in make.__qualname__
    op, params = op_signature(call)
    assert op == call.tag and 0 < len(params) <= 64
    validate(call, sizes)
    for i in range(len(sizes)):      # any operand a byte short is refused, and says which
        with pytest.raises(SlotOutOfRange):
            validate(call, [n - (j == i) for j, n in enumerate(sizes)])
        with pytest.raises(SlotOutOfRange):
            validate(call, sizes[:i])


def test_signatures_tell_views_of_one_operand_apart():
    a, b = (op_signature(KernelCall.AttentionPacked(replace(PACKED, k=R(1, off)))) for off in (0, 128))
    assert a != b
    a, b = (op_signature(KernelCall.KvBlockAppend(replace(APPEND, new=R(0, off)))) for off in (0, 128))
    assert a != b


@pytest.mark.parametrize("make,c,sizes,change,error", [
    (*CALLS[0], dict(heads=7), UnsupportedOp), (*CALLS[0], dict(dtype=2), UnsupportedOp),
    (*CALLS[0], dict(head_dim=1025), UnsupportedOp), (*CALLS[0], dict(q_stride=511), ShapeMismatch),
    (*CALLS[0], dict(k_stride=127), ShapeMismatch), (*CALLS[0], dict(v_stride=1), ShapeMismatch),
    (*CALLS[0], dict(q_stride=513), SlotOutOfRange), (*CALLS[0], dict(output=R(0)), SlotOutOfRange),
    (*CALLS[0], dict(tokens=1 << 31, heads=2, kv_heads=1), UnsupportedOp),
    (*CALLS[1], dict(block_rows=0), UnsupportedOp), (*CALLS[1], dict(bucket_rows=0), UnsupportedOp),
    (*CALLS[1], dict(kv_heads=0), UnsupportedOp), (*CALLS[1], dict(new_stride=127), ShapeMismatch),
    (*CALLS[1], dict(dtype=2), UnsupportedOp), (*CALLS[1], dict(output=R(4), output_scales=R(4)), SlotOutOfRange),
    (*CALLS[1], dict(output=R(0)), SlotOutOfRange), (*CALLS[1], dict(output_scales=R(4, 8)), SlotOutOfRange),
    (*CALLS[1], dict(new=R(3)), SlotOutOfRange), (*CALLS[1], dict(pos=R(4)), SlotOutOfRange),
    (*CALLS[2], dict(heads=9), UnsupportedOp), (*CALLS[2], dict(block_rows=0), UnsupportedOp),
    (*CALLS[2], dict(bucket_rows=1 << 25), UnsupportedOp), (*CALLS[2], dict(q_stride=500), ShapeMismatch),
    (*CALLS[2], dict(output=R(5)), SlotOutOfRange), (*CALLS[2], dict(dtype=1), UnsupportedOp),
    (*CALLS[3], dict(output=R(0)), SlotOutOfRange), (*CALLS[3], dict(dtype=4), UnsupportedOp),
    (*CALLS[3], dict(biases=4096), UnsupportedOp), (*CALLS[3], dict(history_len=524288), UnsupportedOp),
    (*CALLS[3], dict(history=R(1, 2)), SlotOutOfRange), (*CALLS[3], dict(history=NO_BUFFER), SlotOutOfRange),
])
def test_refusals(make, c, sizes, change, error):
    with pytest.raises(error):
        validate(make(replace(c, **change)), sizes)


def test_misaligned_operands_are_refused():
    odd = [n + 16 for n in LOGITS_SIZES]
    for name in ("logits", "output"):
        with pytest.raises(UnsupportedOp):
            validate(KernelCall.LogitsProcess(replace(LOGITS, **{name: R(getattr(LOGITS, name).slot, 1)})), odd)
    for name in ("history", "spans", "params", "bias_ids", "bias_values", "mask"):
        with pytest.raises(UnsupportedOp):
            validate(KernelCall.LogitsProcess(replace(LOGITS, **{name: R(getattr(LOGITS, name).slot, 2)})), odd)
    with pytest.raises(UnsupportedOp):
        validate(KernelCall.AttentionPacked(replace(PACKED, k=R(1, 1))), [n + 16 for n in PACKED_SIZES])
    with pytest.raises(UnsupportedOp):
        validate(KernelCall.AttentionI8Blocks(replace(BLOCKS, lens=R(6, 2))), [n + 16 for n in BLOCKS_SIZES])


def test_absent_operands_and_empty_calls():
    none = replace(LOGITS, history=NO_BUFFER, spans=NO_BUFFER, params=NO_BUFFER, bias_ids=NO_BUFFER,
                   bias_values=NO_BUFFER, mask=NO_BUFFER, history_len=0, biases=0)
    validate(KernelCall.LogitsProcess(none), LOGITS_SIZES)
    for make, c, _ in CALLS[:1] + CALLS[2:3]:
        for change in (dict(tokens=0), dict(batch=0), dict(heads=0), dict(head_dim=0)):
            validate(make(replace(c, **change)), [])
    validate(KernelCall.LogitsProcess(replace(LOGITS, rows=0)), [])
    validate(KernelCall.KvBlockAppend(replace(APPEND, tokens=0)), [0] + APPEND_SIZES[1:])


def test_reference_scale_is_the_least_power_of_two():
    """The restatement the device is held to, on values around the borders."""
    for top in (127.0, np.nextafter(np.float32(127), np.float32(200)), 1.0, 2.0 ** -140, 254.0, 3e38):
        q, s = block_append(np.zeros((1, 1, 16, 1), np.int8), np.zeros((1, 1, 1), np.float32),
                            np.full((1, 1, 1), float(top)), [1], [0], 16)
        assert np.log2(s[0, 0, 0]) == np.floor(np.log2(s[0, 0, 0])) and top <= 127 * float(s[0, 0, 0])
        assert top > 127 * float(s[0, 0, 0]) / 2 or s[0, 0, 0] == 2.0 ** -126
    assert encode(np.array([1.0]), DTYPE_BF16)[0] == 0x3F80


def serving_graph(tokens, batch, heads, kv, d, bucket, block, cols, hist, dtype):
    """One step of a packed batch as a graph: K and V appended, attention over the cache, the
    logits' rules and the pick. The logits are an input (a model's head stands between)."""
    es = 4 if dtype == DTYPE_F32 else 2
    nb = -(-bucket // block)
    w, sizes = HoloWriter(), {}

    def port(ports, name, slot, count, dt, width):
        ports.append(PortDescriptor(name, slot, count, dt, [count]))
        sizes[slot] = count * width
        return BufferRef(slot, 0, count * width)
    qkv = port(w.inputs, "qkv", 0, tokens * (heads + 2 * kv) * d, dtype, es)
    starts = port(w.inputs, "starts", 1, batch + 1, DTYPE_I32, 4)
    pos = port(w.inputs, "pos", 2, batch, DTYPE_I32, 4)
    lens = port(w.inputs, "lens", 3, batch, DTYPE_I32, 4)
    kc_, vc = (port(w.inputs, n, s, batch * kv * bucket * d, 2, 1) for n, s in (("k", 4), ("v", 5)))
    ks, vs = (port(w.inputs, n, s, batch * kv * nb, DTYPE_F32, 4) for n, s in (("ks", 6), ("vs", 7)))
    logits = port(w.inputs, "logits", 8, batch * cols, dtype, es)
    history = port(w.inputs, "history", 9, batch * hist, DTYPE_I32, 4)
    spans = port(w.inputs, "spans", 10, batch * 2, DTYPE_I32, 4)
    params = port(w.inputs, "params", 11, batch * 3, DTYPE_F32, 4)
    ko, vo = (port(w.outputs, n, s, batch * kv * bucket * d, 2, 1) for n, s in (("k'", 12), ("v'", 13)))
    kso, vso = (port(w.outputs, n, s, batch * kv * nb, DTYPE_F32, 4) for n, s in (("ks'", 14), ("vs'", 15)))
    out = port(w.outputs, "attended", 16, tokens * heads * d, dtype, es)
    picks = port(w.outputs, "picks", 17, batch, DTYPE_I32, 4)
    prompt = port(w.outputs, "prompt", 18, tokens * heads * d, dtype, es)
    ruled = BufferRef(19, 0, batch * cols * es)
    stride = (heads + 2 * kv) * d
    view = lambda at: BufferRef(0, at * d * es, tokens * stride * es - at * d * es)  # noqa: E731
    append = lambda at, c, s, oc, os: KernelCall.KvBlockAppend(KvBlockAppendCall(  # noqa: E731
        view(at), starts, pos, c, s, oc, os, tokens, batch, kv, bucket, block, d, stride, dtype))
    w.kernel_calls = [
        append(heads, kc_, ks, ko, kso), append(heads + kv, vc, vs, vo, vso),
        KernelCall.AttentionI8Blocks(AttentionI8BlocksCall(
            view(0), ko, vo, kso, vso, starts, lens, out, tokens, batch, heads, kv, bucket, block, d,
            stride, 0, dtype)),
        KernelCall.AttentionPacked(AttentionPackedCall(
            view(0), view(heads), view(heads + kv), starts, prompt, tokens, batch, heads, kv, d,
            stride, stride, stride, 0, dtype)),
        KernelCall.LogitsProcess(LogitsProcessCall(
            logits, history, spans, params, NO_BUFFER, NO_BUFFER, NO_BUFFER, ruled, batch, cols, hist,
            0, dtype)),
        KernelCall.ArgMax(ArgMaxCall(ruled, picks, batch, cols, dtype))]
    w.exec_plan = [[0, 1, 3, 4], [2, 5]]
    return w.finish()


def test_a_graph_of_them_loads_and_its_appends_move_in_place():
    s = HipSession(None, serving_graph(9, 2, 4, 2, 64, 64, 32, 500, 20, DTYPE_BF16))
    for i in range(s.n_calls):
        c = s.call(i)
        if c.tag == kc.D_KVBA:
            a = c.u.kv_block_append
            assert (a.output.slot, a.output_scales.slot) == (a.cache.slot, a.cache_scales.slot)
    labels = s.output_labels(["blake3:%064x" % i for i in range(12)])
    assert len(set(labels)) == len(labels) == 7


def test_sizes_that_would_wrap_are_refused():
    """A cache whose bytes pass 64 bits does not wrap to one that fits, and a block whose elements
    pass 32 bits is not taken."""
    sizes = [1 << 40, 1 << 40, 1 << 40, 0, 1 << 40]
    big = replace(APPEND, tokens=1, batch=1 << 24, kv_heads=1, bucket_rows=1 << 31, head_dim=512)
    with pytest.raises(UnsupportedOp, match="2\\^50"):
        validate(KernelCall.KvBlockAppend(big), sizes)
    for block, bucket in ((1 << 22, 1 << 23), (1 << 31, (1 << 20) + 1)):
        with pytest.raises(UnsupportedOp, match="2\\^30"):
            validate(KernelCall.KvBlockAppend(replace(APPEND, block_rows=block, bucket_rows=bucket,
                                                      head_dim=1024)), [1 << 50] * 5)
    with pytest.raises(UnsupportedOp):
        validate(KernelCall.AttentionI8Blocks(replace(BLOCKS, batch=1 << 30)), [1 << 40] * 8)
    with pytest.raises(UnsupportedOp):
        validate(KernelCall.LogitsProcess(replace(LOGITS, rows=1 << 31, cols=1 << 20)), [1 << 62] * 8)
