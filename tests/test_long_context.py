"""The calls of a long-context step (130-133) on the host: the codec, the C layouts' packed form,
the op signatures, the refusals, and a dry load of a graph that holds them."""
import struct
from dataclasses import replace

import numpy as np
import pytest

from hologram_amd import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, DTYPE_I32, DTYPE_I8, NO_BUFFER,
                          AttentionI8SelectedCall, BufferRef, ConstantEntry, HipSession, HoloWriter,
                          KernelCall, KvBlockAppendCall, KvBlockBoundsCall, KvBlockSelectCall,
                          PortDescriptor, QkNormRotaryCall, ShapeMismatch, SlotOutOfRange,
                          UnsupportedOp, decode_call, validate)
from hologram_amd import kernel_call as kc
from hologram_amd.kappa import op_signature

R = BufferRef
EPS = struct.unpack("<I", struct.pack("<f", 1e-6))[0]
ROTARY = QkNormRotaryCall(R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), R(8), 10, 3, 8, 2, 64, 48, 0,
                          0, EPS, 0, 3, 1, DTYPE_BF16)
ROTARY_SIZES = [10 * 8 * 64 * 2, 10 * 2 * 64 * 2, 128, 128, 16, 12, 24 * 4, 10 * 8 * 64 * 2,
                10 * 2 * 64 * 2]
BOUNDS = KvBlockBoundsCall(R(0), R(1), R(2), R(3), R(3), 10, 3, 2, 100, 32, 64)
BOUNDS_SIZES = [6 * 100 * 64, 16, 12, 6 * 4 * 2 * 64]
SELECT = KvBlockSelectCall(R(0), R(1), R(2), R(3), R(4), R(5), 10, 3, 8, 2, 100, 32, 64, 0, 3, 1, 1,
                           DTYPE_F16)
SELECT_SIZES = [10 * 8 * 64 * 2, 6 * 4 * 2 * 64, 6 * 4 * 4, 16, 12, 10 * 2 * 3 * 4]
SELECTED = AttentionI8SelectedCall(R(0), R(1), R(2), R(3), R(4), R(5), R(6), R(7), R(8), 10, 3, 8, 2,
                                   100, 32, 64, 0, 3, 0, DTYPE_F32)
SELECTED_SIZES = [10 * 8 * 64 * 4, 6 * 100 * 64, 6 * 100 * 64, 6 * 4 * 4, 6 * 4 * 4, 10 * 2 * 3 * 4, 16,
                  12, 10 * 8 * 64 * 4]
CALLS = [(KernelCall.QkNormRotary, ROTARY, ROTARY_SIZES),
         (KernelCall.KvBlockBounds, BOUNDS, BOUNDS_SIZES),
         (KernelCall.KvBlockSelect, SELECT, SELECT_SIZES),
         (KernelCall.AttentionI8Selected, SELECTED, SELECTED_SIZES)]


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


def test_signatures_tell_scalars_and_views_apart():
    for make, c, _ in CALLS:
        ref = op_signature(make(c))
        for f in c.__dataclass_fields__:
            v = getattr(c, f)
            other = replace(v, offset=v.offset + 64) if isinstance(v, BufferRef) else v ^ 1
            assert op_signature(make(replace(c, **{f: other}))) != ref, f


@pytest.mark.parametrize("make,c,sizes,change,error", [
    (*CALLS[0], dict(heads=7), UnsupportedOp), (*CALLS[0], dict(dtype=2), UnsupportedOp),
    (*CALLS[0], dict(head_dim=1025), UnsupportedOp), (*CALLS[0], dict(rotary_dim=66), ShapeMismatch),
    (*CALLS[0], dict(rotary_dim=47), UnsupportedOp), (*CALLS[0], dict(norms=4), UnsupportedOp),
    (*CALLS[0], dict(interleaved=2), UnsupportedOp), (*CALLS[0], dict(epsilon_bits=0xBF800000), UnsupportedOp),
    (*CALLS[0], dict(epsilon_bits=0x7FC00000), UnsupportedOp),
    (*CALLS[0], dict(epsilon_bits=0x7F800000), UnsupportedOp),
    (*CALLS[0], dict(magnitude_bits=0x7F800000), UnsupportedOp),
    (*CALLS[0], dict(magnitude_bits=0x80000000), UnsupportedOp),
    (*CALLS[0], dict(q_stride=511), ShapeMismatch), (*CALLS[0], dict(k_stride=127), ShapeMismatch),
    (*CALLS[0], dict(q_stride=513), SlotOutOfRange), (*CALLS[0], dict(q_output=R(0)), SlotOutOfRange),
    (*CALLS[0], dict(q_output=R(1)), SlotOutOfRange), (*CALLS[0], dict(k_output=R(7)), SlotOutOfRange),
    (*CALLS[0], dict(k_output=R(6)), SlotOutOfRange), (*CALLS[0], dict(freqs=NO_BUFFER), SlotOutOfRange),
    (*CALLS[0], dict(pos=R(5, 2)), SlotOutOfRange),
    (*CALLS[0], dict(tokens=1 << 31, heads=2, kv_heads=1), UnsupportedOp),
    (*CALLS[1], dict(block_rows=0), UnsupportedOp), (*CALLS[1], dict(bucket_rows=0), UnsupportedOp),
    (*CALLS[1], dict(kv_heads=0), UnsupportedOp), (*CALLS[1], dict(head_dim=0), UnsupportedOp),
    (*CALLS[1], dict(output=R(0)), SlotOutOfRange), (*CALLS[1], dict(output=R(3, 64)), SlotOutOfRange),
    (*CALLS[1], dict(output=R(2)), SlotOutOfRange), (*CALLS[1], dict(head_dim=1025), UnsupportedOp),
    (*CALLS[2], dict(heads=9), UnsupportedOp), (*CALLS[2], dict(dtype=1), UnsupportedOp),
    (*CALLS[2], dict(keep_last=0), UnsupportedOp), (*CALLS[2], dict(keep_first=3), ShapeMismatch),
    (*CALLS[2], dict(keep_first=0xFFFFFFFF), ShapeMismatch), (*CALLS[2], dict(top=1), ShapeMismatch),
    (*CALLS[2], dict(top=(1 << 20) + 1), UnsupportedOp), (*CALLS[2], dict(block_rows=0), UnsupportedOp),
    (*CALLS[2], dict(bucket_rows=1 << 21, block_rows=1), UnsupportedOp),
    (*CALLS[2], dict(heads=1024, kv_heads=2, head_dim=512), UnsupportedOp),
    (*CALLS[2], dict(q_stride=500), ShapeMismatch), (*CALLS[2], dict(output=R(2)), SlotOutOfRange),
    (*CALLS[3], dict(heads=9), UnsupportedOp), (*CALLS[3], dict(dtype=10), UnsupportedOp),
    (*CALLS[3], dict(top=0), UnsupportedOp), (*CALLS[3], dict(top=(1 << 20) + 1), UnsupportedOp),
    (*CALLS[3], dict(bucket_rows=1 << 25), UnsupportedOp), (*CALLS[3], dict(block_rows=0), UnsupportedOp),
    (*CALLS[3], dict(output=R(5)), SlotOutOfRange), (*CALLS[3], dict(q_stride=1), ShapeMismatch),
])
def test_refusals(make, c, sizes, change, error):
    with pytest.raises(error):
        validate(make(replace(c, **change)), sizes)


@pytest.mark.parametrize("make,c,sizes,names", [
    (*CALLS[0], ("q", "k", "q_gamma", "k_gamma", "q_output", "k_output")),
    (*CALLS[0], ("starts", "pos", "freqs")), (*CALLS[1], ("starts", "pos")),
    (*CALLS[2], ("q", "k_scales", "starts", "lens", "output")),
    (*CALLS[3], ("q", "k_scales", "v_scales", "blocks", "starts", "lens", "output"))])
def test_misaligned_operands_are_refused(make, c, sizes, names):
    for name in names:
        ref = getattr(c, name)
        with pytest.raises(UnsupportedOp, match="element-aligned"):
            validate(make(replace(c, **{name: R(ref.slot, 1)})), [n + 16 for n in sizes])


def test_absent_operands_and_empty_calls():
    alone = replace(ROTARY, k=NO_BUFFER, k_gamma=NO_BUFFER, k_output=NO_BUFFER)
    validate(KernelCall.QkNormRotary(alone), ROTARY_SIZES)
    validate(KernelCall.QkNormRotary(replace(ROTARY, q_gamma=NO_BUFFER, k_gamma=NO_BUFFER)), ROTARY_SIZES)
    # what a call does not use is not looked at
    validate(KernelCall.QkNormRotary(replace(ROTARY, norms=0, q_gamma=R(99), k_gamma=R(99))), ROTARY_SIZES)
    validate(KernelCall.QkNormRotary(replace(ROTARY, rotary_dim=0, freqs=NO_BUFFER, pos=NO_BUFFER)), ROTARY_SIZES)
    for make, c, _ in CALLS[:1] + CALLS[2:]:
        for change in (dict(tokens=0), dict(batch=0), dict(heads=0), dict(head_dim=0)):
            validate(make(replace(c, **change)), [])
    validate(KernelCall.KvBlockBounds(replace(BOUNDS, tokens=0)), BOUNDS_SIZES)


def test_sizes_that_would_wrap_are_refused():
    big = dict(tokens=1, batch=1 << 24, bucket_rows=1 << 31)
    with pytest.raises(UnsupportedOp, match="2\\^50"):
        validate(KernelCall.KvBlockBounds(replace(BOUNDS, kv_heads=1, **big)), [1 << 40] * 4)
    with pytest.raises(UnsupportedOp, match="2\\^50"):
        validate(KernelCall.KvBlockSelect(replace(SELECT, heads=1, kv_heads=1, block_rows=1 << 20, **big)),
                 [1 << 40] * 6)
    with pytest.raises(UnsupportedOp, match="2\\^30"):
        validate(KernelCall.KvBlockBounds(replace(BOUNDS, bucket_rows=1 << 23, block_rows=1 << 22, head_dim=1024)),
                 [1 << 50] * 4)
    with pytest.raises(UnsupportedOp, match="launch"):
        validate(KernelCall.KvBlockSelect(replace(SELECT, tokens=1 << 24, heads=2, kv_heads=2, head_dim=24)), [1 << 50] * 6)
    with pytest.raises(UnsupportedOp, match="launch"):
        validate(KernelCall.AttentionI8Selected(replace(SELECTED, tokens=1 << 26, heads=2)), [1 << 60] * 9)
    with pytest.raises(UnsupportedOp, match="launch"):
        validate(KernelCall.QkNormRotary(replace(ROTARY, tokens=1 << 25, heads=2, kv_heads=2, head_dim=2,
                                                 rotary_dim=2)), [1 << 60] * 9)


def long_step_graph(tokens, batch, heads, kv, d, bucket, block, top, dtype, gamma, freqs, rot, interleaved=0):
    """A step over a long cache as a graph: q and k of the projection's output normed and rotated,
    K and V appended, the touched blocks' bounds, each row's blocks and the attention over them."""
    es = 4 if dtype == DTYPE_F32 else 2
    nb = -(-bucket // block)
    w = HoloWriter()

    def port(ports, name, slot, count, dt, width):
        ports.append(PortDescriptor(name, slot, count, dt, [count]))
        return BufferRef(slot, 0, count * width)
    qkv = port(w.inputs, "qkv", 0, tokens * (heads + 2 * kv) * d, dtype, es)
    starts = port(w.inputs, "starts", 1, batch + 1, DTYPE_I32, 4)
    pos = port(w.inputs, "pos", 2, batch, DTYPE_I32, 4)
    lens = port(w.inputs, "lens", 3, batch, DTYPE_I32, 4)
    kc_, vc = (port(w.inputs, n, s, batch * kv * bucket * d, DTYPE_I8, 1) for n, s in (("k", 4), ("v", 5)))
    ks, vs = (port(w.inputs, n, s, batch * kv * nb, DTYPE_F32, 4) for n, s in (("ks", 6), ("vs", 7)))
    kb = port(w.inputs, "bounds", 8, batch * kv * nb * 2 * d, DTYPE_I8, 1)
    w.constants = [ConstantEntry(9, dtype, gamma.tobytes()), ConstantEntry(10, DTYPE_F32, freqs.tobytes())]
    g, f = BufferRef(9, 0, gamma.nbytes), BufferRef(10, 0, freqs.nbytes)
    ko, vo = (port(w.outputs, n, s, batch * kv * bucket * d, DTYPE_I8, 1) for n, s in (("k'", 11), ("v'", 12)))
    kso, vso = (port(w.outputs, n, s, batch * kv * nb, DTYPE_F32, 4) for n, s in (("ks'", 13), ("vs'", 14)))
    kbo = port(w.outputs, "bounds'", 15, batch * kv * nb * 2 * d, DTYPE_I8, 1)
    lists = port(w.outputs, "blocks", 16, tokens * kv * top, DTYPE_I32, 4)
    out = port(w.outputs, "attended", 17, tokens * heads * d, dtype, es)
    q = port(w.outputs, "q", 18, tokens * heads * d, dtype, es)
    k = port(w.outputs, "k rows", 19, tokens * kv * d, dtype, es)
    stride = (heads + 2 * kv) * d
    view = lambda at: BufferRef(qkv.slot, at * d * es, tokens * stride * es - at * d * es)  # noqa: E731
    shape = (tokens, batch, kv, bucket, block, d)
    w.kernel_calls = [
        KernelCall.QkNormRotary(QkNormRotaryCall(view(0), view(heads), g, g, starts, pos, f, q, k, tokens, batch,
                                                 heads, kv, d, rot, stride, stride, EPS, 0, 3, interleaved, dtype)),
        KernelCall.KvBlockAppend(KvBlockAppendCall(k, starts, pos, kc_, ks, ko, kso, *shape, 0, dtype)),
        KernelCall.KvBlockAppend(KvBlockAppendCall(view(heads + kv), starts, pos, vc, vs, vo, vso, *shape, stride,
                                                   dtype)),
        KernelCall.KvBlockBounds(KvBlockBoundsCall(ko, starts, pos, kb, kbo, *shape)),
        KernelCall.KvBlockSelect(KvBlockSelectCall(q, kbo, kso, starts, lens, lists, tokens, batch, heads, kv, bucket,
                                                   block, d, 0, top, 1, 2, dtype)),
        KernelCall.AttentionI8Selected(AttentionI8SelectedCall(
            q, ko, vo, kso, vso, lists, starts, lens, out, tokens, batch, heads, kv, bucket, block, d, 0, top, 0,
            dtype))]
    w.exec_plan = [[0, 2], [1], [3], [4], [5]]
    return w.finish()


def test_a_graph_of_them_loads_and_its_caches_move_in_place():
    s = HipSession(None, long_step_graph(9, 2, 4, 2, 64, 256, 16, 4, DTYPE_BF16, np.ones(64, np.uint16),
                                         np.ones(32, np.float32), 64))
    moved = 0
    for i in range(s.n_calls):
        c = s.call(i)
        if c.tag == kc.D_KVBA:
            a = c.u.kv_block_append
            moved += (a.output.slot, a.output_scales.slot) == (a.cache.slot, a.cache_scales.slot)
        if c.tag == kc.D_KVBB:
            moved += c.u.kv_block_bounds.output.slot == c.u.kv_block_bounds.bounds.slot
    assert moved == 3
    labels = s.output_labels(["blake3:%064x" % i for i in range(9)])
    assert len(set(labels)) == len(labels) == 9


def test_an_output_for_k_without_k_is_refused():
    """The call would not write it, but a session would label it as written."""
    for change in (dict(k=NO_BUFFER), dict(k=NO_BUFFER, k_gamma=NO_BUFFER), dict(k=NO_BUFFER, norms=0, rotary_dim=0)):
        with pytest.raises(UnsupportedOp, match="k_output"):
            validate(KernelCall.QkNormRotary(replace(ROTARY, **change)), ROTARY_SIZES)
    w = HoloWriter()
    w.inputs = [PortDescriptor("q", 0, 640, DTYPE_BF16, [640]), PortDescriptor("starts", 1, 2, DTYPE_I32, [2])]
    w.outputs = [PortDescriptor("q'", 2, 640, DTYPE_BF16, [640]), PortDescriptor("k'", 3, 640, DTYPE_BF16, [640])]
    alone = QkNormRotaryCall(R(0, 0, 1280), NO_BUFFER, NO_BUFFER, NO_BUFFER, R(1, 0, 8), NO_BUFFER, NO_BUFFER,
                             R(2, 0, 1280), R(3, 0, 1280), 10, 1, 1, 0, 64, 0)
    w.kernel_calls, w.exec_plan = [KernelCall.QkNormRotary(alone)], [[0]]
    with pytest.raises(UnsupportedOp, match="k_output"):
        HipSession(None, w.finish())


@pytest.mark.parametrize("head_dim,rot", [(2, 2), (16, 16), (128, 32)])
def test_the_largest_launches_that_the_header_names_are_taken(head_dim, rot):
    """Right below each call's bound, in whatever form the sizes take."""
    huge = [1 << 60] * 9
    alone = replace(ROTARY, k=NO_BUFFER, k_output=NO_BUFFER, heads=1, kv_heads=0, head_dim=head_dim, rotary_dim=rot)
    validate(KernelCall.QkNormRotary(replace(alone, tokens=(1 << 26) - 4)), huge)
    with pytest.raises(UnsupportedOp, match="launch"):
        validate(KernelCall.QkNormRotary(replace(alone, tokens=1 << 26)), huge)
    for bucket in (100, 640 * 32, 641 * 32):
        most = ((1 << 23) - 1) // (-(-bucket // 32) // 256 + 1)
        for tokens, batch in ((16, most - 1), (16 * (most - 3), 2)):
            c = replace(SELECT, tokens=min(tokens, (1 << 24) - 1), batch=batch, heads=1, kv_heads=1, head_dim=head_dim,
                        bucket_rows=bucket)
            validate(KernelCall.KvBlockSelect(c), huge)
    for block in (32, 33):
        c = replace(SELECTED, tokens=(1 << 24) - 1, batch=2, heads=1, kv_heads=1, head_dim=head_dim, block_rows=block,
                    top=1 << 20)
        validate(KernelCall.AttentionI8Selected(c), huge)
