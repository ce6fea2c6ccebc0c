"""A call of frozen parts is packed once."""
from dataclasses import replace

from hologram_amd import BufferRef
from hologram_amd import kernel_call as kc


def test_the_packed_form_stays_with_a_frozen_call():
    """Equal calls keep equal forms, a changed copy packs its own, and a call that holds anything
    that could change is packed anew."""
    u = kc.UnaryCall(BufferRef(0), BufferRef(1, 64), 8)
    a, b = kc.KernelCall(13, u), kc.KernelCall(13, u)
    first = kc.dispatch_form(a)
    assert kc.dispatch_form(a) is first and first == bytes(a.to_c()) == kc.dispatch_form(b)
    assert a == b and hash(a) == hash(b) and repr(a) == repr(kc.KernelCall(13, u))
    c = replace(a, tag=14)
    assert kc.dispatch_form(c) == bytes(c.to_c()) != first
    mm = kc.MatMulCall(BufferRef(0), BufferRef(1), BufferRef(2), 1, 2, 3)
    d = kc.KernelCall.MatMulActivation(kc.MatMulActivationCall(mm, 1))
    assert kc.dispatch_form(d) is kc.dispatch_form(d)

    class Ref:
        slot, offset, length = 1, 0, 0
    ref = Ref()
    e = kc.KernelCall(13, replace(u, input=ref))
    before = kc.dispatch_form(e)
    ref.slot = 2
    assert kc.dispatch_form(e) != before
