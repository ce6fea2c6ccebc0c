"""A call of frozen parts is packed once."""
import sys
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


def test_whether_a_call_is_frozen_costs_the_same_for_any_number_of_operands():
    """A call that is dispatched once pays for that question and has nothing from its answer, so
    it is not asked operand by operand: nine operands take no more Python calls than two."""
    r = BufferRef
    few = kc.KernelCall(13, kc.UnaryCall(r(0), r(1), 8))
    many = kc.KernelCall.LogitsProcess(kc.LogitsProcessCall(*[r(i) for i in range(8)], 1, 2, 3, 4, kc.DTYPE_BF16))
    counts = []
    for call in (few, many):
        seen = []
        sys.setprofile(lambda frame, event, arg: seen.append(event) if event in ("call", "c_call") else None)
        try:
            form = kc.dispatch_form(call)
        finally:
            sys.setprofile(None)
        assert isinstance(form, bytes) and kc.dispatch_form(call) is form
        counts.append(len(seen))
    assert counts[0] == counts[1], counts


def test_a_number_that_is_not_an_int_is_packed_anew():
    class Flag:
        value = 0

        def __int__(self):
            return self.value
    flag = Flag()
    r = BufferRef
    c = kc.KernelCall(kc.D_MATMUL, replace(kc.MatMulCall(r(0), r(1), r(2), 1, 2, 3), b_packed=flag))
    before = kc.dispatch_form(c)
    assert isinstance(before, bytes)
    flag.value = 1
    assert kc.dispatch_form(c) == bytes(c.to_c()) != before
