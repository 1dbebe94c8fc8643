"""zrl_last_error without a context, between the sequence operators' messages and
calls that were given no context.  No GPU."""
import ctypes as C

from zealot_b200 import native as N


def refuse(L):
    assert L.zrl_dropout(64, None, None, -1, 8, 0, 0.1, 1, 0, None, 64, None) == N.INVALID_ARG
    assert b"dropout" in L.zrl_last_error(None)


def test_a_call_without_a_context_does_not_answer_with_an_older_message():
    L = N.lib()
    null, out = b"null context", C.c_void_p()
    calls = (lambda: L.zrl_set_params(None, 64, 1), lambda: L.zrl_get_params(None, 64, 1),
             lambda: L.zrl_update(None, None, None, None),
             lambda: L.zrl_set_wait_limit(None, 1 << 30),
             lambda: L.zrl_create(None, 0, None, C.byref(out)))
    for call in calls:
        refuse(L)
        assert call() == N.INVALID_ARG
        assert L.zrl_last_error(None) == null
    # and the operators' messages come back
    refuse(L)
