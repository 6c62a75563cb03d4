"""The policy operators beside a pass on the same context, on a context without a device, and the arguments of
the calls on move lists."""

import threading

import pytest

from marina_b200 import _lib
from marina_b200.network import MoveRules, NetworkError
from tests.test_policy_args import P, Q, net  # noqa: F401


def on_a_thread(call):
    """Starts `call` on a thread of its own; returns the thread and what it returned or raised."""
    got = []

    def run():
        try:
            got.append(call())
        except NetworkError as e:
            got.append(e)

    thread = threading.Thread(target=run, daemon=True)
    thread.start()
    return thread, got


CALLS = {
    "slot_table": (lambda n, **kw: n.slot_table(4, 224, P, 9, P, Q, Q + 20, **kw),
                   lambda n, **kw: n.slot_table(-1, 224, P, 9, P, Q, Q + 20, **kw)),
    "adjust_logits": (lambda n, **kw: n.adjust_logits(8, 100, P, out_ptr=Q, **kw),
                      lambda n, **kw: n.adjust_logits(8, 0, P, out_ptr=Q, **kw)),
    "choose_actions": (lambda n, **kw: n.choose_actions(8, 100, P, None, Q, **kw),
                       lambda n, **kw: n.choose_actions(8, 0, P, None, Q, **kw)),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_call_on_the_callers_stream_does_not_wait_for_a_pass(net, name):  # noqa: F811
    lib = _lib.load_test()
    good, bad = CALLS[name]
    threads = []
    lib.mrn_test_context_lock(net._ctx)  # as a synchronous pass of another thread holds it
    try:
        for call, code in ((good, 2), (bad, 1)):
            thread, got = on_a_thread(lambda: call(net, stream=1))
            threads.append(thread)
            thread.join(20)
            assert not thread.is_alive() and got[0].code == code and "failed: " in str(got[0])
        # the context's own stream may be in the middle of a capture: this one waits
        thread, got = on_a_thread(lambda: good(net, stream=None))
        threads.append(thread)
        thread.join(0.3)
        assert thread.is_alive()
    finally:
        lib.mrn_test_context_unlock(net._ctx)
        for thread in threads:
            thread.join(20)
    assert got[0].code == 2


@pytest.mark.parametrize("name", ["repetition", "presence", "frequency"])
@pytest.mark.parametrize("history", [None, [[]], [[1, 2]]])
def test_penalties_are_checked_with_and_without_a_history(name, history):
    with pytest.raises(ValueError, match=name):
        MoveRules(history=history, **{name: [1.0] * 5}).packed(3)
    for value in (1.5, [1.0, 2.0, 3.0]):
        packed = MoveRules(history=history, **{name: value}).packed(3)
        assert packed.history_len == (2 if history == [[1, 2]] else 0)
        assert bool(getattr(packed, name)) == (history is not None)
