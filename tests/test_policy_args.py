"""What the policy operators refuse (mrn_slot_table, mrn_adjust_logits, mrn_choose_actions), on a
context without a device: each bad argument comes back as MRN_ERR_ARGUMENT with a message before any
CUDA call, and a good call on a machine without a GPU comes back as a CUDA error."""

import ctypes

import pytest

from marina_b200 import _lib
from marina_b200.network import B200Network, LogitRules, NetworkError

P = 1 << 20  # addresses that are never read
Q = 1 << 30
FAR = 1 << 40


class _Library:
    """The test library under the names B200Network calls."""

    def __init__(self):
        lib = _lib.load_test()
        self.mrn_slot_table, self.mrn_adjust_logits = lib.mrn_slot_table, lib.mrn_adjust_logits
        self.mrn_choose_actions, self.mrn_last_error = lib.mrn_choose_actions, lib.mrn_test_context_error


@pytest.fixture
def net():
    n = B200Network.__new__(B200Network)
    n._lib, ctx = _Library(), ctypes.c_void_p(_lib.load_test().mrn_test_context(1 << 20))  # no such device
    n._ctx = ctx
    yield n
    n._ctx = None
    _lib.load_test().mrn_test_context_free(ctx)


def refused(call, *words):
    with pytest.raises(NetworkError) as e:
        call()
    assert e.value.code == 1, str(e.value)
    for w in words:
        assert w in str(e.value), str(e.value)


def reaches_the_device(call):
    with pytest.raises(NetworkError) as e:
        call()
    assert e.value.code == 2, str(e.value)


def test_null_context():
    lib = _lib.load()
    assert lib.mrn_slot_table(None, 1, 1, P, 1, P, P, P, P, None) == 1
    assert lib.mrn_adjust_logits(None, 1, 1, P, 0, 1, None, None, Q, 1, None, 0, None) == 1
    assert lib.mrn_choose_actions(None, 1, 1, P, 0, 1, None, None, None, None, None, Q, None, None, None) == 1


SLOTS = dict(rows=4, width=224, lengths_ptr=P, count=9, entries_ptr=P, starts_ptr=Q, table_ptr=Q + 20, map_ptr=FAR)


@pytest.mark.parametrize("change,words", [
    ({"starts_ptr": P + 12}, "overlaps an input"), ({"map_ptr": P + 32}, "overlaps an input"),
    ({"table_ptr": P - 4 * 224 * 4 + 4}, "overlaps an input"), ({"table_ptr": Q + 16}, "two outputs"),
    ({"map_ptr": Q + 20}, "two outputs"),
    ({"rows": -1}, "rows -1"), ({"width": 0}, "width 0"), ({"count": -1}, "count -1"),
    ({"rows": 1 << 20, "width": 1 << 11}, "2^31 - 1"), ({"lengths_ptr": None}, "NULL"), ({"entries_ptr": None}, "NULL"),
    ({"starts_ptr": None}, "NULL"), ({"table_ptr": None}, "NULL"), ({"map_ptr": P + 2}, "aligned"),
    ({"lengths_ptr": P + 1}, "aligned"),
])
def test_slot_table_refuses(net, change, words):
    good = SLOTS
    reaches_the_device(lambda: net.slot_table(**good))
    refused(lambda: net.slot_table(**{**good, **change}), words)


RULES = dict(columns=P, columns_stride=224, mask=P, mask_stride=146, bias_actions=P, bias_values=P, bias_len=3,
             bias_stride=0, history=P, history_lens=P, history_len=5, history_stride=5, repetition=P, presence=P,
             frequency=P)

BAD_RULES = [
    ({"actions": 0}, "actions 0"), ({"columns": None, "actions": 200}, "200 actions for 224 columns"),
    ({"columns_stride": 223}, "columns_stride 223"), ({"columns_stride": -1}, "columns_stride -1"),
    ({"mask_stride": 145}, "mask_stride 145"), ({"mask_stride": -146}, "mask_stride"), ({"bias_len": -1}, "negative"),
    ({"history_len": -2}, "negative"), ({"bias_len": (1 << 20) + 1}, "longer than 1048576"),
    ({"history_len": (1 << 20) + 1, "history_stride": 1 << 21}, "longer than 1048576"), ({"bias_actions": None}, "bias_actions"), ({"bias_values": None}, "bias_values"),
    ({"bias_stride": 2}, "bias_stride 2"), ({"history": None}, "without history"), ({"history_stride": 4}, "history_stride 4"),
    *[({name: P + 2}, "aligned") for name in ("columns", "mask", "bias_actions", "bias_values", "history", "history_lens",
                                              "repetition", "presence", "frequency")],
]


@pytest.mark.parametrize("change,words", BAD_RULES)
def test_rules_refuse(net, change, words):
    parts = {**RULES, "actions": 4672, **change}
    rules = LogitRules(parts.pop("actions"), **parts)
    refused(lambda: net.adjust_logits(8, 224, P, rules, out_ptr=Q), words)
    refused(lambda: net.choose_actions(8, 224, P, rules, Q), words)


def test_rules_that_are_fine(net):
    for rules in (None, LogitRules(4672, **RULES), LogitRules(4672, mask=P), LogitRules(224)):
        reaches_the_device(lambda: net.adjust_logits(8, 224, P, rules, out_ptr=Q, priors_ptr=FAR))
        reaches_the_device(lambda: net.choose_actions(8, 224, P, rules, Q))
    with pytest.raises(TypeError):
        LogitRules(4672, penalty=P)


@pytest.mark.parametrize("change,words", [
    ({"rows": -1}, "rows = -1"), ({"rows": (1 << 27) + 1, "stride": 0}, "rows = 134217729"), ({"width": 0}, "width 0"),
    ({"width": (1 << 18) + 1, "stride": 1 << 20}, "width 262145"),
    ({"logits_ptr": None}, "logits is NULL"), ({"stride": 223}, "stride 223"), ({"stride": -224}, "stride -224"),
    ({"logits_ptr": P + 1}, "aligned"), ({"temperature_ptr": P + 2}, "aligned"),
])
def test_logits_refuse(net, change, words):
    good = dict(rows=8, width=224, logits_ptr=P, rules=None, dtype="f16")
    call = {**good, **change}
    refused(lambda: net.adjust_logits(**call, out_ptr=Q), words)
    refused(lambda: net.choose_actions(**call, column_ptr=Q), words)


def test_type_refused(net):
    with pytest.raises(ValueError):
        net.adjust_logits(1, 8, P, out_ptr=Q, dtype="f64")
    with pytest.raises(ValueError):
        net.choose_actions(1, 8, P, None, Q, dtype="fp8")
    lib = _lib.load_test()
    assert lib.mrn_adjust_logits(net._ctx, 1, 8, P, 3, 8, None, None, Q, 8, None, 0, None) == 1


@pytest.mark.parametrize("change,words", [
    ({"out_ptr": None}, "neither"), ({"out_ptr": Q + 2}, "aligned"), ({"priors_ptr": Q + 1}, "aligned"),
    ({"out_stride": 99}, "out_stride 99"), ({"priors_ptr": FAR, "priors_stride": 7}, "priors_stride 7"),
    ({"out_ptr": P + 400}, "overlaps"),                      # the logits' second row
    ({"out_ptr": P, "out_stride": 128}, "overlaps"),         # in place, but with other rows
    ({"priors_ptr": P}, "overlaps"), ({"priors_ptr": Q + 40}, "overlaps"),
])
def test_adjust_refuses_its_outputs(net, change, words):
    good = dict(rows=8, width=100, logits_ptr=P, rules=None, out_ptr=Q)
    refused(lambda: net.adjust_logits(**{**good, **change}), words)


def test_outputs_beside_the_logits(net):
    """Column ranges of one matrix share no byte, and the logits' own place is an output."""
    reaches_the_device(lambda: net.adjust_logits(8, 100, P, out_ptr=P))
    reaches_the_device(lambda: net.adjust_logits(8, 100, P, stride=200, out_ptr=P + 400, out_stride=200))
    reaches_the_device(lambda: net.adjust_logits(8, 100, P + 400, stride=200, out_ptr=P, out_stride=200))
    refused(lambda: net.adjust_logits(8, 100, P, stride=199, out_ptr=P + 400, out_stride=199), "overlaps")
    refused(lambda: net.adjust_logits(8, 100, P + 396, stride=199, out_ptr=P, out_stride=199), "overlaps")
    reaches_the_device(lambda: net.adjust_logits(1, 100, P, stride=100, out_ptr=P + 400, out_stride=100))
    reaches_the_device(lambda: net.adjust_logits(1, 100, P, stride=0, out_ptr=P))


def test_choose_refuses_its_outputs(net):
    refused(lambda: net.choose_actions(4, 100, P, None, None), "column is NULL")
    for name in ("action_ptr", "prob_ptr", "top_k_ptr", "top_p_ptr", "uniform_ptr"):
        refused(lambda: net.choose_actions(4, 100, P, None, Q, **{name: Q + 2}), "aligned")


def test_no_rows_is_no_work(net):
    net.adjust_logits(0, 100, None, out_ptr=Q)
    net.choose_actions(0, 100, None, None, None)
