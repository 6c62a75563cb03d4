"""mrn_evaluate_moves and mrn_choose_moves: the pass on move lists, with the policy operators behind it,
against mrn_evaluate's priors and the raw logits of mrn_logits."""

import numpy as np
import pytest

from marina_b200 import chess, model, weights
from marina_b200.network import B200Network, MoveRules, NetworkError
from tests.test_policy_gpu import U, Rules, plain_adjusted, plain_choice, plain_priors

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small(cuda):
    arch = model.Architecture(128, 2, 4, 256)
    net = B200Network(arch, weights.random_init(arch, seed=3, std=0.2), device=0, max_batch=70, precision="bf16")
    boards, legal, counts, _ = chess.random_positions(17, 70, 0, 80)
    yield net, boards, legal, counts
    net.close()


def lists(legal, counts):
    return np.concatenate([legal[i, :c] for i, c in enumerate(counts)]) if len(counts) else np.zeros(0, np.int32)


def slot_logits(net, boards, legal):
    policy, _ = net.logits(boards)
    return np.where(legal >= 0, np.take_along_axis(policy, np.maximum(legal, 0).astype(np.int64), 1), -np.inf).astype(np.float32)


@pytest.mark.parametrize("n", [1, 5, 64, 70])
def test_priors_are_the_padded_call_s(small, n):
    net, boards, legal, counts = small
    boards, legal, counts = boards[:n], legal[:n], counts[:n].copy()
    if n > 2:
        counts[2] = 0  # a position without moves
        legal = legal.copy()
        legal[2] = -1
    want, want_wdl = net.evaluate_packed(boards, legal)
    got, wdl = net.evaluate_moves(boards, counts, lists(legal, counts))
    assert np.array_equal(wdl, want_wdl)
    # Both are softmaxes of the same f32 logits: each within some 40 roundings of the exact one (the
    # exponent's two, the exponential, a sum of up to 224 terms, the quotient).
    assert np.abs(got - lists(want, counts)).max() <= 80 * U
    again, _ = net.evaluate_packed(boards, legal)
    assert np.array_equal(again, want)


def rules_for(rng, n, legal, counts, shared):
    m = 1 if shared else n
    mask = rng.random((m, 4672)) < 0.7
    played = np.stack([rng.choice(legal[i, : max(counts[i], 1)], 12) for i in range(m)]).astype(np.int32)
    bias = (played[:, :4].copy(), rng.standard_normal((m, 4)).astype(np.float32))
    rep, fre = (1 + rng.random(n)).astype(np.float32), rng.random(n).astype(np.float32)
    host = MoveRules(mask=mask, bias=bias, history=played, repetition=rep, presence=0.25, frequency=fre)
    plain = Rules(4672, legal, mask, bias, played, None, rep, np.full(n, 0.25, np.float32), fre)
    return host, plain


@pytest.mark.parametrize("n,shared", [(1, False), (7, True), (70, False), (70, True)])
def test_rules_and_temperature(small, n, shared):
    net, boards, legal, counts = small
    boards, legal, counts = boards[:n], legal[:n], counts[:n]
    rng = np.random.default_rng(n)
    host, plain = rules_for(rng, n, legal, counts, shared)
    t = (0.5 + rng.random(n)).astype(np.float32)
    a = plain_adjusted(slot_logits(net, boards, legal), plain)
    got, wdl = net.evaluate_moves(boards, counts, lists(legal, counts), host, t)
    want = plain_priors(a, t)
    assert np.array_equal(wdl, net.evaluate_packed(boards, legal)[1])
    # logits of this network are below 40 in size: an exponent is off by at most 4 * 160 U
    assert np.abs(got - lists(want, counts)).max() <= 1000 * U
    u = rng.random(n).astype(np.float32)
    k, p = rng.integers(1, 12, n).astype(np.int32), rng.random(n).astype(np.float32)
    for kw in (dict(), dict(top_k=k), dict(top_p=p), dict(top_k=k, top_p=p)):
        move, prob, _ = net.choose_moves(boards, counts, lists(legal, counts), u, host, t, **kw)
        col, pr = plain_choice(a, t, kw.get("top_k"), kw.get("top_p"), u)
        assert np.array_equal(move, col)
        assert np.abs(prob - pr).max() <= 2 * U
    move, _, _ = net.choose_moves(boards, counts, lists(legal, counts), rules=host)
    assert np.array_equal(move, plain_choice(a, None, None, None, None)[0])
    assert net.status_word() == 0


def test_calls_of_growing_and_shrinking_sizes(small):
    net, boards, legal, counts = small
    for n in (3, 70, 1, 40, 70):
        got, _ = net.evaluate_moves(boards[:n], counts[:n], lists(legal[:n], counts[:n]), MoveRules(), 1.0)
        want, _ = net.evaluate_packed(boards[:n], legal[:n])
        assert np.abs(got - lists(want, counts[:n])).max() <= 80 * U
    got, wdl = net.evaluate_moves(boards[:0], counts[:0], legal[0, :0])
    assert got.shape == (0,) and wdl.shape == (0, 3)
    got, wdl = net.evaluate_moves(boards[:2], np.zeros(2, np.int32), legal[0, :0])  # no moves anywhere
    assert got.shape == (0,) and np.array_equal(wdl, net.evaluate_packed(boards[:2], np.full((2, 224), -1))[1])
    move, prob, _ = net.choose_moves(boards[:2], np.zeros(2, np.int32), legal[0, :0], 0.5)
    assert (move == -1).all() and (prob == 0).all()


def test_refusals(small):
    net, boards, legal, counts = small
    flat = lists(legal[:3], counts[:3])

    def code(call, *words):
        with pytest.raises(NetworkError) as e:
            call()
        assert all(w in str(e.value) for w in words), str(e.value)
        return e.value.code

    assert code(lambda: net.evaluate_moves(np.zeros((71, 66)), np.zeros(71), np.zeros(0)), "max_batch 70") == 3
    assert code(lambda: net.evaluate_moves(boards[:1], [225], np.zeros(225)), "225 legal moves") == 4
    for bad in (-1, 4672, 2**31 - 1):
        wrong = flat.copy()
        wrong[counts[0] + 1] = bad
        assert code(lambda: net.evaluate_moves(boards[:3], counts[:3], wrong), "position 1", str(bad)) == 7
        assert code(lambda: net.choose_moves(boards[:3], counts[:3], wrong, 0.5), "position 1") == 7
    board = boards[:3].copy()
    board[2, 5] = 13
    assert code(lambda: net.evaluate_moves(board, counts[:3], flat), "position 2") == 1
    with pytest.raises(ValueError):
        net.evaluate_moves(boards[:3], counts[:3], flat[:-1])
    with pytest.raises(ValueError):
        net.evaluate_moves(boards[:3], counts[:3], flat, MoveRules(mask=np.ones((2, 4672))))
    with pytest.raises(ValueError):
        net.evaluate_moves(boards[:3], counts[:3], flat, MoveRules(bias=([[1, 2]], [[1.0]])))
    with pytest.raises(ValueError):
        net.choose_moves(boards[:3], counts[:3], flat, np.zeros(2))
    lib = net._lib
    from marina_b200.network import LogitRules
    a, l, f = boards[:3].copy(), counts[:3].astype(np.int32), flat.astype(np.int32)
    out, wdl = np.zeros(len(f), np.float32), np.zeros((3, 3), np.float32)

    def raw(rules):
        return lib.mrn_evaluate_moves(net._ctx, 3, a.ctypes.data, l.ctypes.data, f.ctypes.data, rules, None,
                                      out.ctypes.data, wdl.ctypes.data)

    assert raw(LogitRules(4672, columns=f.ctypes.data)) == 1 and raw(LogitRules(100)) == 1 and raw(LogitRules(4672)) == 0
    assert lib.mrn_choose_moves(net._ctx, 3, a.ctypes.data, l.ctypes.data, f.ctypes.data, None, None, None, None, None,
                                None, None, wdl.ctypes.data) == 1
    # the context serves the next call
    got, _ = net.evaluate_moves(boards[:3], counts[:3], flat)
    assert np.abs(got - lists(net.evaluate_packed(boards[:3], legal[:3])[0], counts[:3])).max() <= 80 * U
