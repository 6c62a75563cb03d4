"""The policy operators at the ends of what they accept, against the plain implementations of
test_policy_gpu.py."""

import threading

import numpy as np
import pytest

from marina_b200 import chess, model, weights
from marina_b200.network import B200Network, NetworkError
from tests.test_policy_gpu import (TYPES, Rules, call_choose, check_adjust, check_choose, check_priors, check_state,  # noqa: F401
                                   clean_status, dev, here, make_state, net, plain_adjusted, plain_choice,
                                   plain_slot_table, some_logits, some_rules, together)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width", [(1, 2**31 - 4), (1, 2**31 - 1), (2, 2**30 - 1)])
def test_slot_rows_of_as_many_slots_as_there_may_be(net, rows, width):  # noqa: F811
    """A table of 2^31 - 1 slots or a little less: the column behind a row's last does not wrap around."""
    count, guard = 200, 64
    lengths = np.full(rows, count // rows, np.int32)
    entries, n = np.arange(7, 7 + count, dtype=np.int32), count // rows
    whole = torch.full((guard + rows * width + guard,), -6, dtype=torch.int32, device="cuda:0")
    table = whole[guard: guard + rows * width]  # 256 bytes in: its alignment is the buffer's
    starts = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda:0")
    where = torch.full((count,), -7, dtype=torch.int32, device="cuda:0")
    le, en = dev(lengths), dev(entries)
    net.slot_table(rows, width, le.data_ptr(), count, en.data_ptr(), starts.data_ptr(), table.data_ptr(),
                   where.data_ptr(), stream=here())
    torch.cuda.synchronize()
    assert (whole[:guard] == -6).all() and (whole[guard + rows * width:] == -6).all()
    assert starts.tolist() == [n * r for r in range(rows + 1)]
    for r in range(rows):
        row = table[r * width: (r + 1) * width]
        assert np.array_equal(row[:n].cpu().numpy(), entries[r * n: (r + 1) * n])
        assert int(row[n:].max()) == -1 == int(row[n:].min())
    assert np.array_equal(where.cpu().numpy(), np.concatenate([r * width + np.arange(n) for r in range(rows)]))
    assert net.status_word() == 0


@pytest.mark.parametrize("width,history,bias", [(513, 1, 0), (640, 0, 1), (700, 190, 2), (700, 190, 3), (2047, 40, 1023), (2048, 2000, 1024),
                                                (2049, 333, 1025), (6000, 5000, 3000), (20000, 700, 90),
                                                (40000, 3000, 200), (262144, 900, 60)])
def test_wide_slot_rows(net, width, history, bias):  # noqa: F811
    """Slot rows above 512 columns, whose lists are looked up in 2048 of them at a time: actions that a row
    names once, twice and in places far apart, biases whose sum depends on their order."""
    rng = np.random.default_rng(width)
    rows, actions = 3, 2 * width
    columns = rng.integers(0, actions, (rows, width)).astype(np.int32)  # many of them twice
    columns[0] = rng.permutation(actions)[:width]
    columns[1, [0, width // 2, width - 1]] = 77
    columns[2, rng.random(width) < 0.4] = -1
    values = (rng.standard_normal((rows, bias)) * 10.0 ** rng.integers(-4, 5, (rows, bias))).astype(np.float32)
    ids = rng.integers(-1, actions + 2, (rows, bias)).astype(np.int32)
    ids[:, ::3] = 77
    played = rng.integers(-2, actions + 2, (rows, history)).astype(np.int32)
    played[:, ::2] = columns[:, :1]
    rules = Rules(actions, columns, rng.random((rows, actions)) < 0.7, (ids, values) if bias else None,
                  played if history else None, rng.integers(0, history + 1, rows).astype(np.int32) if history else None,
                  (1 + rng.random(rows)).astype(np.float32), rng.random(rows).astype(np.float32),
                  rng.random(rows).astype(np.float32) / 4)
    rules.mask[:, 77] = True
    for dtype in ("f32", "bf16"):
        x = some_logits(rng, rows, width, dtype)
        check_adjust(net, x, rules, None, dtype)
        check_choose(net, x, rules, None, None, None, rng.random(rows).astype(np.float32), dtype)
        check_choose(net, x, rules, None, np.full(rows, 9, np.int32), np.full(rows, 0.8, np.float32),
                     rng.random(rows).astype(np.float32), dtype)
    assert net.status_word() == 0


def milliseconds(call):
    call()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    call()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b)


@pytest.mark.parametrize("rows,width,entries", [(2, 4096, 1 << 16)])
def test_long_lists_over_wide_slot_rows(net, rows, width, entries):  # noqa: F811
    """The lists are gone through once for a few thousand columns, not once for each column: 2^16 entries
    of each list against 4096 columns are 5e8 comparisons a row, which took 86 ms; a look-up of each entry
    takes 3 to 4. The bound lies between, a factor of four from either."""
    rng = np.random.default_rng(1)
    columns = np.stack([rng.permutation(2 * width)[:width] for _ in range(rows)]).astype(np.int32)
    rules = Rules(2 * width, columns, None,
                  (rng.integers(0, 2 * width, (rows, entries)).astype(np.int32),
                   rng.standard_normal((rows, entries)).astype(np.float32)),
                  rng.integers(0, 2 * width, (rows, entries)).astype(np.int32)).on_device()
    x = dev(rng.standard_normal((rows, width)).astype(np.float32))
    out = torch.empty_like(x)
    column = torch.empty(rows, dtype=torch.int32, device="cuda:0")
    adjust = lambda: net.adjust_logits(rows, width, x.data_ptr(), rules, out_ptr=out.data_ptr(), stream=here())
    choose = lambda: net.choose_actions(rows, width, x.data_ptr(), rules, column.data_ptr(), stream=here())
    took = milliseconds(adjust), milliseconds(choose)
    assert max(took) < 20, took


F32 = np.finfo(np.float32)
TINY = np.float32(2.0 ** -149)  # the smallest f32 above 0


def far_rows(rng, width):
    """Logits and temperatures whose difference leaves f32, or whose quotient needs a scale that does."""
    z = rng.integers(0, 9, (12, width)).astype(np.float64)  # how many temperatures below the largest, about
    z[:, rng.integers(0, width, 3)] = 0
    t = np.array([1e38, 1e-40, TINY, F32.max, 1e-39, 2.0 ** 100, 2.0 ** 100 * 1.5, 2.0 ** -100, 2.0 ** -101, 1e-38, 1e-35, 1e-33],
                 np.float32)
    x = np.empty((12, width))
    x[0] = 3e38 - z[0] * 0.75e38                 # the lowest 6e38 below the largest
    x[1] = -z[1] * 1e-40
    x[2] = (3 - z[2]) * TINY
    x[3] = F32.max * (1 - z[3] / 4)              # two temperatures from end to end
    x[4] = rng.standard_normal(width) * 1e-39
    x[5:9] = (z[5:9] - 4) * t[5:9, None]
    x[9] = 2.0 ** 20 - z[9] / 8                   # a step of f32 away: 2^120 temperatures
    x[10] = -3e38 * (1 + z[10] / 64)
    x[11] = 2.0 ** 20 - 2.0 ** -4 - z[11] / 16
    return x.astype(np.float32), t


@pytest.mark.parametrize("width", [40, 224, 500, 5000, 40000])
def test_priors_of_logits_far_apart(net, width):  # noqa: F811
    x, t = far_rows(np.random.default_rng(width), width)
    check_adjust(net, dev(x), None, t)
    mask = np.random.default_rng(width + 1).random(x.shape) < 0.5
    x[~mask] = -np.inf
    check_adjust(net, dev(x), Rules(width, mask=mask), t)
    check_adjust(net, dev(x), None, np.full(len(t), np.inf, np.float32))  # all that is left, in equal shares


@pytest.mark.parametrize("width", [40, 224, 500, 5000, 40000])
def test_choice_of_logits_far_apart(net, width):  # noqa: F811
    rng = np.random.default_rng(width + 2)
    x, t = far_rows(rng, width)
    rows = len(t)
    rules = Rules(width, mask=rng.random(x.shape) < 0.5)
    for u in (rng.random(rows).astype(np.float32), np.full(rows, 1 - 2.0 ** -24, np.float32), None):
        for k in (None, np.full(rows, 5, np.int32), np.full(rows, width // 2, np.int32)):
            for p in (None, np.full(rows, 0.9, np.float32)):
                check_choose(net, dev(x), None, t, k, p, u)
                check_choose(net, dev(x), rules, t, k, p, u)


def test_message_of_an_operators_bad_slot(net):  # noqa: F811
    """The status word that an operator leaves fails the next synchronous call, whose message names the
    operators' limit beside the pass's; the call after it is served."""
    boards, legal, _, _ = chess.random_positions(3, 2, 0, 20)
    want = net.evaluate_packed(boards, legal)
    rules = Rules(70, np.array([[5, 70, 6, -1]], np.int32)).on_device()
    x, out = torch.zeros((1, 4), device="cuda:0"), torch.zeros((1, 4), device="cuda:0")
    net.adjust_logits(1, 4, x.data_ptr(), rules, out_ptr=out.data_ptr(), stream=here())
    torch.cuda.synchronize()
    with pytest.raises(NetworkError) as e:
        net.evaluate_packed(boards, legal)
    assert e.value.code == 7 and "rules.actions" in str(e.value)
    assert all(np.array_equal(a, b) for a, b in zip(net.evaluate_packed(boards, legal), want))


# Widths on both sides of a change of the kernel, of the columns that its threads hold, of the blocks of a row.
BORDERS = [63, 64, 65, 256, 257, 511, 512, 513, 16383, 16384, 16385, 32768, 32769, 65536, 65537]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", BORDERS)
def test_widths_where_the_kernels_change(net, width, dtype):  # noqa: F811
    rng = np.random.default_rng(width)
    rows = 3
    x = some_logits(rng, rows, width, dtype)
    t, u = (0.3 + rng.random(rows)).astype(np.float32), rng.random(rows).astype(np.float32)
    k, p = np.array([3, width // 3, width - 1], np.int32), rng.random(rows).astype(np.float32)
    for rules in (None, some_rules(rng, rows, width, width, False, history=700, bias=40),
                  some_rules(rng, rows, width, 2 * width, True, history=30, bias=5)):
        check_adjust(net, x, rules, t, dtype)
        for kk, pp in ((None, None), (k, None), (None, p), (k, p)):
            check_choose(net, x, rules, t, kk, pp, u, dtype)
    # few distinct values: the cut-offs fall among equals, and lists of one value overflow
    ties = torch.from_numpy(rng.integers(-1, 2, (rows, width)).astype(np.float32)).to("cuda:0").to(TYPES[dtype])
    ties[0] = 1.0
    for kk, pp in ((k, None), (None, p), (k, p)):
        check_choose(net, ties, None, t, kk, pp, u, dtype)
    assert net.status_word() == 0


@pytest.mark.parametrize("cut", ["none", "k", "p"])
@pytest.mark.parametrize("width", [50, 224, 512, 513, 4672, 16385, 40000])
def test_numbers_outside_the_unit_interval(net, width, cut):  # noqa: F811
    """From 1 on they draw the last column that is kept, below 0 and as NaN the first."""
    rng = np.random.default_rng(width)
    rows = 7
    x = some_logits(rng, rows, width, "f32")
    u = np.array([1, 2, np.inf, -1, -np.inf, np.nan, -0.0], np.float32)
    k = np.full(rows, 20, np.int32) if cut == "k" else None
    p = np.full(rows, 0.9, np.float32) if cut == "p" else None
    want = plain_choice(x.cpu().numpy(), None, k, p, np.array([2, 2, 2, 0, 0, 0, 0], np.float32))[0]
    assert np.array_equal(call_choose(net, x, None, None, k, p, u)[0], want)


@pytest.mark.parametrize("shift,width,rows", [(1, 224, 100), (2, 8, 20000), (3, 512, 17000), (0, 500, 20000),
                                              (0, 1000, 300), (1, 1001, 17000), (0, 30000, 5)])
@pytest.mark.parametrize("with_map", [False, True])
def test_slot_tables_anywhere(net, shift, width, rows, with_map):  # noqa: F811
    """Tables that start at any element, of widths above a position's slots, with and without the map."""
    rng = np.random.default_rng(width)
    lengths = rng.integers(0, min(width, 40) + 1, rows).astype(np.int32)
    lengths[rng.random(rows) < 0.02] = width
    count = int(lengths.sum())
    entries = rng.integers(0, 2**31 - 1, count).astype(np.int32)
    whole = torch.full((shift + (rows + 1) * width,), -6, dtype=torch.int32, device="cuda:0")
    starts = torch.full((rows + 2,), -5, dtype=torch.int32, device="cuda:0")
    where = torch.full((count + 3,), -7, dtype=torch.int32, device="cuda:0")
    le, en = dev(lengths), dev(entries)
    net.slot_table(rows, width, le.data_ptr(), count, en.data_ptr(), starts.data_ptr(), whole[shift:].data_ptr(),
                   where.data_ptr() if with_map else None, stream=here())
    torch.cuda.synchronize()
    want_starts, want, want_map = plain_slot_table(lengths, width, count, entries)
    assert (whole[:shift] == -6).all() and (whole[shift + rows * width:] == -6).all()
    assert np.array_equal(whole[shift: shift + rows * width].view(rows, width).cpu().numpy(), want)
    assert np.array_equal(starts[:-1].cpu().numpy(), want_starts) and int(starts[-1]) == -5
    assert np.array_equal(where[:count].cpu().numpy(), want_map if with_map else np.full(count, -7)) and (where[count:] == -7).all()
    assert net.status_word() == 0


def test_as_many_rows_as_there_may_be(net):  # noqa: F811
    rows = 1 << 27
    x = torch.full((1,), 2.0, device="cuda:0")
    column, action = (torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda:0") for _ in range(2))
    prob = torch.full((rows + 1,), -9.0, device="cuda:0")
    net.choose_actions(rows, 1, x.data_ptr(), None, column.data_ptr(), action.data_ptr(), prob.data_ptr(), stride=0,
                       stream=here())
    priors, out = torch.full((rows + 1,), -9.0, device="cuda:0"), torch.full((rows + 1,), -9.0, device="cuda:0")
    net.adjust_logits(rows, 1, x.data_ptr(), None, out.data_ptr(), priors.data_ptr(), stride=0, stream=here())
    torch.cuda.synchronize()
    for got, want in ((column, 0), (action, 0), (prob, 1), (priors, 1), (out, 2)):
        assert int((got[:-1] != want).sum()) == 0 and int(got[-1]) == -9


def test_threads_beside_passes(cuda):
    """Two threads run the operators on streams of theirs, a third on the context's own, while a fourth runs
    passes on the same context, the first of each batch size with its capture."""
    arch = model.Architecture(64, 1, 2, 128)
    ctx = B200Network(arch, weights.random_init(arch), device=0, max_batch=64, precision="bf16")
    boards, legal, _, _ = chess.random_positions(5, 64, 0, 40)
    states = [make_state(20 + i, rows=300) for i in range(3)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    failures, results = [], {}

    def run(call):
        try:
            call()
        except Exception as e:  # handed to the test's thread
            failures.append(e)

    def operators(i):
        for _ in range(100):
            together(ctx, states[i], streams[i].cuda_stream if i < 2 else None)

    def passes():
        for n in (1, 2, 3, 5, 9, 17, 33, 64, 40, 20, 10):
            results[n] = ctx.evaluate_packed(boards[:n], legal[:n])

    threads = [threading.Thread(target=run, args=(lambda i=i: operators(i),)) for i in range(3)]
    threads.append(threading.Thread(target=run, args=(passes,)))
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failures and not any(t.is_alive() for t in threads), failures
    torch.cuda.synchronize()
    for s in states:
        check_state(s)
    for n, got in results.items():
        assert all(np.array_equal(a, b) for a, b in zip(got, ctx.evaluate_packed(boards[:n], legal[:n])))
    assert ctx.status_word() == 0
    ctx.close()


def test_large_calls_in_a_graph(net):  # noqa: F811
    """A slot table in three launches, rows of several blocks and long lists over wide slot rows, captured once
    and replayed with other inputs in the same buffers."""
    rows, width, tall = 4, 20000, 20000
    rng = np.random.default_rng(4)
    lengths, entries = torch.zeros(tall, dtype=torch.int32, device="cuda:0"), torch.zeros(9 * tall, dtype=torch.int32, device="cuda:0")
    starts, table = torch.zeros(tall + 1, dtype=torch.int32, device="cuda:0"), torch.zeros((tall, 9), dtype=torch.int32, device="cuda:0")
    where = torch.zeros(9 * tall, dtype=torch.int32, device="cuda:0")
    rules = some_rules(rng, rows, width, 2 * width, True, history=300, bias=50)
    r = rules.on_device()
    x, out, priors = (torch.zeros((rows, width), device="cuda:0") for _ in range(3))
    u, p = torch.zeros(rows, device="cuda:0"), torch.full((rows,), 0.8, device="cuda:0")
    column = torch.zeros(rows, dtype=torch.int32, device="cuda:0")

    def calls():
        s = torch.cuda.current_stream().cuda_stream
        net.slot_table(tall, 9, lengths.data_ptr(), 9 * tall, entries.data_ptr(), starts.data_ptr(), table.data_ptr(),
                       where.data_ptr(), stream=s)
        net.adjust_logits(rows, width, x.data_ptr(), r, out_ptr=out.data_ptr(), priors_ptr=priors.data_ptr(), stream=s)
        net.choose_actions(rows, width, x.data_ptr(), r, column.data_ptr(), top_p_ptr=p.data_ptr(), uniform_ptr=u.data_ptr(),
                           stream=s)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for _ in range(3):
        n = rng.integers(0, 10, tall).astype(np.int32)
        e = rng.integers(0, 99, 9 * tall).astype(np.int32)
        lengths.copy_(dev(n)), entries.copy_(dev(e)), where.fill_(-7)
        x.copy_(some_logits(rng, rows, width, "f32")), u.copy_(torch.rand(rows, device="cuda:0"))
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((starts, table, where), plain_slot_table(n, 9, 9 * tall, e)):
            assert np.array_equal(got.cpu().numpy(), want)
        a = plain_adjusted(x.cpu().numpy(), rules)
        assert np.array_equal(out.cpu().numpy(), a)
        check_priors(priors.cpu().numpy(), a, None)
        assert np.array_equal(column.cpu().numpy(), plain_choice(a, None, None, p.cpu().numpy(), u.cpu().numpy())[0])
    assert net.status_word() == 0
