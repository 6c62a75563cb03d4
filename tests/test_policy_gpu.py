"""The policy operators on the GPU -- slot tables, adjusted logits, the choice of an action -- against
plain implementations of their definitions: whole numbers and adjusted logits to the bit (the
definition fixes each f32 rounding), priors and probabilities against 64-bit arithmetic within bounds
derived beside them."""

import numpy as np
import pytest

from marina_b200 import model, weights
from marina_b200.network import B200Network, LogitRules

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module")
def net(cuda):
    arch = model.Architecture(64, 1, 2, 128)
    n = B200Network(arch, weights.random_init(arch), device=0, max_batch=4, precision="bf16")
    yield n
    n.close()


@pytest.fixture(autouse=True)
def clean_status(net):
    yield
    torch.cuda.synchronize()
    net.status_word()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def here():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream


# ---- plain implementations ------------------------------------------------------------------
def plain_slot_table(lengths, width, count, entries):
    n = np.clip(lengths.astype(np.int64), 0, width)
    starts = np.concatenate([[0], np.cumsum(n)])
    table = np.full((len(n), width), -1, np.int32)
    where = np.full(count, -7, np.int32)
    for r in range(len(n)):
        for s in range(n[r]):
            if starts[r] + s < count:
                table[r, s] = entries[starts[r] + s]
                where[starts[r] + s] = r * width + s
    return starts.astype(np.int32), table, where


class Rules:
    """The rules of a batch as numpy arrays, [rows or 1, ...]."""

    def __init__(self, actions, columns=None, mask=None, bias=None, history=None, lens=None, repetition=None,
                 presence=None, frequency=None):
        self.actions, self.columns, self.mask, self.bias = actions, columns, mask, bias
        self.history, self.lens = history, lens
        self.repetition, self.presence, self.frequency = repetition, presence, frequency

    def on_device(self):
        keep, parts = [], {}

        def put(name, a, stride=None):
            if a is None:
                return
            keep.append(dev(a))
            parts[name] = keep[-1].data_ptr()
            if stride:
                parts[stride] = 0 if a.shape[0] == 1 else a.shape[1]

        put("columns", self.columns, "columns_stride")
        if self.mask is not None:
            put("mask", pack_bits(self.mask).view(np.int32), "mask_stride")
        if self.bias is not None:
            put("bias_actions", self.bias[0], "bias_stride")
            put("bias_values", self.bias[1])
            parts["bias_len"] = self.bias[0].shape[1]
        if self.history is not None:
            put("history", self.history, "history_stride")
            parts["history_len"] = self.history.shape[1]
            put("history_lens", self.lens)
            for name in ("repetition", "presence", "frequency"):
                put(name, getattr(self, name))
        r = LogitRules(self.actions, **parts)
        r.keep = keep
        return r


def pack_bits(allowed):
    rows, actions = allowed.shape
    words = (actions + 31) // 32
    full = np.zeros((rows, words * 32), np.uint8)
    full[:, :actions] = allowed
    return np.packbits(full, axis=1, bitorder="little").view(np.uint32)


def of_row(a, r):
    return None if a is None else a[0 if a.shape[0] == 1 else r]


def plain_adjusted(x, rules):
    """[rows, width] f32 logits under `rules`, each step rounded to f32."""
    x = x.astype(np.float32).copy()
    if rules is None:
        return x
    f = np.float32
    with np.errstate(all="ignore"):
        for r in range(x.shape[0]):
            ids = of_row(rules.columns, r)
            ids = np.arange(x.shape[1]) if ids is None else ids.astype(np.int64)
            live = (ids >= 0) & (ids < rules.actions)
            safe = np.where(live, ids, 0)
            if rules.history is not None:
                h = of_row(rules.history, r)
                if rules.lens is not None:
                    h = h[: min(max(int(rules.lens[r]), 0), len(h))]
                h = h[(h >= 0) & (h < rules.actions)]
                c = np.where(live, np.bincount(h, minlength=rules.actions)[safe], 0)
                rep, pre, fre = (f(d) if a is None else a[r] for a, d in
                                 ((rules.repetition, 1), (rules.presence, 0), (rules.frequency, 0)))
                y = np.where(x[r] > 0, x[r] / rep, x[r] * rep).astype(f)
                y = ((y - (fre * c.astype(f)).astype(f)).astype(f) - pre).astype(f)
                x[r] = np.where(c > 0, y, x[r])
            if rules.bias is not None:
                for a, v in zip(of_row(rules.bias[0], r), of_row(rules.bias[1], r)):
                    if 0 <= a < rules.actions:
                        x[r, live & (ids == a)] += v
            if rules.mask is not None:
                live = live & of_row(rules.mask, r)[safe]
            x[r, ~live] = -np.inf
    return x


def plain_priors(x, t):
    """64-bit softmax of adjusted logits [rows, width] at temperatures t, by the header's rules."""
    out = np.zeros(x.shape)
    for r in range(x.shape[0]):
        v, tr = x[r].astype(np.float64), 1.0 if t is None else float(t[r])
        left = ~(v == -np.inf)
        if np.isnan(v).any() or np.isnan(tr):
            out[r, left] = np.nan
        elif left.any():
            m = v.max()
            if tr <= 0:
                out[r, np.argmax(v)] = 1
            elif m == np.inf:
                out[r] = (v == m) / (v == m).sum()
            else:
                e = np.where(left, np.exp((v - m) / tr), 0)
                out[r] = e / e.sum()
    return out


def plain_choice(x, t, top_k, top_p, uniform):
    rows = x.shape[0]
    column, prob = np.full(rows, -1, np.int32), np.zeros(rows)
    for r in range(rows):
        v, tr = x[r].astype(np.float64), 1.0 if t is None else float(t[r])
        if np.isnan(v).any() or np.isnan(tr):
            prob[r] = np.nan
            continue
        left = np.flatnonzero(v > -np.inf)
        if not left.size:
            continue
        best = left[np.argsort(-v[left], kind="stable")]
        if tr <= 0:
            column[r], prob[r] = best[0], 1
            continue
        k = 0 if top_k is None else int(top_k[r])
        best = best[:k] if k > 0 else best
        m = v[best[0]]
        w = (v[best] == m).astype(np.float64) if m == np.inf else np.exp((v[best] - m) / tr)
        p = np.float64(1.0 if top_p is None else top_p[r])
        if p < 1:
            ahead = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            keep = (ahead < p * w.sum()) | (np.arange(w.size) == 0)
            best, w = best[keep], w[keep]
        total = w.sum()
        if uniform is None:
            column[r], prob[r] = best[0], w[0] / total
            continue
        order = np.argsort(best)
        best, w = best[order], w[order]
        at = min(int(np.searchsorted(np.cumsum(w), float(uniform[r]) * total, side="right")), w.size - 1)
        while w[at] == 0:  # only at the last border of the row
            at -= 1
        column[r], prob[r] = best[at], w[at] / total
    return column, prob


# ---- calls -----------------------------------------------------------------------------------
def call_adjust(net, x, rules, t, out=True, priors=True, dtype="f32"):
    rows, width = x.shape
    o = torch.full_like(x, 5.0) if out else None
    q = torch.full((rows, width), 5.0, device="cuda:0") if priors else None
    r = None if rules is None else rules.on_device()
    tt = None if t is None else dev(t)
    net.adjust_logits(rows, width, x.data_ptr(), r, dtype=dtype, out_ptr=None if o is None else o.data_ptr(),
                      priors_ptr=None if q is None else q.data_ptr(), stride=x.stride(0),
                      temperature_ptr=None if tt is None else tt.data_ptr(), out_stride=width, stream=here())
    torch.cuda.synchronize()
    return (None if o is None else o.float().cpu().numpy()), (None if q is None else q.cpu().numpy())


def call_choose(net, x, rules, t, top_k, top_p, uniform, dtype="f32"):
    rows, width = x.shape
    col, act = (torch.full((rows,), -9, dtype=torch.int32, device="cuda:0") for _ in range(2))
    prob = torch.full((rows,), 5.0, device="cuda:0")
    r = None if rules is None else rules.on_device()
    a = [None if v is None else dev(v) for v in (t, top_k, top_p, uniform)]
    ptr = [None if v is None else v.data_ptr() for v in a]
    net.choose_actions(rows, width, x.data_ptr(), r, col.data_ptr(), act.data_ptr(), prob.data_ptr(), dtype=dtype,
                       stride=x.stride(0), temperature_ptr=ptr[0], top_k_ptr=ptr[1], top_p_ptr=ptr[2],
                       uniform_ptr=ptr[3], stream=here())
    torch.cuda.synchronize()
    return col.cpu().numpy(), act.cpu().numpy(), prob.cpu().numpy()


def check_priors(got, x, t):
    want = plain_priors(x, t)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # An exponent z = (x - m) / t has two roundings (z up to |z| U off each), the exponential one step
    # (2 U) and at most 2 U more where it runs as a power of two (a product and its rounding of a
    # z * log2(e): |z| U again); sums of `width` terms in a fixed tree are off by U for each addition a
    # term passes, at most width / 32 + 32 of them however a row is split; the quotient is two more.
    with np.errstate(all="ignore"):
        m = np.nanmax(np.where(x == -np.inf, -3e38, x), axis=1, keepdims=True).astype(np.float64)
        tt = np.ones((x.shape[0], 1)) if t is None else t.astype(np.float64)[:, None]
        z = np.where((x > -np.inf) & (tt > 0) & np.isfinite(m), np.abs((x - m) / tt), 0.0)
        # the row's sum carries the errors of its terms, weighted by their shares
        mean_z = np.nansum(np.where(want > 0, want * z, 0), axis=1, keepdims=True)
        bound = want * U * (4 * z + 4 * mean_z + x.shape[1] / 32 + 48) + 2.0 ** -125
    ok = np.isnan(want) | (np.abs(got - want) <= bound)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5])
    assert (got[x == -np.inf] == 0).all()


def rounded(x, dtype):
    return torch.from_numpy(x).to(TYPES[dtype]).float().numpy()


def check_adjust(net, x, rules, t, dtype="f32", **kw):
    a = plain_adjusted(x.float().cpu().numpy(), rules)
    out, priors = call_adjust(net, x, rules, t, dtype=dtype, **kw)
    if out is not None:
        assert np.array_equal(out, rounded(a, dtype), equal_nan=True)
    if priors is not None:
        check_priors(priors, a, t)


def check_choose(net, x, rules, t, top_k, top_p, uniform, dtype="f32"):
    a = plain_adjusted(x.float().cpu().numpy(), rules)
    want, want_prob = plain_choice(a, t, top_k, top_p, uniform)
    col, act, prob = call_choose(net, x, rules, t, top_k, top_p, uniform, dtype)
    assert np.array_equal(col, want), np.argwhere(col != want)[:5].tolist()
    if rules is not None and rules.columns is not None:
        rows = np.arange(len(col))
        c = rules.columns if rules.columns.shape[0] > 1 else np.repeat(rules.columns, len(col), 0)
        want_act = np.where(col >= 0, c[rows, np.maximum(col, 0)], -1)
    else:
        want_act = col
    assert np.array_equal(act, want_act)
    assert np.array_equal(np.isnan(prob), np.isnan(want_prob))
    # One rounding to f32 of a quotient of whole multiples of 2^-40: each term is half of one off.
    fine = ~np.isnan(want_prob)
    assert (np.abs(prob - want_prob)[fine] <= want_prob[fine] * 2 * U + a.shape[1] * 2.0 ** -41).all()


def some_rules(rng, rows, width, actions, slots, history=24, bias=6, masked=True, shared=False):
    n = 1 if shared else rows
    columns = None
    if slots:
        columns = np.stack([rng.permutation(actions)[:width] for _ in range(rows)]).astype(np.int32)
        for r in range(rows):
            columns[r, rng.integers(0, width + 1):] = -1
    mask = rng.random((n, actions)) < 0.4 if masked else None
    pick = rng.integers(-2, min(actions, 4 * history + 4), (rows, max(history, 1))).astype(np.int32)
    if slots:
        near = np.take_along_axis(columns, rng.integers(0, width, pick.shape), 1)
        pick = np.where(rng.random(pick.shape) < 0.8, near, pick).astype(np.int32)
    return Rules(actions, columns, mask,
                 None if not bias else (rng.integers(-1, actions + 2, (n, bias)).astype(np.int32),
                                        rng.standard_normal((n, bias)).astype(np.float32)),
                 pick if history else None, rng.integers(-1, history + 3, rows).astype(np.int32) if history else None,
                 (1 + rng.random(rows)).astype(np.float32), rng.random(rows).astype(np.float32),
                 rng.random(rows).astype(np.float32) / 4)


def some_logits(rng, rows, width, dtype):
    return torch.from_numpy((rng.standard_normal((rows, width)) * 3).astype(np.float32)).to("cuda:0").to(TYPES[dtype])


# ---- slot tables -----------------------------------------------------------------------------
def run_slot_table(net, lengths, width, count, entries):
    rows = len(lengths)
    starts = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda:0")
    table = torch.full((rows + 1, width), -6, dtype=torch.int32, device="cuda:0")
    where = torch.full((count + 3,), -7, dtype=torch.int32, device="cuda:0")
    le, en = dev(lengths), dev(entries)
    net.slot_table(rows, width, le.data_ptr(), count, en.data_ptr(), starts.data_ptr(), table.data_ptr(),
                   where.data_ptr(), stream=here())
    torch.cuda.synchronize()
    assert (table[rows] == -6).all() and (where[count:] == -7).all()  # nothing behind the last row
    return starts.cpu().numpy(), table[:rows].cpu().numpy(), where[:count].cpu().numpy()


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 224), (3, 7), (31, 224), (33, 33), (257, 224), (1000, 5),
                                        (2049, 224), (4096, 100), (40001, 16), (70000, 3)])
def test_slot_table(net, rows, width):
    rng = np.random.default_rng(rows + width)
    lengths = rng.integers(0, width + 1, rows).astype(np.int32)
    lengths[rng.random(rows) < 0.2] = 0
    lengths[rng.random(rows) < 0.1] = width
    total = int(lengths.sum())
    entries = rng.integers(0, 4672, max(total, 1)).astype(np.int32)
    for got, want in zip(run_slot_table(net, lengths, width, total, entries),
                         plain_slot_table(lengths, width, total, entries)):
        assert np.array_equal(got, want)
    assert net.status_word() == 0


@pytest.mark.parametrize("rows", [5, 3000, 20000])
@pytest.mark.parametrize("fault", ["short", "negative", "long", "unused"])
def test_slot_table_of_lists_that_do_not_fit(net, rows, fault):
    rng = np.random.default_rng(rows)
    width = 9
    lengths = rng.integers(0, width + 1, rows).astype(np.int32)
    if fault == "negative":
        lengths[rows // 2] = -2**31
    if fault == "long":
        lengths[rows // 2] = 2**31 - 1
    total = int(np.clip(lengths.astype(np.int64), 0, width).sum())
    count = total - 11 if fault == "short" else total + 40 if fault == "unused" else total
    entries = rng.integers(0, 99, count).astype(np.int32)
    for got, want in zip(run_slot_table(net, lengths, width, count, entries),
                         plain_slot_table(lengths, width, count, entries)):
        assert np.array_equal(got, want)
    assert net.status_word() == (0 if fault == "unused" else 17)


def test_slot_table_of_nothing(net):
    starts = torch.full((1,), -5, dtype=torch.int32, device="cuda:0")
    net.slot_table(0, 224, None, 0, None, starts.data_ptr(), None, stream=here())
    torch.cuda.synchronize()
    assert int(starts) == 0
    lengths = np.zeros(4, np.int32)
    s, t, _ = run_slot_table(net, lengths, 8, 0, np.zeros(1, np.int32))
    assert (s == 0).all() and (t == -1).all()


# ---- adjusted logits and the choice ----------------------------------------------------------
SHAPES = [  # rows, width, actions, slots
    (1, 1, 1, False), (1, 224, 4672, True), (5, 7, 40, True), (9, 32, 33, True), (67, 224, 4672, True),
    (300, 35, 4672, True), (3, 500, 600, True), (2, 1025, 4672, True), (2, 4672, 4672, False), (5, 4097, 5000, False),
    (3, 255, 255, False), (70, 256, 256, False), (9, 257, 300, False), (4, 1023, 1023, False), (3, 8193, 8193, False),
    (2, 20011, 20011, False), (2, 50021, 50021, False), (1, 131072, 131072, False), (1, 262144, 262144, False),
    (200, 33000, 33000, False),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,actions,slots", SHAPES)
def test_adjust(net, rows, width, actions, slots, dtype):
    rng = np.random.default_rng(width)
    x = some_logits(rng, rows, width, dtype)
    rules = some_rules(rng, rows, width, actions, slots)
    t = (0.3 + rng.random(rows)).astype(np.float32)
    check_adjust(net, x, rules, t, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,actions,slots", SHAPES)
def test_choose(net, rows, width, actions, slots, dtype):
    rng = np.random.default_rng(width + 1)
    x = some_logits(rng, rows, width, dtype)
    rules = some_rules(rng, rows, width, actions, slots)
    t = (0.3 + rng.random(rows)).astype(np.float32)
    t[rng.random(rows) < 0.1] = 0
    k = rng.integers(-1, max(2, width // 2), rows).astype(np.int32)
    p = rng.random(rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    for kk in (None, k):
        for pp in (None, p):
            check_choose(net, x, rules, t, kk, pp, u, dtype)
    check_choose(net, x, rules, t, k, p, None, dtype)


PARTS = [dict(history=0, bias=0, masked=False), dict(history=0, bias=0), dict(history=0, masked=False),
         dict(bias=0, masked=False), dict(history=300, bias=70, shared=True), dict(history=1, bias=1),
         dict(history=5000, bias=200)]


@pytest.mark.parametrize("parts", PARTS)
@pytest.mark.parametrize("rows,width,slots", [(6, 100, True), (6, 224, True), (5, 700, True), (3, 224, False), (3, 6000, False),
                                              (2, 40000, False)])
def test_parts_of_the_rules(net, rows, width, slots, parts):
    rng = np.random.default_rng(width)
    actions = 4672 if slots else width
    x = some_logits(rng, rows, width, "f32")
    rules = some_rules(rng, rows, width, actions, slots, **parts)
    t = (0.3 + rng.random(rows)).astype(np.float32)
    check_adjust(net, x, rules, t)
    check_adjust(net, x, rules, None, out=False)
    check_adjust(net, x, rules, t, priors=False)
    check_choose(net, x, rules, t, None, (0.5 + rng.random(rows) / 2).astype(np.float32),
                 rng.random(rows).astype(np.float32))
    assert net.status_word() == 0


@pytest.mark.parametrize("width", [64, 224, 5000, 70000])
def test_without_rules(net, width):
    rng = np.random.default_rng(width)
    x = some_logits(rng, 3, width, "f32")
    check_adjust(net, x, None, None)
    check_choose(net, x, None, None, None, None, rng.random(3).astype(np.float32))
    check_choose(net, x, None, None, None, None, None)
    # penalties of 1 and 0 where the arrays are absent
    h = rng.integers(0, width, (3, 9)).astype(np.int32)
    check_adjust(net, x, Rules(width, history=h), None)
    check_adjust(net, x, Rules(width, history=h[:1], frequency=np.full(3, 0.5, np.float32)), None)


@pytest.mark.parametrize("width", [100, 224, 300, 5000, 40000])
def test_rows_that_need_a_rule(net, width):
    """Empty rows, NaN and infinities in masked places and in places that are left, a lone column,
    zeros of both signs, temperatures at their ends."""
    rows = 14
    rng = np.random.default_rng(width)
    x = (rng.standard_normal((rows, width)) * 2).astype(np.float32)
    mask = rng.random((rows, width)) < 0.5
    x[~mask] = rng.choice([np.nan, np.inf, -np.inf, 3e38], size=int((~mask).sum()))
    mask[0] = False                          # nothing left
    mask[1] = False
    mask[1, width // 3] = True               # one left
    x[1, width // 3] = -40
    x[2, mask[2]] = -np.inf                  # left, but at -inf
    x[3, np.flatnonzero(mask[3])[2]] = np.nan
    x[4, np.flatnonzero(mask[4])[[1, 4]]] = np.inf
    x[5, mask[5]] = rng.choice([0.0, -0.0], size=int(mask[5].sum()))
    x[6, mask[6]] = -3e38
    x[6, np.flatnonzero(mask[6])[3]] = 3e38
    x[11, np.flatnonzero(mask[11])[0]] = np.inf
    t = np.ones(rows, np.float32)
    t[7], t[8], t[9], t[10], t[11] = 0, np.inf, np.nan, 1e-30, np.inf
    t[12], t[13] = -1, 1e30
    xd = dev(x)
    rules = Rules(width, mask=mask)
    check_adjust(net, xd, rules, t)
    u = rng.random(rows).astype(np.float32)
    for k in (None, np.full(rows, 3, np.int32)):
        for p in (None, np.full(rows, 0.6, np.float32)):
            for uu in (u, np.zeros(rows, np.float32), np.full(rows, 1 - 2.0 ** -24, np.float32), None):
                check_choose(net, xd, rules, t, k, p, uu)


@pytest.mark.parametrize("width", [50, 224, 4672, 30000])
def test_cutoffs_at_their_ends(net, width):
    rng = np.random.default_rng(width)
    rows = 12
    x = some_logits(rng, rows, width, "f32")
    u = rng.random(rows).astype(np.float32)
    k = np.array([1, 2, width - 1, width, width + 1, 2**31 - 1, 0, -1, -2**31, 3, width // 2, 7], np.int32)
    p = np.array([0, -1, 1, 2, np.nan, 1e-30, 0.5, 1 - 2.0 ** -24, np.inf, -np.inf, 0.25, 0.75], np.float32)
    check_choose(net, x, None, None, k, None, u)
    check_choose(net, x, None, None, None, p, u)
    check_choose(net, x, None, None, k, p, u)
    check_choose(net, x, None, None, k[::-1].copy(), p, u)
    # numbers outside [0, 1) are taken as its nearest end; NaN as 0
    col, _, _ = call_choose(net, x, None, None, None, None,
                            np.array([1, 2, np.inf, -1, -np.inf, np.nan] * 2, np.float32))
    low, _, _ = call_choose(net, x, None, None, None, None, np.zeros(rows, np.float32))
    assert np.array_equal(col.reshape(2, 6)[:, 3:], low.reshape(2, 6)[:, 3:])
    assert (col >= low).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [60, 224, 4672, 40000])
def test_ties_go_to_the_lower_column(net, width, dtype):
    """Rows of few distinct values: every cut-off falls among equals."""
    rng = np.random.default_rng(width)
    rows = 10
    x = torch.from_numpy(rng.integers(-2, 3, (rows, width)).astype(np.float32)).to("cuda:0").to(TYPES[dtype])
    x[0] = 1.0  # all equal
    for seed in range(3):
        u = rng.random(rows).astype(np.float32)
        k = rng.integers(1, width, rows).astype(np.int32)
        p = rng.random(rows).astype(np.float32)
        check_choose(net, x, None, None, k, None, u, dtype)
        check_choose(net, x, None, None, k, p, u, dtype)
    check_choose(net, x, None, None, None, None, None, dtype)
    check_choose(net, x, None, np.zeros(rows, np.float32), None, None, u, dtype)


@pytest.mark.parametrize("width", [40, 224, 900])
def test_the_same_action_twice(net, width):
    """An action in two slots, twice in the bias list (values whose sum depends on the order) and many
    times in the history."""
    rng = np.random.default_rng(width)
    rows, actions = 4, 60
    columns = rng.integers(-1, actions, (rows, width)).astype(np.int32)
    ids = rng.integers(0, 6, (rows, 40)).astype(np.int32)
    values = (rng.standard_normal((rows, 40)) * 10.0 ** rng.integers(-4, 5, (rows, 40))).astype(np.float32)
    rules = Rules(actions, columns, None, (ids, values), rng.integers(0, 9, (rows, 500)).astype(np.int32))
    rules.frequency = np.full(rows, 0.01, np.float32)
    x = some_logits(rng, rows, width, "f32")
    check_adjust(net, x, rules, None)
    check_choose(net, x, rules, None, None, None, rng.random(rows).astype(np.float32))
    # and without slots
    rules.columns, rules.actions = None, width
    check_adjust(net, x, rules, None)


@pytest.mark.parametrize("width,slots", [(12, True), (600, True)])
def test_ids_outside_the_actions(net, width, slots):
    rng = np.random.default_rng(3)
    rows, actions = 5, 70
    rules = some_rules(rng, rows, min(width, 70), actions, True)
    columns = np.full((rows, width), -1, np.int32)
    columns[:, : rules.columns.shape[1]] = rules.columns
    rules.columns = columns
    columns[1, 2], columns[3, 0], columns[4, 5] = actions, 2**31 - 1, -2**31
    x = some_logits(rng, rows, width, "f32")
    check_adjust(net, x, rules, None)
    assert net.status_word() == 16
    check_choose(net, x, rules, None, None, None, rng.random(rows).astype(np.float32))
    assert net.status_word() == 16


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("width", [33, 224, 1000, 4672, 40001])
@pytest.mark.parametrize("shift,pad", [(1, 3), (2, 6), (4, 4), (3, 0)])
def test_rows_anywhere(net, width, shift, pad, dtype):
    """Rows that start at any element and lie any distance apart, outputs beside the logits, and in
    place; nothing around them changes."""
    rng = np.random.default_rng(width + shift)
    rows, stride = 5, width + pad
    big = some_logits(rng, 1, shift + rows * stride + 8, dtype)[0]
    x = big[shift: shift + rows * stride].view(rows, stride)[:, :width]
    rules = some_rules(rng, rows, width, width, False)
    a = plain_adjusted(x.float().cpu().numpy(), rules)
    r = rules.on_device()
    before = big.clone()
    out = torch.full_like(big, 9.0)
    pri = torch.full((big.numel(),), 9.0, device="cuda:0")
    net.adjust_logits(rows, width, x.data_ptr(), r, dtype=dtype, stride=stride,
                      out_ptr=out[shift + 1:].data_ptr(), out_stride=stride, priors_ptr=pri[shift + 2:].data_ptr(),
                      priors_stride=stride, stream=here())
    torch.cuda.synchronize()
    assert torch.equal(big, before)
    for buf, at in ((out, shift + 1), (pri, shift + 2)):
        rest = torch.ones_like(buf, dtype=torch.bool)
        for q in range(rows):
            rest[at + q * stride: at + q * stride + width] = False
        assert (buf[rest] == 9).all()
    got = torch.as_strided(out, (rows, width), (stride, 1), shift + 1).float().cpu().numpy()
    assert np.array_equal(got, rounded(a, dtype))
    check_priors(torch.as_strided(pri, (rows, width), (stride, 1), shift + 2).cpu().numpy(), a, None)
    u = rng.random(rows).astype(np.float32)
    check_choose(net, x, rules, None, None, None, u, dtype)
    # in place, with the priors at the same time
    pri.fill_(9.0)
    net.adjust_logits(rows, width, x.data_ptr(), r, dtype=dtype, stride=stride, out_ptr=x.data_ptr(), out_stride=stride,
                      priors_ptr=pri.data_ptr(), stream=here())
    torch.cuda.synchronize()
    assert np.array_equal(x.float().cpu().numpy(), rounded(a, dtype))
    check_priors(pri[: rows * width].view(rows, width).cpu().numpy(), a, None)
    rest = torch.ones_like(big, dtype=torch.bool)
    for q in range(rows):
        rest[shift + q * stride: shift + q * stride + width] = False
    assert torch.equal(big[rest], before[rest])


def test_one_row_for_all(net):
    """A stride of 0: every row reads the same logits, slots, mask and lists."""
    rng = np.random.default_rng(8)
    rows, width = 20, 224
    x = some_logits(rng, 1, width, "f32")
    rules = some_rules(rng, 1, width, 4672, True, shared=True)
    rules.lens = rules.repetition = rules.presence = rules.frequency = None
    t = (0.2 + rng.random(rows)).astype(np.float32)
    want = np.repeat(plain_adjusted(x.cpu().numpy(), rules), rows, 0)
    out, pri = torch.empty((rows, width), device="cuda:0"), torch.empty((rows, width), device="cuda:0")
    r, td = rules.on_device(), dev(t)
    net.adjust_logits(rows, width, x.data_ptr(), r, stride=0, out_ptr=out.data_ptr(), priors_ptr=pri.data_ptr(),
                      temperature_ptr=td.data_ptr(), stream=here())
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    check_priors(pri.cpu().numpy(), want, t)


def test_rows_far_apart(net):
    """Offsets that pass 32 bits: three rows 1.2e9 elements apart."""
    rng = np.random.default_rng(9)
    rows, width, stride = 3, 5001, 1_200_000_007
    big = torch.empty(2 * stride + width, dtype=torch.float16, device="cuda:0")
    x = torch.as_strided(big, (rows, width), (stride, 1))
    x.copy_(some_logits(rng, rows, width, "f16"))
    rules = some_rules(rng, rows, width, width, False)
    a = plain_adjusted(x.float().cpu().numpy(), rules)
    check_choose(net, x, rules, None, None, None, rng.random(rows).astype(np.float32), "f16")
    r = rules.on_device()
    net.adjust_logits(rows, width, x.data_ptr(), r, dtype="f16", stride=stride, out_ptr=x.data_ptr(), out_stride=stride,
                      stream=here())
    torch.cuda.synchronize()
    assert np.array_equal(x.float().cpu().numpy(), rounded(a, "f16"))


# ---- streams, graphs, and the three together ---------------------------------------------------
def together(net, state, stream):
    s = state
    net.slot_table(s["rows"], 224, s["lengths"].data_ptr(), s["count"], s["entries"].data_ptr(), s["starts"].data_ptr(),
                   s["table"].data_ptr(), s["map"].data_ptr(), stream=stream)
    net.adjust_logits(s["rows"], 224, s["logits"].data_ptr(), s["rules"], out_ptr=s["out"].data_ptr(),
                      priors_ptr=s["priors"].data_ptr(), stream=stream)
    net.choose_actions(s["rows"], 224, s["out"].data_ptr(), s["plain"], s["column"].data_ptr(), s["action"].data_ptr(),
                       s["prob"].data_ptr(), top_p_ptr=s["top_p"].data_ptr(), uniform_ptr=s["uniform"].data_ptr(),
                       stream=stream)


def make_state(seed, rows=50):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, 60, rows).astype(np.int32)
    lengths[0], lengths[1] = 0, 224
    entries = np.concatenate([np.sort(rng.permutation(4672)[:n]) for n in lengths]).astype(np.int32)
    s = {"rows": rows, "count": len(entries), "lengths": dev(lengths), "entries": dev(entries),
         "starts": torch.zeros(rows + 1, dtype=torch.int32, device="cuda:0"),
         "table": torch.zeros((rows, 224), dtype=torch.int32, device="cuda:0"),
         "map": torch.zeros(len(entries), dtype=torch.int32, device="cuda:0"),
         "logits": some_logits(rng, rows, 224, "f32"), "out": torch.zeros((rows, 224), device="cuda:0"),
         "priors": torch.zeros((rows, 224), device="cuda:0"),
         "column": torch.zeros(rows, dtype=torch.int32, device="cuda:0"),
         "action": torch.zeros(rows, dtype=torch.int32, device="cuda:0"), "prob": torch.zeros(rows, device="cuda:0"),
         "top_p": dev(rng.random(rows).astype(np.float32)), "uniform": dev(rng.random(rows).astype(np.float32)),
         "history": dev(np.stack([rng.permutation(entries)[:30] for _ in range(rows)]).astype(np.int32)),
         "repetition": dev((1 + rng.random(rows)).astype(np.float32))}
    s["rules"] = LogitRules(4672, columns=s["table"].data_ptr(), columns_stride=224, history=s["history"].data_ptr(),
                            history_len=30, history_stride=30, repetition=s["repetition"].data_ptr())
    s["plain"] = LogitRules(4672, columns=s["table"].data_ptr(), columns_stride=224)
    return s


def check_state(s):
    lengths, entries = s["lengths"].cpu().numpy(), s["entries"].cpu().numpy()
    starts, table, where = plain_slot_table(lengths, 224, s["count"], entries)
    assert np.array_equal(s["starts"].cpu().numpy(), starts) and np.array_equal(s["table"].cpu().numpy(), table)
    assert np.array_equal(s["map"].cpu().numpy(), where)
    rules = Rules(4672, table, history=s["history"].cpu().numpy(), repetition=s["repetition"].cpu().numpy())
    a = plain_adjusted(s["logits"].cpu().numpy(), rules)
    assert np.array_equal(s["out"].cpu().numpy(), a)
    check_priors(s["priors"].cpu().numpy(), a, None)
    want, _ = plain_choice(a, None, None, s["top_p"].cpu().numpy(), s["uniform"].cpu().numpy())
    assert np.array_equal(s["column"].cpu().numpy(), want)
    rows = np.arange(s["rows"])
    assert np.array_equal(s["action"].cpu().numpy(), np.where(want >= 0, table[rows, np.maximum(want, 0)], -1))


def test_together_on_a_stream_and_in_two_graphs(net):
    """The three operators in a row: eagerly on a stream of the caller's, and as two captured graphs
    replayed at the same time on two streams, with new inputs in their buffers."""
    a, b = make_state(1), make_state(2, rows=77)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    together(net, a, s1.cuda_stream)
    together(net, b, s2.cuda_stream)
    torch.cuda.synchronize()
    check_state(a), check_state(b)
    graphs = []
    for state in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            together(net, state, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for seed in (3, 4):
        for state, other in ((a, make_state(seed)), (b, make_state(seed + 10, rows=77))):
            n = min(state["count"], other["count"])
            lengths = other["lengths"].clone()
            # the captured calls name their number of entries: cut the new lists to it
            over = int(lengths.sum()) - n
            for r in range(len(lengths) - 1, -1, -1):
                cut = min(over, int(lengths[r]))
                lengths[r] -= cut
                over -= cut
            state["lengths"].copy_(lengths)
            state["entries"][:n].copy_(other["entries"][:n])
            for name in ("logits", "uniform", "top_p", "history", "repetition"):
                state[name].copy_(other[name])
            state["map"].fill_(-7)
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
        torch.cuda.synchronize()
        check_state(a), check_state(b)
    assert net.status_word() == 0


def test_same_bits_every_time(net):
    rng = np.random.default_rng(5)
    for rows, width in ((40, 224), (7, 4672), (2, 60001)):
        x = some_logits(rng, rows, width, "f32")
        rules = some_rules(rng, rows, width, width, False)
        first = call_adjust(net, x, rules, None)[1]
        for _ in range(3):
            assert np.array_equal(call_adjust(net, x, rules, None)[1], first)


def test_the_context_s_own_stream_and_the_callers_device(net):
    """stream None is the context's own; the caller's current device stays what it was."""
    s = make_state(6)
    torch.cuda.synchronize()
    together(net, s, None)
    torch.cuda.synchronize()
    check_state(s)
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("width", [224, 513, 4672, 20011])
def test_cutoffs_around_the_short_way(net, width, masked):
    """top_k on both sides of what one warp or block draws from, and top_p alone over equal logits."""
    rng = np.random.default_rng(width + 7)
    ks = [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 400]
    rows = len(ks)
    x = some_logits(rng, rows, width, "f32")
    rules = Rules(width, mask=rng.random((rows, width)) < 0.3) if masked else None
    u, k = rng.random(rows).astype(np.float32), np.array(ks, np.int32)
    t = (0.4 + 2 * rng.random(rows)).astype(np.float32)
    check_choose(net, x, rules, t, k, None, u)
    check_choose(net, x, rules, t, k, rng.random(rows).astype(np.float32), u)
    few = torch.from_numpy(rng.integers(0, 3, (rows, width)).astype(np.float32)).to("cuda:0")
    few[0] = -2.5
    check_choose(net, few, rules, None, None, rng.random(rows).astype(np.float32), u)
    check_choose(net, few, rules, t, k, rng.random(rows).astype(np.float32), u)


@pytest.mark.parametrize("width", [35, 224, 500, 4672, 40000])
@pytest.mark.parametrize("cut", ["none", "k", "p"])
def test_every_part_of_the_unit_interval(net, width, cut):
    """One row drawn from many times, at evenly spread numbers."""
    rng = np.random.default_rng(width)
    rows = 2000 if width < 5000 else 300
    one = some_logits(rng, 1, width, "f32")
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    k = np.full(rows, 20, np.int32) if cut == "k" else None
    p = np.full(rows, 0.9, np.float32) if cut == "p" else None
    x = one.expand(rows, width)
    assert x.stride(0) == 0
    a = plain_adjusted(one.cpu().numpy(), None)
    want, want_prob = plain_choice(np.broadcast_to(a, (rows, width)), None, k, p, u)
    col, act, prob = call_choose(net, x, None, None, k, p, u)
    assert np.array_equal(col, want) and np.array_equal(act, want)
    assert (np.abs(prob - want_prob) <= want_prob * 2 * U + width * 2.0 ** -41).all()


def test_long_lists(net):
    """Histories and bias lists of thousands of entries, over slots and over actions, each action many times."""
    rng = np.random.default_rng(12)
    for rows, width, actions, slots in ((3, 224, 4672, True), (3, 600, 4672, True), (3, 300, 300, False), (2, 9001, 9001, False)):
        x = some_logits(rng, rows, width, "f32")
        rules = some_rules(rng, rows, width, actions, slots, history=20000, bias=3000)
        check_adjust(net, x, rules, None)
