"""Timed cases of the policy operators: slot tables from move-list lengths, logits under penalties,
biases and masks, and the choice of one action per row.

``own`` selects the side: False computes each operator in elementary torch operations, True makes the
calls a user makes of ``marina_b200.network.B200Network``. A case's rows are positions (or requests),
its columns either legal slots, each naming an action through a table, or every action in order.
"""

import math

import numpy as np
import torch

own = False

ACTIONS = 4672  # 64 squares x 73 policy planes
SLOTS = 224     # legal slots a position has at most

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The root of a search: one position's move list becomes its slot row.
        {"name": "slots-1", "op": "slots", "rows": 1, "width": SLOTS},
        # The leaves of one evaluator batch.
        {"name": "slots-4096", "op": "slots", "rows": 4096, "width": SLOTS},
        # A scan over stored games, laid out at once before it is evaluated in chunks.
        {"name": "slots-262144", "op": "slots", "rows": 262144, "width": SLOTS},
        # One move to make: the root's slots, moves that repeat a position made less likely.
        {"name": "adjust-slots-1", "op": "adjust", "rows": 1, "width": SLOTS, "type": "f32", "slots": True,
         "history": 16, "bias": 8, "masked": False, "out": True, "priors": True},
        # A batch of games in parallel, one move each.
        {"name": "adjust-slots-8192", "op": "adjust", "rows": 8192, "width": SLOTS, "type": "f32", "slots": True,
         "history": 40, "bias": 8, "masked": False, "out": True, "priors": True},
        # Raw logits over every action with a legality mask per row, to priors.
        {"name": "adjust-actions-4096", "op": "adjust", "rows": 4096, "width": ACTIONS, "type": "f32", "slots": False,
         "history": 40, "bias": 16, "masked": True, "out": True, "priors": True},
        # A wide vocabulary of odd size under a grammar mask, half precision, long histories, in logits.
        {"name": "adjust-wide-100", "op": "adjust", "rows": 100, "width": 100003, "type": "f16", "slots": False,
         "history": 4096, "bias": 300, "masked": True, "out": True, "priors": False},
        # One move drawn for one game.
        {"name": "choose-slots-1", "op": "choose", "rows": 1, "width": SLOTS, "type": "f32", "slots": True,
         "history": 16, "bias": 8, "masked": False, "top_k": 0, "top_p": True},
        # One move drawn for each of a batch of games.
        {"name": "choose-slots-8192", "op": "choose", "rows": 8192, "width": SLOTS, "type": "f32", "slots": True,
         "history": 40, "bias": 8, "masked": False, "top_k": 0, "top_p": True},
        # Drawn from raw logits over every action, with both cut-offs.
        {"name": "choose-actions-2048", "op": "choose", "rows": 2048, "width": ACTIONS, "type": "f32", "slots": False,
         "history": 40, "bias": 0, "masked": True, "top_k": 40, "top_p": True},
        # A single row over a wide vocabulary, where latency counts.
        {"name": "choose-wide-1", "op": "choose", "rows": 1, "width": 131072, "type": "bf16", "slots": False,
         "history": 2000, "bias": 32, "masked": False, "top_k": 50, "top_p": True},
        # A decoding batch over a wide vocabulary of odd size, nearly the whole mass kept.
        {"name": "choose-wide-64", "op": "choose", "rows": 64, "width": 150001, "type": "bf16", "slots": False,
         "history": 500, "bias": 32, "masked": True, "top_k": 0, "top_p": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "adjust", "choose"])
    if op == "slots":
        width = _log(rng, 16, 512)
        return {"op": op, "rows": _log(rng, 1, min(262144, 262144 * SLOTS // width)), "width": width}
    slots = rng.random() < 0.4
    if slots:
        width = _log(rng, 8, 256)
        rows = _log(rng, 1, 8192 * SLOTS // max(width, SLOTS))
        history, bias = rng.choice([0, _log(rng, 1, 128)]), rng.choice([0, _log(rng, 1, 32)])
    else:
        width = _log(rng, 500, 200000)
        rows = _log(rng, 1, max(1, min(4096, (9_600_000 if op == "choose" else 19_000_000) // width)))
        history = rng.choice([0, _log(rng, 1, 4096)])
        bias = rng.choice([0, _log(rng, 1, min(300, width // 2))])
    case = {"op": op, "rows": rows, "width": width, "type": rng.choice(list(_TYPES)), "slots": slots,
            "history": history, "bias": bias, "masked": not slots and rng.random() < 0.6}
    if op == "adjust":
        kind = rng.choice(["both", "out", "priors"])
        case.update(out=kind != "priors", priors=kind != "out")
    else:
        case.update(top_k=rng.choice([0, _log(rng, 1, 200)]), top_p=rng.random() < 0.7)
    return case


def _lengths(rows, width, g):
    """Move-list lengths: about thirty of 224 slots, some positions with none, some with every slot."""
    dev = g.device
    # The lengths' distribution at evenly spread quantiles, in an order of the seed's: batches of one
    # size hold the same number of moves.
    q = (torch.arange(rows, device=dev) + 0.5) / rows
    n = torch.exp(torch.erfinv(2 * q - 1) * (0.6 * math.sqrt(2)) + math.log(max(1.0, width * 0.14)))
    n = n.round().clamp(1, width).to(torch.int32)
    if rows > 1:
        n[: (rows + 99) // 100] = 0
        n[rows - (rows + 199) // 200:] = width
    return n[torch.randperm(rows, generator=g, device=dev)]


def _distinct(rows, count, limit, g):
    """[rows, count] distinct ids below `limit` in each row, ascending."""
    step = torch.randint(1, max(2, limit // count + 1), (rows, count), generator=g, device=g.device, dtype=torch.int64)
    return (step.cumsum(1) - 1).to(torch.int32)


_network = None


def _net():
    """The evaluator a user's program holds; these calls need no more of it than its device and streams."""
    global _network
    if _network is None:
        from marina_b200 import model, weights
        from marina_b200.network import B200Network

        arch = model.Architecture(64, 1, 2, 128)
        _network = B200Network(arch, weights.random_init(arch), device=torch.cuda.current_device(), max_batch=1,
                               precision="bf16")
    return _network


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, width = case["rows"], case["width"]
    if case["op"] == "slots":
        lengths = _lengths(rows, width, g)
        total = int(lengths.sum())
        s = {"op": "slots", "rows": rows, "width": width, "lengths": lengths, "total": total,
             "entries": torch.randint(0, ACTIONS, (max(total, 1),), generator=g, device=dev, dtype=torch.int32)[:total]}
        if own:
            s["net"] = _net()
            s["starts"] = torch.empty(rows + 1, dtype=torch.int32, device=dev)
            s["table"] = torch.empty((rows, width), dtype=torch.int32, device=dev)
            s["map"] = torch.empty(total, dtype=torch.int32, device=dev)
        return s

    actions = ACTIONS if case["slots"] else width
    s = {"op": case["op"], "rows": rows, "width": width, "actions": actions, "type": case["type"]}
    logits = torch.randn((rows, width), generator=g, device=dev) * 2.5
    if case["slots"]:
        n = _lengths(rows, width, g)
        ids = _distinct(rows, width, actions, g)
        empty = torch.arange(width, device=dev)[None, :] >= n[:, None]
        s["columns"] = ids.masked_fill(empty, -1)
        logits.masked_fill_(empty, -math.inf)  # what the policy head leaves in empty slots
    if case["masked"]:
        words = (actions + 31) // 32
        few = torch.randint(-2**31, 2**31, (4, rows, words), generator=g, device=dev, dtype=torch.int64)
        mask = (few[0] & few[1] & few[2] & few[3]).to(torch.int32)  # about one action in sixteen
        mask[:, : min(words, 2)] |= few[0][:, : min(words, 2)].to(torch.int32)
        if rows > 8:
            mask[rows // 2] = 0  # a row that nothing is left of
        s["mask"] = mask
        # Masked places hold whatever the producer left there.
        junk = torch.randint(0, width, (rows, 4), generator=g, device=dev)
        allowed = (mask.gather(1, junk // 32) >> (junk % 32).to(torch.int32)) & 1
        values = torch.tensor([math.nan, math.inf, -math.inf, 60000.0], device=dev).expand(rows, 4)
        logits.scatter_(1, junk, torch.where(allowed == 1, torch.zeros_like(values), values))
    s["logits"] = logits.to(_TYPES[case["type"]])
    if case["history"]:
        h = case["history"]
        pick = torch.rand((rows, h), generator=g, device=dev) ** 3  # some actions many times, most never
        history = (pick * min(width, 4 * h + 8)).to(torch.int64).clamp(max=width - 1)
        history = s["columns"].gather(1, history) if case["slots"] else (history * 7 % width).to(torch.int32)
        s["history"] = history.contiguous()
        s["history_lens"] = torch.randint(0, h + 1, (rows,), generator=g, device=dev, dtype=torch.int32)
        s["repetition"] = 1 + torch.rand(rows, generator=g, device=dev) * 0.3
        s["presence"] = torch.rand(rows, generator=g, device=dev) * 0.4
        s["frequency"] = torch.rand(rows, generator=g, device=dev) * 0.2
    if case["bias"]:
        s["bias_actions"] = _distinct(1, case["bias"], actions, g)  # one list that every row shares
        s["bias_values"] = torch.randn((1, case["bias"]), generator=g, device=dev)
    t = 0.4 + torch.rand(rows, generator=g, device=dev)
    if case["op"] == "adjust":
        s["temperature"] = t
        s["out"], s["priors"] = case["out"], case["priors"]
    else:
        t[torch.rand(rows, generator=g, device=dev) < 0.05] = 0.0  # the largest logit's action
        s["temperature"] = t
        s["uniform"] = torch.rand(rows, generator=g, device=dev)
        if case["top_k"]:
            s["top_k"] = torch.randint(1, 2 * case["top_k"] + 1, (rows,), generator=g, device=dev, dtype=torch.int32)
        if case["top_p"]:
            s["top_p"] = 0.8 + 0.2 * torch.rand(rows, generator=g, device=dev)
    if own:
        from marina_b200.network import LogitRules

        s["net"] = _net()
        ptr = {k: s[k].data_ptr() for k in ("columns", "mask", "bias_actions", "bias_values", "history", "history_lens",
                                            "repetition", "presence", "frequency") if k in s}
        s["rules"] = LogitRules(actions, columns_stride=width, mask_stride=(actions + 31) // 32,
                                bias_len=case["bias"], bias_stride=0, history_len=case["history"],
                                history_stride=case["history"], **ptr)
        if case["op"] == "adjust":
            s["out_buf"] = torch.empty_like(s["logits"]) if s["out"] else None
            s["priors_buf"] = torch.empty((rows, width), device=dev) if s["priors"] else None
        else:
            s["column_buf"] = torch.empty(rows, dtype=torch.int32, device=dev)
            s["action_buf"] = torch.empty(rows, dtype=torch.int32, device=dev)
            s["prob_buf"] = torch.empty(rows, device=dev)
    return s


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "slots":
        return _plain_slots(s)
    x = _plain_adjusted(s)
    return _plain_priors(s, x) if s["op"] == "adjust" else _plain_choice(s, x)


def _run_own(s):
    # The legacy default stream has the handle 1; 0 would name the evaluator's own stream.
    stream = torch.cuda.current_stream().cuda_stream or 1
    net, rows, width = s["net"], s["rows"], s["width"]
    if s["op"] == "slots":
        net.slot_table(rows, width, s["lengths"].data_ptr(), s["total"], s["entries"].data_ptr(),
                       s["starts"].data_ptr(), s["table"].data_ptr(), s["map"].data_ptr(), stream=stream)
        return {"starts": s["starts"], "table": s["table"], "map": s["map"]}
    if s["op"] == "adjust":
        out, priors = s["out_buf"], s["priors_buf"]
        net.adjust_logits(rows, width, s["logits"].data_ptr(), s["rules"], dtype=s["type"],
                          temperature_ptr=s["temperature"].data_ptr(),
                          out_ptr=None if out is None else out.data_ptr(),
                          priors_ptr=None if priors is None else priors.data_ptr(), stream=stream)
        return {k: v for k, v in (("logits", out), ("priors", priors)) if v is not None}
    net.choose_actions(rows, width, s["logits"].data_ptr(), s["rules"], s["column_buf"].data_ptr(),
                       s["action_buf"].data_ptr(), s["prob_buf"].data_ptr(), dtype=s["type"],
                       temperature_ptr=s["temperature"].data_ptr(),
                       top_k_ptr=s["top_k"].data_ptr() if "top_k" in s else None,
                       top_p_ptr=s["top_p"].data_ptr() if "top_p" in s else None,
                       uniform_ptr=s["uniform"].data_ptr(), stream=stream)
    return {"column": s["column_buf"], "action": s["action_buf"], "prob": s["prob_buf"]}


# ---- plain forms ---------------------------------------------------------------------------
def _plain_slots(s):
    rows, width, n = s["rows"], s["width"], s["lengths"].to(torch.int64)
    dev = n.device
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), n.cumsum(0)])
    t = torch.arange(s["total"], device=dev)
    row = torch.searchsorted(starts, t, right=True) - 1
    at = row * width + t - starts[row]
    table = torch.full((rows * width,), -1, dtype=torch.int32, device=dev)
    table[at] = s["entries"]
    return {"starts": starts.to(torch.int32), "table": table.view(rows, width), "map": at.to(torch.int32)}


def _plain_adjusted(s):
    """The adjusted logits in f32: each step of the definition rounded once, in its order."""
    rows, actions = s["rows"], s["actions"]
    x = s["logits"].float()
    dev = x.device
    columns = s.get("columns")
    safe = None if columns is None else columns.clamp(min=0).to(torch.int64)
    per_column = (lambda v: v) if columns is None else (lambda v: v.expand(rows, actions).gather(1, safe))
    if "history" in s:
        h = s["history"].to(torch.int64)
        live = (torch.arange(h.shape[1], device=dev)[None, :] < s["history_lens"][:, None]) & (h >= 0)
        count = torch.zeros((rows, actions), dtype=torch.int32, device=dev)
        count.scatter_add_(1, h.clamp(min=0), live.to(torch.int32))
        c = per_column(count).float()
        r = s["repetition"][:, None]
        y = torch.where(x > 0, x / r, x * r)
        y = y - s["frequency"][:, None] * c
        y = y - s["presence"][:, None]
        x = torch.where(c > 0, y, x)
    if "bias_actions" in s:
        delta = torch.zeros((1, actions), device=dev)
        delta.scatter_(1, s["bias_actions"].to(torch.int64), s["bias_values"])
        x = x + per_column(delta)
    if columns is not None:
        x = torch.where(columns >= 0, x, -math.inf)
    if "mask" in s:
        a = torch.arange(actions, device=dev)
        allowed = (s["mask"][:, a // 32] >> (a % 32).to(torch.int32)) & 1
        x = torch.where(per_column(allowed) == 1, x, -math.inf)
    return x


def _plain_priors(s, x):
    got = {}
    if s["out"]:
        got["logits"] = x.to(s["logits"].dtype)
    if s["priors"]:
        m = x.amax(1, keepdim=True)
        e = torch.where(x == -math.inf, 0.0, ((x - m) / s["temperature"][:, None]).exp())
        total = e.sum(1, keepdim=True)
        got["priors"] = torch.where(total > 0, e / total, 0.0)
    return got


def _plain_choice(s, x):
    rows, width = x.shape
    dev = x.device
    t = s["temperature"].double()[:, None]
    order = x.sort(stable=True, dim=1, descending=True)[1]
    z = x.double()
    z = (z - z.amax(1, keepdim=True)) / torch.where(t > 0, t, 1.0)
    w = torch.where(x == -math.inf, 0.0, z.exp()).gather(1, order)
    rank = torch.arange(width, device=dev)[None, :]
    if "top_k" in s:
        w = torch.where(rank < s["top_k"][:, None], w, 0.0)
    if "top_p" in s:
        p = s["top_p"].double()[:, None]
        before = w.cumsum(1) - w
        w = torch.where((p >= 1) | (rank == 0) | (before < p * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.zeros_like(w).scatter(1, order, w)
    total = w.sum(1)
    cum = w.cumsum(1)
    column = (cum <= (s["uniform"].double() * total)[:, None]).sum(1).clamp(max=width - 1)
    prob = w.gather(1, column[:, None])[:, 0] / total
    greedy = t[:, 0] <= 0
    column = torch.where(greedy, order[:, 0], column)
    prob = torch.where(greedy, 1.0, prob)
    empty = ~(total > 0)
    column = torch.where(empty, -1, column).to(torch.int32)
    action = column if s.get("columns") is None else \
        torch.where(empty, -1, s["columns"].gather(1, column.clamp(min=0).to(torch.int64)[:, None])[:, 0])
    return {"column": column, "action": action, "prob": torch.where(empty, 0.0, prob).float()}


# ---- the work of a pass --------------------------------------------------------------------
def work(case):
    rows, width = case["rows"], case["width"]
    if case["op"] == "slots":
        listed_moves = rows * width * 0.17  # mean share of the slots that hold a move
        return {"bytes": rows * 4 + (rows + 1) * 4 + listed_moves * 8 + rows * width * 4, "flops": 0}
    actions = ACTIONS if case["slots"] else width
    size = 4 if case["type"] == "f32" else 2
    b = rows * width * size + rows * 4 * 4
    b += rows * width * 4 if case["slots"] else 0
    b += rows * ((actions + 31) // 32) * 4 if case["masked"] else 0
    b += rows * (case["history"] * 4 + 16) if case["history"] else 0
    b += case["bias"] * 8
    if case["op"] == "adjust":
        b += rows * width * ((size if case["out"] else 0) + (4 if case["priors"] else 0))
    else:
        b += rows * 12
    return {"bytes": b, "flops": rows * width * 6}


# ---- the definition in 64 bits --------------------------------------------------------------
def _host(s):
    return {k: v.detach().float().cpu().numpy() if v.dtype in (torch.float16, torch.bfloat16)
            else v.detach().cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}


def _exact_row(s, a, r, step):
    """Row r's adjusted logits; `step` is the type each step is rounded to."""
    x = a["logits"][r].astype(step)
    ids = a["columns"][r] if "columns" in a else np.arange(x.size)
    live = ids >= 0
    if "history" in a:
        h = a["history"][r, : a["history_lens"][r]]
        count = np.bincount(h[h >= 0], minlength=s["actions"])[np.where(live, ids, 0)]
        seen = np.flatnonzero((count > 0) & live)
        rep, pre, fre = (step(a[k][r]) for k in ("repetition", "presence", "frequency"))
        y = x[seen]
        with np.errstate(invalid="ignore"):
            y = np.where(y > 0, y / rep, y * rep)
            x[seen] = (y - fre * count[seen].astype(step)) - pre
    if "bias_actions" in a:
        where = {int(i): c for c, i in enumerate(ids) if i >= 0} if "columns" in a else None
        for i, v in zip(a["bias_actions"][0], a["bias_values"][0]):
            c = int(i) if where is None else where.get(int(i))
            if c is not None:
                x[c] += step(v)
    if "mask" in a:
        bits = np.unpackbits(a["mask"][r].view(np.uint8), bitorder="little")[: s["actions"]]
        live = live & (bits[np.where(live, ids, 0)] == 1)
    x[~live] = -np.inf
    return x


def exact(case, seed):
    s = prepare(case, seed)
    a = _host(s)
    rows, width = case["rows"], case["width"]
    if case["op"] == "slots":
        return None  # whole numbers all through
    if case["op"] == "adjust":
        x = np.stack([_exact_row(s, a, r, np.float64) for r in range(rows)])
        got = {"logits": x} if case["out"] else {}
        if case["priors"]:
            m = x.max(1, keepdims=True)
            m[m == -np.inf] = 0
            e = np.exp((x - m) / a["temperature"].astype(np.float64)[:, None])
            total = e.sum(1, keepdims=True)
            got["priors"] = e / np.where(total > 0, total, 1)
        return got
    column, prob = np.full(rows, -1), np.zeros(rows)
    for r in range(rows):
        # Adjusted logits are f32 values by definition, each step rounded; what follows is exact.
        x = _exact_row(s, a, r, np.float32).astype(np.float64)
        left = np.flatnonzero(x > -np.inf)
        if left.size == 0:
            continue
        best = left[np.argsort(-x[left], kind="stable")]
        t = float(a["temperature"][r])
        if t <= 0:
            column[r], prob[r] = best[0], 1.0
            continue
        if "top_k" in a:
            best = best[: a["top_k"][r]]
        w = np.exp((x[best] - x[best[0]]) / t)
        if "top_p" in a and a["top_p"][r] < 1:
            ahead = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            kept = (ahead < float(a["top_p"][r]) * w.sum()) | (np.arange(w.size) == 0)
            best, w = best[kept], w[kept]
        order = np.argsort(best)
        best, w = best[order], w[order]
        cum = np.cumsum(w)
        at = min(int(np.searchsorted(cum, float(a["uniform"][r]) * cum[-1], side="right")), w.size - 1)
        column[r], prob[r] = best[at], w[at] / cum[-1]
    action = column if "columns" not in a else np.where(column >= 0, a["columns"][np.arange(rows), np.maximum(column, 0)], -1)
    return {"column": column.astype(np.int32), "action": action.astype(np.int32), "prob": prob}
